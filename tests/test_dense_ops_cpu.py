"""What the operators around the grouped GEMM refuse, on the host: checked before anything is launched."""
import pytest
import torch

A = 0x100000           # stands for an aligned device address; nothing reads it
INVALID, CUDA = 1, 2


@pytest.fixture(scope="module")
def cabi():
    import paired_nvfp4_kernels  # noqa: F401
    from paired_nvfp4_kernels import _cabi
    return _cabi


NORM = dict(x=A, x_stride=64, residual=A, residual_stride=64, weight=A, f32=0, eps=1e-6, rows=5, width=64, y=A, residual_out=A, q=A, q_sf=A,
            sms=0, stream=None)
QUANT = dict(x=A, x_stride=64, rows=5, k=64, q=A, q_sf=A, stream=None)
LINEAR = dict(out=A, out_f32=0, x=A, x_stride=64, w=A, bias=A, bias_f32=0, residual=A, residual_stride=128, rows=5, features=128, k=64, act=2,
              gated=0, beta=1.0, linear_beta=-1.0, sms=0, stream=None)
MX8 = dict(out=A, x=A, x_sf=A, w=A, w_sf=A, bias=A, bias_f32=0, residual=A, residual_stride=128, rows=5, features=128, k=64, act=2, gated=0,
           beta=1.0, linear_beta=-1.0, sms=0, stream=None)
ROUTE = dict(logits=A, bf16=0, stride=64, rows=5, experts=64, topk=8, sigmoid=0, bias=A, groups=4, topk_groups=2, renorm=1, scale=1.0, w=A, ids=A,
             sms=0, stream=None)

CASES = [
    ("pnv_add_rms_norm", NORM, [
        (dict(rows=-1), "row count"), (dict(width=0), "1 to"), (dict(width=32769), "1 to"), (dict(y=None, q=None, q_sf=None), "at least one"),
        (dict(q_sf=None), "null"), (dict(width=40), "multiple of 32"), (dict(eps=-1.0), "eps"), (dict(x=None), "null"), (dict(weight=None), "null"),
        (dict(residual_out=None), "null"), (dict(residual=None), "null"), (dict(x_stride=63), "overlap"), (dict(residual_stride=63), "overlap"),
        (dict(x=A + 1), "aligned"), (dict(weight=A + 2, f32=1), "aligned"), (dict(q=A + 4), "aligned"), (dict(q_sf=A + 2), "aligned"),
        (dict(y=A + 1), "aligned"), (dict(eps=float("nan")), "eps")]),
    ("pnv_quant_mx8", QUANT, [
        (dict(k=0), "multiple"), (dict(k=48), "multiple"), (dict(rows=-1), "row count"), (dict(rows=1 << 31), "row count"), (dict(x=None), "null"),
        (dict(q=None), "null"), (dict(q_sf=None), "null"), (dict(x_stride=60), "overlap"), (dict(x_stride=68), "16 bytes"), (dict(x=A + 8), "aligned"),
        (dict(q=A + 8), "aligned"), (dict(q_sf=A + 2), "aligned"), (dict(rows=(1 << 31) - 1, k=512, x_stride=512), "too many")]),
    ("pnv_linear", LINEAR, [
        (dict(rows=-1), "row count"), (dict(rows=(1 << 31) - 1), "row count"), (dict(features=0), "positive"), (dict(k=0), "positive"),
        (dict(k=60), "multiple of 8"), (dict(k=1 << 29), "too large"), (dict(act=1), "activation"), (dict(act=5), "activation"),
        (dict(act=2, gated=1), "activation"), (dict(act=0, gated=1, features=96), "multiple of 64"), (dict(act=1, gated=1, beta=0.0), "beta"),
        (dict(out=None), "null"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(x_stride=56), "overlap"), (dict(x_stride=68), "16 bytes"),
        (dict(x=A + 8), "aligned"), (dict(w=A + 2), "aligned"), (dict(out=A + 1), "aligned"), (dict(out=A + 2, out_f32=1), "aligned"),
        (dict(bias=A + 2, bias_f32=1), "aligned"), (dict(residual=A + 1), "aligned"), (dict(residual_stride=127), "overlap")]),
    ("pnv_linear_mx8", MX8, [
        (dict(k=48), "multiple of 32"), (dict(x_sf=None), "null"), (dict(w_sf=None), "null"), (dict(x_sf=A + 8), "aligned"), (dict(w_sf=A + 4), "aligned"),
        (dict(x=A + 8), "aligned"), (dict(act=4, gated=1), "activation")]),
    ("pnv_route_topk", ROUTE, [
        (dict(rows=-1), "row count"), (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(groups=0), "groups"), (dict(groups=5), "groups"),
        (dict(groups=64), "groups"), (dict(topk_groups=0), "topk_groups"), (dict(topk_groups=5), "topk_groups"), (dict(topk=0), "topk"),
        (dict(topk=33), "topk"), (dict(topk_groups=1, topk=17), "topk"), (dict(logits=None), "null"), (dict(w=None), "null"), (dict(ids=None), "null"),
        (dict(stride=63), "overlap"), (dict(logits=A + 2), "aligned"), (dict(logits=A + 1, bf16=1), "aligned"), (dict(bias=A + 2), "aligned")]),
]


@pytest.mark.parametrize("name,base,refused", CASES, ids=[c[0] for c in CASES])
def test_refusals(cabi, name, base, refused):
    for change, what in refused:
        rc = getattr(cabi.lib, name)(*{**base, **change}.values())
        msg = cabi.lib.pnv_last_error().decode()
        assert rc == INVALID and what in msg, (change, rc, msg)


@pytest.mark.parametrize("name,base", [c[:2] for c in CASES], ids=[c[0] for c in CASES])
def test_no_rows_is_no_call(cabi, name, base):
    """Nothing is launched, nothing dereferenced: pointers may be null."""
    args = {**base, "rows": 0}
    for k in args:
        if args[k] == A and k not in ("y",):
            args[k] = None
    if name == "pnv_add_rms_norm":
        args.update(y=A)
    assert getattr(cabi.lib, name)(*args.values()) == 0, cabi.lib.pnv_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls would be launched; their pointers stand for nothing")
@pytest.mark.parametrize("name,base", [c[:2] for c in CASES], ids=[c[0] for c in CASES])
def test_what_is_allowed_passes_the_checks(cabi, name, base):
    """Without a device the launch or its set-up fails, with another code."""
    assert getattr(cabi.lib, name)(*base.values()) == CUDA


def test_schemas(cabi):
    ns = torch.ops.paired_nvfp4
    assert "bool out_bf16=True, bool out_mx8=False" in str(ns.add_rms_norm.default._schema)
    assert 'str activation="none", bool gated=False, bool float_out=False' in str(ns.linear.default._schema)
    assert "Tensor q, Tensor q_sf, Tensor weight, Tensor weight_sf" in str(ns.linear_mx8.default._schema)
    assert 'str scoring="softmax", Tensor? bias=None, int groups=1, int topk_groups=1' in str(ns.route_topk.default._schema)


def test_cpu_tensors_are_rejected_not_computed(cabi):
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((64, 64), dtype=torch.bfloat16)
    for call in (lambda: torch.ops.paired_nvfp4.add_rms_norm(x, None, w[0]), lambda: torch.ops.paired_nvfp4.quant_mx8(x),
                 lambda: torch.ops.paired_nvfp4.linear(x, w), lambda: torch.ops.paired_nvfp4.route_topk(x, 2)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_float_results_say_that_they_have_no_backward(cabi):
    """torch's autograd fallback is left in place (it marks floating-point results)."""
    for op in ("add_rms_norm", "quant_mx8", "linear", "linear_mx8", "route_topk"):
        assert not torch._C._dispatch_has_kernel_for_dispatch_key(f"paired_nvfp4::{op}", "AutogradCUDA")
