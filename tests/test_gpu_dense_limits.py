"""The operators around the grouped GEMM where calls meet their limits: offsets past 32 bits, few SMs, a first call inside a
capture, several host threads."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import dense_reference as ref
from test_gpu_linear import check, rows
from test_gpu_norm import F32, check_codes

pytestmark = pytest.mark.gpu

WIDE = 8192
MANY = 2 ** 31 // WIDE + 1000        # rows of WIDE elements that pass 2^31 elements


@pytest.fixture(scope="module")
def ops():
    from paired_nvfp4_kernels import ops as module
    yield torch.ops.paired_nvfp4
    assert module.linear_device_status() == 0


@pytest.fixture(scope="module")
def big():
    """[MANY, WIDE] bf16: one block of random rows over and over, every row scaled by its number."""
    x = torch.empty((MANY, WIDE), dtype=torch.bfloat16, device="cuda")
    base = rows(4096, WIDE, 1)
    for i in range(0, MANY, 4096):
        n = min(4096, MANY - i)
        x[i:i + n] = base[:n] * (1 + (i // 4096) % 7)
    yield x
    del x
    torch.cuda.empty_cache()


def test_norm_and_quantizer_past_32_bits(ops, big):
    w = (1 + 0.1 * torch.randn(WIDE, generator=torch.Generator().manual_seed(2))).cuda()
    y, res, q, sf = ops.add_rms_norm(big, big, w, 1e-6, True, True)
    last = big[-300:].cpu()
    v, n = ref.norm(last, last, w.cpu(), 1e-6)
    assert bool(((y[-300:].cpu().double() - n).abs() <= n.abs() * (ref.BF16 + 2 * F32)).all())
    assert torch.equal(res[-300:].cpu(), v.float().to(torch.bfloat16))
    first = (MANY - 300) // 128 * 128                             # whole atoms from here on
    v, n = ref.norm(big[first:].cpu(), big[first:].cpu(), w.cpu(), 1e-6)
    check_codes(q[first:], sf[first // 128 * (WIDE // 128) * 512:], n, MANY - first, WIDE)
    del y, res, q, sf
    q, sf = ops.quant_mx8(big)
    code, want = ref.encode(big[first:].cpu().double())
    assert torch.equal(q[first:].view(torch.uint8).cpu(), code)
    tail = sf.view(torch.uint8)[first // 128 * (WIDE // 128) * 512:]
    assert torch.equal(ref.scale_rows(tail, MANY - first, WIDE)[:MANY - first, :WIDE // 32], want)


@pytest.mark.parametrize("n", [40, 600])
def test_linear_past_32_bits(ops, big, n):
    w = rows(n, WIDE, 3, WIDE ** -0.5)
    residual = big[:, :n]                                         # rows WIDE apart
    out = ops.linear(big, w, None, residual)
    want, bound = ref.linear(big[-300:], w, None, residual[-300:], "none", False)
    check(out[-300:], want, bound)
    out = ops.linear(big, w, float_out=True)
    want, bound = ref.linear(big[-300:], w, None, None, "none", False, chunk=512, out_eps=2.0 ** -24)
    check(out[-300:], want, bound)


@pytest.mark.parametrize("mx8", [False, True])
def test_output_past_32_bits(ops, mx8):
    t, n, k = 40000, 60000, 64
    x, w = rows(t, k, 4), rows(n, k, 5, 0.125)
    if mx8:
        (q, sf), (wq, wsf) = ops.quant_mx8(x), ops.quant_mx8(w)
        out = ops.linear_mx8(q, sf, wq, wsf)
        x = ref.decode(q, ref.scale_rows(sf, t, k)[:t, :k // 32]).cuda()
        w = ref.decode(wq, ref.scale_rows(wsf, n, k)[:n, :k // 32]).cuda()
    else:
        out = ops.linear(x, w)
    assert out.numel() > 2 ** 31
    for r, c in ((slice(-200, None), slice(-300, None)), (slice(0, 200), slice(0, 300)), (slice(35700, 35900), slice(29900, 30200))):
        want, bound = ref.linear(x[r], w[c], None, None, "none", False, k_step=32 if mx8 else 16)
        check(out[r, c], want, bound)


def test_routing_past_32_bits(ops):
    experts, t = 1000, 2 ** 31 // 1000 + 500
    logits = torch.empty((t, experts), dtype=torch.bfloat16, device="cuda")
    base = torch.randn((5000, experts), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").to(torch.bfloat16)
    for i in range(0, t, 5000):
        n = min(5000, t - i)
        logits[i:i + n] = base[:n].roll(i // 5000, 1)
    w, ids = ops.route_topk(logits, 8)
    want_w, want_ids = ref.route(logits[-40:], 8, "softmax")
    assert torch.equal(ids[-40:].cpu(), want_ids) and bool(((w[-40:].cpu().double() - want_w).abs() <= want_w * 48 * 2.0 ** -24).all())


def test_few_sms(ops):
    from paired_nvfp4_kernels import ops as module
    sizes = ((1, 256, 4096), (64, 2048, 2048), (777, 2880, 512), (3000, 2304, 256))
    calls = [(rows(t, k, t), rows(n, k, n, 0.02)) for t, n, k in sizes]
    logits = torch.randn((500, 128), generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    want = [ref.linear(x, w, None, None, "none", False) for x, w in calls]
    _, ids = ops.route_topk(logits, 8)
    try:
        for margin in (100, 146, 147):
            module.set_sm_margin(margin)
            for (x, w), (v, bound) in zip(calls, want):
                check(ops.linear(x, w), v, bound)
                check(ops.linear(x, w, float_out=True), v, bound)
            assert torch.equal(ops.route_topk(logits, 8)[1], ids)
    finally:
        module.set_sm_margin(0)


FIRST_CALL = """
import sys, torch
sys.path.insert(0, {package!r})
import paired_nvfp4_kernels
ops = torch.ops.paired_nvfp4
x = torch.randn((300, 512), device="cuda").to(torch.bfloat16)
w = torch.randn((640, 512), device="cuda").to(torch.bfloat16)
logits = torch.randn((300, 64), device="cuda")
scale = torch.ones(512, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = [ops.linear(x, w), ops.linear(x[:3], w, float_out=True), *ops.quant_mx8(x), *ops.add_rms_norm(x, x, scale, 1e-6, True, True),
           *ops.route_topk(logits, 4), ops.linear_mx8(*ops.quant_mx8(x), *ops.quant_mx8(w))]
graph.replay()
torch.cuda.synchronize()
want = [ops.linear(x, w), ops.linear(x[:3], w, float_out=True), *ops.quant_mx8(x), *ops.add_rms_norm(x, x, scale, 1e-6, True, True),
        *ops.route_topk(logits, 4), ops.linear_mx8(*ops.quant_mx8(x), *ops.quant_mx8(w))]
assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
print("captured")
"""


def test_first_call_inside_a_capture():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grouped-sparse-gemm_b200")
    p = subprocess.run([sys.executable, "-c", FIRST_CALL.format(package=package)], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]


def test_several_host_threads(ops):
    """Calls from four threads, each on a stream and on operands of its own."""
    work = []
    for i in range(4):
        x, w = rows(50 + 40 * i, 1024, i), rows(512 + 64 * i, 1024, 10 + i, 0.03)
        work.append((x, w, ops.linear(x, w), ops.linear_mx8(*ops.quant_mx8(x), *ops.quant_mx8(w))))
    torch.cuda.synchronize()
    bad = []

    def call(x, w, want, want8):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                a, b = ops.linear(x, w), ops.linear_mx8(*ops.quant_mx8(x), *ops.quant_mx8(w))
            torch.cuda.current_stream().synchronize()
            if not (torch.equal(a, want) and torch.equal(b, want8)):
                bad.append(x.size(0))

    threads = [threading.Thread(target=call, args=a) for a in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_float_results_warn_in_backward(ops):
    import warnings
    x = rows(4, 64, 1).requires_grad_()
    w = rows(64, 64, 2)
    y = ops.linear(x * 1, w)
    assert y.requires_grad and y.grad_fn is not None
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        y.float().sum().backward()
    assert any("autograd kernel was not registered" in str(m.message) for m in seen)
