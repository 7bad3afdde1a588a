"""GELU where its factor 1 + erf would cancel: products that are known exactly, negative ones out to where the result underflows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from paired_nvfp4_kernels import ops as module
    yield torch.ops.paired_nvfp4
    assert module.linear_device_status() == 0


def bound(v, y, out_eps):
    """exp(-v^2 / 2) t Q(t) |v|, units of 2^-23: the fit 0.3; Q's rounded coefficients and steps 2 (its terms' magnitudes add up to
    twice the sum); t 1.5, which t Q(t) answers with up to 1.6 times that; the exponential 2; three products 1.5; in all less than 10.
    The exponent v^2 log2(e) / 2 is rounded twice, 2^-24 of v^2 / 2 each and as much for its constant: less than v^2 more.  Numbers
    below the smallest normal one may come out as anything up to it."""
    rel = (10 + v * v) * 2.0 ** -23
    return y.abs() * (rel + out_eps * (1 + rel)) + torch.finfo(torch.float32).tiny


# tokens: a narrow and a wide tile of the split kernel, the pair kernel (bf16 results)
@pytest.mark.parametrize("t,n", [(1, 512), (100, 640), (3000, 2304)])
@pytest.mark.parametrize("float_out", [False, True])
def test_gelu_of_known_products(ops, t, n, float_out):
    v = torch.linspace(-14, 6, n).to(torch.bfloat16)
    x, w = torch.zeros((t, 64), dtype=torch.bfloat16), torch.zeros((n, 64), dtype=torch.bfloat16)
    x[:, 5], w[:, 5] = 1, v
    got = ops.linear(x.cuda(), w.cuda(), activation="gelu", float_out=float_out).double().cpu()
    v = v.double()
    want = 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    off, allowed = (got - want).abs(), bound(v, want, 0.0 if float_out else torch.finfo(torch.bfloat16).eps / 2)
    assert bool((off <= allowed).all()), (v[(off > allowed).any(0)][:5], float((off / allowed).max()))


def test_gelu_of_known_products_mx8(ops):
    """The same through 8-bit operands: powers of two and their sums, which the codes hold exactly."""
    v = -torch.tensor([0.25, 0.5, 1, 1.5, 2, 2.5, 3, 3.5, 4, 4.5, 5, 5.5, 6, 6.5, 7, 7.5, 8, 9, 10, 11, 12, 13]).repeat(7)[:130]
    for t in (3, 2600):
        x, w = torch.zeros((t, 64), dtype=torch.bfloat16), torch.zeros((130, 64), dtype=torch.bfloat16)
        x[:, 5], w[:, 5] = 1, v.to(torch.bfloat16)
        got = ops.linear_mx8(*ops.quant_mx8(x.cuda()), *ops.quant_mx8(w.cuda()), activation="gelu").double().cpu()
        want = 0.5 * v.double() * torch.special.erfc(-v.double() / math.sqrt(2))
        off, allowed = (got - want).abs(), bound(v.double(), want, torch.finfo(torch.bfloat16).eps / 2)
        assert bool((off <= allowed).all()), v[(off > allowed).any(0)][:5]


def test_gelu_of_infinities_and_nan(ops):
    """The limits: infinity, and 0 below."""
    x, w = torch.zeros((3, 64), dtype=torch.bfloat16), torch.zeros((130, 64), dtype=torch.bfloat16)
    x[:, 5], w[:, 5] = torch.tensor([math.inf, -math.inf, math.nan]), 1
    for many in (1, 900):
        got = ops.linear(x.repeat(many, 1).cuda(), w.cuda(), activation="gelu").view(many, 3, -1)
        assert bool((got[:, 0] == math.inf).all()) and bool((got[:, 1] == 0).all()) and bool(torch.isnan(got[:, 2]).all())
