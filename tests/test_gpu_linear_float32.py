"""float32 results of linear: the tensor core's accumulators are emptied every 512 K, or their truncation would show.

Adding 16 products to an accumulator drops what lies below its last bit, towards zero: less than one unit, 2^-23 of the sum so
far.  Of products of one sign a piece of 512 K (32 instructions) has i / 32 of its sum after i of them, so it loses less than
(1 + ... + 32) / 32 = 16.5 units, 2.0e-6, whatever K is, and half a unit per instruction, 0.7 of a unit to a power of two, on average:
7e-7.  The pieces' additions round to nearest.  One accumulator over all of K = 7168 loses about 14 times as much, two of them half
of that each.  Random products lose less (their partial sums are smaller than the sum of magnitudes, and cancel): the slope of the
result on the exact one is held to the 1e-6 that the header states."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ONE_SIGN = 16.5 * 2.0 ** -23 + 8 * 2.0 ** -24        # the pieces' and partners' additions among it
STATED = 1e-6


@pytest.fixture(scope="module")
def ops():
    from paired_nvfp4_kernels import ops as module
    yield torch.ops.paired_nvfp4
    assert module.linear_device_status() == 0


def operands(t, n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple(torch.randn((r, k), generator=g, device="cuda").to(torch.bfloat16) for r in (t, n))


def sample(t, n):
    """Up to 128 rows and 512 columns, the last ones among them."""
    r, c = (torch.unique(torch.cat([torch.randperm(m, generator=torch.Generator().manual_seed(m))[:s - 1], torch.tensor([m - 1])])).cuda()
            for m, s in ((t, 128), (n, 512)))
    return r, c


def split_of(t, n, k):
    from paired_nvfp4_kernels import ops as module
    kind, tokens, split = module.linear_plan(t, n, k, float_out=True)
    return split


# one CTA to a tile's K (chunks of 512 in each of two accumulators), and clusters that share it
SIZES = [(1024, 4096, 7168, False), (200, 20000, 14336, False), (2000, 2560, 7160, False), (16, 256, 7168, True), (64, 2048, 14336, True),
         (128, 1024, 28672, True)]


@pytest.mark.parametrize("t,n,k,shared", SIZES)
def test_one_sign(ops, t, n, k, shared):
    assert (split_of(t, n, k) > 1) == shared
    x, w = (v.abs() for v in operands(t, n, k, t))
    r, c = sample(t, n)
    got = ops.linear(x, w, float_out=True)[r][:, c].double()
    want = x[r].double() @ w[c].double().T
    assert float(((got - want).abs() / want).max()) <= ONE_SIGN


@pytest.mark.parametrize("t,n,k,shared", SIZES)
def test_slope_of_random_sums(ops, t, n, k, shared):
    x, w = operands(t, n, k, t + 1)
    r, c = sample(t, n)
    got = ops.linear(x, w, float_out=True)[r][:, c].double()
    want = x[r].double() @ w[c].double().T
    assert abs(float(((got - want) * want).sum() / (want * want).sum())) <= STATED
    assert float((got - want).square().mean().sqrt() / want.square().mean().sqrt()) <= STATED


@pytest.mark.parametrize("margin", [100, 146, 147])
def test_few_sms(ops, margin):
    from paired_nvfp4_kernels import ops as module
    try:
        module.set_sm_margin(margin)
        for t, n, k in ((1, 256, 7168), (64, 2048, 7168), (777, 512, 7168)):
            x, w = operands(t, n, k, margin)
            want = x.double() @ w.double().T
            got = ops.linear(x, w, float_out=True).double()
            assert float((got - want).square().mean().sqrt() / want.square().mean().sqrt()) <= STATED
            x, w = x.abs(), w.abs()
            want = x.double() @ w.double().T
            assert float(((ops.linear(x, w, float_out=True).double() - want).abs() / want).max()) <= ONE_SIGN
    finally:
        module.set_sm_margin(0)
