"""Every kernel variant of the dense layers is reached and held to the bound, and a seeded random sweep over sizes and options."""
import math
import random

import pytest
import torch

from test_gpu_linear import ops, run  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu

# (tokens, features, K) with the variant that the choice is expected to make for bf16 operands, and for 8-bit ones
SIZES = [(1, 28672, 1024), (1, 7168, 2048), (1, 4096, 4096), (1, 256, 7168), (20, 28672, 1024), (20, 6000, 2048), (20, 2048, 7168), (24, 256, 7168),
         (40, 28672, 1024), (64, 4096, 2048), (64, 2048, 7168), (64, 256, 7168), (128, 4096, 1024), (300, 2880, 1440), (300, 2048, 7168),
         (128, 256, 7168), (450, 256, 7168), (777, 128, 7168), (1500, 256, 7168), (100, 28672, 512), (777, 2048, 1024), (777, 2880, 1440), (1500, 2048, 1024),
         (2048, 7168, 512), (4096, 4096, 1024), (1500, 4096, 1024), (4096, 2880, 512), (2500, 7168, 1024)]


def plan(t, n, k, **kw):
    from paired_nvfp4_kernels import ops as module
    return module.linear_plan(t, n, k, **kw)


@pytest.mark.parametrize("mx8", [False, True])
def test_every_variant_is_reached(ops, mx8):  # noqa: F811
    seen = {}
    for t, n, k in SIZES + [(t, n, k) for t in (1, 20, 40, 100, 129, 200, 300, 450, 777, 1000, 1300, 1500, 2000, 3000, 4000)
                            for n in (64, 128, 256, 1024, 2048, 2880, 4096, 5760, 7168, 12000) for k in (512, 2048, 7168)]:
        if t * n * k <= 2 ** 34:
            seen.setdefault(plan(t, n, k, mx8=mx8), (t, n, k))
    split = {p[1:] for p in seen if p[0] == "split"}
    assert {s[0] for s in split} == {16, 32, 64, 128} and {s[1] for s in split} == {1, 2, 4, 8}
    assert {p[1] for p in seen if p[0] == "pair"} >= ({128, 192, 256} if mx8 else {128, 160, 192, 224, 256})
    for (t, n, k) in seen.values():
        run(ops, t, n, k, mx8=mx8, bias=torch.bfloat16, residual=True, seed=t + n + k)


@pytest.mark.parametrize("t,n,k", SIZES)
@pytest.mark.parametrize("mx8", [False, True])
def test_sizes_between_the_variants(ops, t, n, k, mx8):  # noqa: F811
    run(ops, t, n, k, mx8=mx8, seed=n)
    if n % 64 == 0:
        run(ops, t, n, k, mx8=mx8, gated=True, activation="silu", residual=True, seed=n + 1)


# 8-bit operands, several tiles a pair of CTAs: with two accumulators (192 features) and with one (256)
@pytest.mark.parametrize("t,n,k,width", [(1056, 4096, 2048, 192), (4674, 2048, 768, 192), (834, 5120, 2048, 192), (1550, 2880, 512, 192), (4096, 4096, 1024, 256)])
def test_accumulators_in_turn(ops, t, n, k, width):  # noqa: F811
    assert plan(t, n, k, mx8=True) == ("pair", width) and -(-t // 256) * -(-n // width) > 74
    for residual in (False, True):
        run(ops, t, n, k, mx8=True, residual=residual, seed=t)
    run(ops, t, n, k, mx8=True, bias=torch.float32, activation="gelu", seed=t + 1)


# weights that come from memory, not from L2: the copies of a stage ring land out of order
@pytest.mark.parametrize("t", [8, 32, 40, 128, 300])
@pytest.mark.parametrize("mx8", [False, True])
def test_weights_larger_than_l2(ops, t, mx8):  # noqa: F811
    from test_gpu_linear import rows
    n, k = 40960, 4096
    x, w = rows(t, k, 1), rows(n, k, 2, 1 / 64)
    got = ops.linear_mx8(*ops.quant_mx8(x), *ops.quant_mx8(w)) if mx8 else ops.linear(x, w)
    part = torch.randperm(n, generator=torch.Generator().manual_seed(3))[:512].cuda()
    want = ops.linear_mx8(*ops.quant_mx8(x), *ops.quant_mx8(w[part])) if mx8 else ops.linear(x, w[part])
    # the same sums in another order of pieces: an instruction's error and the rounding of either
    mag = x.double().abs() @ w[part].double().abs().T * (1.07 if mx8 else 1.0)
    off = (got[:, part].double() - want.double()).abs()
    assert bool((off <= mag * (k // 16) * 2.0 ** -21 + want.double().abs() * 2.0 ** -7).all())


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


@pytest.mark.parametrize("seed", range(60))
def test_random_calls(ops, seed):  # noqa: F811
    rng = random.Random(seed)
    mx8, gated = rng.random() < 0.5, rng.random() < 0.35
    k = 32 * _log(rng, 1, 256) if mx8 else 8 * _log(rng, 1, 1024)
    n = 64 * _log(rng, 1, 96) if gated else _log(rng, 1, 6000)
    t = _log(rng, 1, max(2, min(6000, 2 ** 33 // (n * k))))
    activation = rng.choice(["silu", "situ"]) if gated else rng.choice(["none", "none", "relu", "silu", "gelu"])
    run(ops, t, n, k, mx8=mx8, gated=gated, activation=activation, bias=rng.choice([None, torch.bfloat16, torch.float32]),
        residual=rng.random() < 0.5, float_out=not mx8 and rng.random() < 0.3, beta=1.702, linear_beta=rng.choice([1.0, -1.0]), seed=seed)
