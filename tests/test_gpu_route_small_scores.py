"""Renormalized weights of route_topk where the scores of the chosen are too small for 32 bits: a bias (a mask of -infinity, say)
chooses experts far below the row's best, or all sigmoids of a row are tiny."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import paired_nvfp4_kernels  # noqa: F401
    return torch.ops.paired_nvfp4


def check(w, ids, logits, scoring, scale):
    """In logarithms, in 64 bits.  The exponent is a difference d of logits, rounded: 2^-24 of d; then what the weights' other tests
    count, 48 units of 2^-24."""
    chosen = logits.cpu().double().gather(1, ids.cpu().long())
    log_score = chosen if scoring == "softmax" else torch.nn.functional.logsigmoid(chosen)
    d = log_score - log_score.amax(-1, keepdim=True)
    want = torch.softmax(log_score, -1) * scale
    off = (w.cpu().double() - want).abs()
    assert bool((off <= want * (48 + d.abs()) * 2.0 ** -24 + 1e-37).all()), (off / want).max()
    assert bool(((w.sum(-1) - scale).abs() <= 48 * 2.0 ** -24 * scale).all())


@pytest.mark.parametrize("gap", [20.0, 88.0, 95.0, 104.0, 150.0, 1e4])
@pytest.mark.parametrize("experts,topk,groups", [(8, 1, 1), (8, 3, 1), (64, 8, 1), (64, 6, 8), (256, 8, 1), (500, 32, 1)])
@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_softmax_of_experts_far_below_the_best(ops, gap, experts, topk, groups, masked, dtype):
    """The first half's logits are `gap` above; a bias keeps them out, or brings the others in."""
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn((20, experts), generator=g)
    logits[:, :experts // 2] += gap
    logits = logits.to(dtype).cuda()
    bias = torch.zeros(experts)
    if masked:
        bias[:experts // 2] = -math.inf
    else:
        bias[experts // 2:] = 10.0
    w, ids = ops.route_topk(logits, topk, "softmax", bias.cuda(), groups, max(1, groups // 2), True, 2.5)
    assert bool((ids >= experts // 2).all())
    check(w, ids, logits.float(), "softmax", 2.5)


@pytest.mark.parametrize("level", [-10.0, -17.0, -30.0, -80.0, -88.0, -100.0, -104.0, -500.0, -1e5])
@pytest.mark.parametrize("experts,topk,groups", [(8, 1, 1), (64, 8, 1), (64, 6, 8), (300, 32, 1)])
@pytest.mark.parametrize("biased", [True, False])
def test_small_sigmoids(ops, level, experts, topk, groups, biased):
    g = torch.Generator().manual_seed(experts)
    logits = (level + 2 * torch.randn((20, experts), generator=g)).cuda()
    bias = 0.1 * torch.randn(experts, generator=g).cuda() if biased else None
    w, ids = ops.route_topk(logits, topk, "sigmoid", bias, groups, max(1, groups // 2), True, 2.5)
    check(w, ids, logits, "sigmoid", 2.5)


def test_scores_that_are_zero(ops):
    """Nothing to renormalize: weights 0."""
    inf = math.inf
    logits = torch.tensor([[-inf] * 4 + [1.0] * 4, [-inf, -inf, -inf, -90.0] + [1.0] * 4, [1.0, 2.0, 3.0, 4.0] + [inf] * 4]).cuda()
    bias = torch.tensor([0.0] * 4 + [-inf] * 4).cuda()
    for scoring in ("softmax", "sigmoid"):
        w, ids = ops.route_topk(logits, 2, scoring, bias)
        assert w[0].tolist() == [0, 0] and ids[0].tolist() == [0, 1]
        assert w[1].tolist() == [1, 0] and ids[1].tolist() == [3, 0]
    w, _ = ops.route_topk(logits[2:], 2, "softmax", bias)
    assert w[0].tolist() == [0, 0]
    w, ids = ops.route_topk(logits[:1, :4], 2, "sigmoid")
    assert w[0].tolist() == [0, 0]


def test_not_renormalized_sigmoids_reach_down(ops):
    """exp(l) below -17: to the smallest numbers that 32 bits hold."""
    l = torch.linspace(-16, -103, 64)
    w, ids = ops.route_topk(l[None].cuda(), 32, "sigmoid", renormalize=False)
    want = torch.sigmoid(l[:32].double())
    assert ids[0].tolist() == list(range(32)) and bool(((w[0].cpu().double() - want).abs() <= want * 48 * 2.0 ** -24).all())
    w, ids = ops.route_topk(l[None, 32:].contiguous().cuda(), 32, "sigmoid", renormalize=False)
    want = torch.sigmoid(l[32:].double())
    assert bool(((w[0].cpu().double() - want).abs() <= want * 48 * 2.0 ** -24 + 2.0 ** -149).all())
