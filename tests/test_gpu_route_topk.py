"""route_topk against a row-by-row selection in 64 bits; ids have to be equal."""
import math

import pytest
import torch

import dense_reference as ref

pytestmark = pytest.mark.gpu

# weights: exponentials (2 units), their sum (tree and up to 32 in a row), quotients
WEIGHT = 48 * 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    import paired_nvfp4_kernels  # noqa: F401
    return torch.ops.paired_nvfp4


def check(ops, logits, topk, scoring="softmax", bias=None, groups=1, topk_groups=1, renormalize=True, scale=1.0):
    w, ids = ops.route_topk(logits, topk, scoring, bias, groups, topk_groups, renormalize, scale)
    want_w, want_ids = ref.route(logits.cpu(), topk, scoring, None if bias is None else bias.cpu(), groups, topk_groups, renormalize, scale)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), want_ids)
    assert bool(((w.cpu().double() - want_w).abs() <= want_w.abs() * WEIGHT + 1e-37).all())


def make(rows, experts, seed, std=1.5):
    return torch.randn((rows, experts), generator=torch.Generator().manual_seed(seed)).mul(std).cuda()


@pytest.mark.parametrize("rows,experts,topk", [(1, 1, 1), (3, 3, 3), (7, 8, 2), (65, 32, 4), (33, 33, 8), (100, 128, 8), (64, 256, 8), (9, 257, 32),
                                               (20, 500, 6), (12, 1000, 31), (6, 1024, 32)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_without_bias(ops, rows, experts, topk, scoring, renormalize):
    check(ops, make(rows, experts, 1), topk, scoring, renormalize=renormalize, scale=1.0 if renormalize else 2.5)


@pytest.mark.parametrize("rows,experts,topk,groups,topk_groups", [(5, 8, 2, 1, 1), (200, 256, 8, 8, 4), (50, 256, 8, 1, 1), (40, 160, 6, 8, 3),
                                                                  (30, 64, 6, 32, 16), (9, 1024, 16, 16, 5), (17, 48, 4, 3, 2), (8, 6, 2, 6, 2),
                                                                  (11, 500, 8, 10, 1)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [True, False])
def test_groups_and_bias(ops, rows, experts, topk, groups, topk_groups, scoring, biased):
    bias = torch.randn(experts, generator=torch.Generator().manual_seed(7)).mul(0.1).cuda() if biased else None
    check(ops, make(rows, experts, 2), topk, scoring, bias, groups, topk_groups, True, 2.5)


def test_bf16_logits_with_many_ties(ops):
    logits = (make(300, 128, 3) * 4).round().div(4).to(torch.bfloat16)
    check(ops, logits, 8)
    check(ops, logits, 8, "sigmoid", torch.zeros(128, device="cuda"), 4, 2)
    check(ops, torch.zeros((5, 64), device="cuda"), 6)
    check(ops, torch.zeros((5, 64), device="cuda"), 6, "sigmoid", torch.zeros(64, device="cuda"), 8, 3)


def test_keys_closer_than_32_bits_can_order(ops):
    """Scores that differ by less than a float's unit: sigmoid saturates for large logits, and biases cancel differences."""
    g = torch.Generator().manual_seed(4)
    logits = (20 + torch.randn((200, 64), generator=g) * 0.5).cuda()
    check(ops, logits, 8, "sigmoid", torch.randn(64, generator=g).mul(1e-7).cuda())
    check(ops, logits, 8, "sigmoid", torch.randn(64, generator=g).mul(1e-7).cuda(), 8, 4)
    logits = make(200, 64, 5, 1e-6)
    check(ops, logits, 8, "softmax", torch.randn(64, generator=g).mul(1e-9).cuda(), 4, 3)


@pytest.mark.parametrize("spread", [1e-6, 3e-7, 1e-7, 2e-8])
@pytest.mark.parametrize("offset", [0.0, 4.0, -4.0])
def test_keys_around_the_doubt(ops, spread, offset):
    """Keys whose differences are about as large as the error of 32 bits, at several magnitudes of the bias, cancelling ones too."""
    g = torch.Generator().manual_seed(11)
    logits = make(400, 64, 12)
    base = offset * torch.where(torch.arange(64) % 2 == 0, 1.0, -1.0)
    bias = (base.double() - torch.sigmoid(logits[0].cpu().double()) + spread * torch.randn(64, generator=g).double()).float().cuda()
    rows = logits[:1].expand(400, 64) + torch.randn((400, 64), generator=g).cuda() * spread
    check(ops, rows.contiguous(), 8, "sigmoid", bias)
    check(ops, rows.contiguous(), 8, "sigmoid", bias, 8, 4)


def test_rows_of_infinities_and_nan(ops):
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[-inf] * 8, [-inf, 1, -inf, 2, -inf, -inf, -inf, -inf], [nan, 1, 2, 3, 4, 5, nan, 7], [inf, 1, inf, 2, 3, 4, 5, 6],
                           [torch.finfo(torch.float32).min] * 8, [0.0, -0.0, 0.0, -0.0, -0.0, 0.0, 0.0, 0.0]]).cuda()
    w, ids = ops.route_topk(logits, 4)
    assert ids[0].tolist() == [0, 1, 2, 3] and w[0].tolist() == [0, 0, 0, 0]
    assert ids[1].tolist() == [3, 1, 0, 2] and w[1, 2:].tolist() == [0, 0] and abs(float(w[1].sum()) - 1) < 1e-6
    assert ids[2].tolist() == [7, 5, 4, 3] and bool(torch.isfinite(w[2]).all())
    assert ids[3].tolist() == [0, 2, 7, 6] and w[3].tolist() == [0.5, 0.5, 0, 0]
    assert ids[4].tolist() == [0, 1, 2, 3] and w[4].tolist() == [0.25] * 4
    assert ids[5].tolist() == [0, 1, 2, 3] and w[5].tolist() == [0.25] * 4
    w, ids = ops.route_topk(logits, 4, renormalize=False)
    assert w[0].tolist() == [0, 0, 0, 0] and w[4].tolist() == [0.125] * 4
    w, ids = ops.route_topk(logits[:3], 8, "sigmoid", torch.zeros(8, device="cuda"))
    assert ids[0].tolist() == list(range(8)) and w[0].tolist() == [0] * 8
    assert ids[2].tolist() == [7, 5, 4, 3, 2, 1, 0, 6] and bool(torch.isnan(w[2]).all())       # a NaN that had to be chosen
    _, ids = ops.route_topk(logits[:1], 2, "sigmoid", torch.arange(8.0, device="cuda"), 4, 1)
    assert ids[0].tolist() == [7, 6]


def test_strided_and_empty_rows(ops):
    wide = make(50, 100, 6)
    check(ops, wide[:, 3:67], 8)
    check(ops, wide.to(torch.bfloat16)[:, 1:34], 5)
    w, ids = ops.route_topk(wide[:0], 8)
    assert w.shape == ids.shape == (0, 8)


def test_ids_feed_the_plan(ops):
    logits = make(77, 16, 8)
    w, ids = ops.route_topk(logits, 4)
    counts, dest, _, _ = ops.dispatch_plan(ids, 0, 16, 77)
    assert counts.cpu().tolist() == torch.bincount(ids.cpu().flatten().long(), minlength=16).tolist() and bool((dest >= 0).all())


def test_refusals(ops):
    x = make(4, 64, 9)
    for kw, what in ((dict(topk=0), "topk"), (dict(topk=33), "topk"), (dict(topk=9, groups=8, topk_groups=1), "topk"), (dict(topk=2, groups=5), "groups"),
                     (dict(topk=2, groups=4, topk_groups=5), "topk_groups"), (dict(topk=2, scoring="tanh"), "scoring"),
                     (dict(topk=2, bias=torch.zeros(63, device="cuda")), "bias"), (dict(topk=2, bias=torch.zeros(64)), "device"),
                     (dict(topk=2, groups=64, topk_groups=64), "groups")):
        with pytest.raises(RuntimeError, match=what):
            ops.route_topk(x, **kw)
    with pytest.raises(RuntimeError, match="experts"):
        ops.route_topk(make(1, 1025, 1), 2)
    with pytest.raises(RuntimeError, match="float32 or bf16"):
        ops.route_topk(x.double(), 2)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        ops.route_topk(x.t(), 2)
