"""route_topk on rows that have a NaN and nothing above -infinity: what became of a token must not look like a choice."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def ops():
    import paired_nvfp4_kernels  # noqa: F401
    return torch.ops.paired_nvfp4


def order(row, topk, bias, groups, topk_groups):
    """Ids of a row of -infinity and NaN: without a bias -infinity ranks ahead of NaN, with one every key is a NaN; ties go to
    the lowest index, for groups (ranked by their best) as for experts."""
    last = [bias or v != v for v in row]
    n = len(row) // groups
    keep = sorted(range(groups), key=lambda g: (all(last[g * n:(g + 1) * n]), g))[:topk_groups]
    return sorted((e for e in range(len(row)) if e // n in keep), key=lambda e: (last[e], e))[:topk]


@pytest.mark.parametrize("experts,topk,groups,topk_groups", [(8, 3, 1, 1), (8, 2, 2, 1), (64, 6, 1, 1), (64, 6, 8, 3), (256, 8, 8, 4), (500, 32, 1, 1),
                                                             (500, 7, 10, 2), (1024, 5, 32, 1)])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_softmax_of_a_row_without_a_number(ops, experts, topk, groups, topk_groups, renormalize, biased, dtype):
    nan_at = lambda *at: [NAN if e in at else -INF for e in range(experts)]  # noqa: E731
    broken = [[NAN] * experts, nan_at(0), nan_at(experts - 1), nan_at(*range(1, experts)), nan_at(*range(experts // 2))]
    fine = torch.randn(experts, generator=torch.Generator().manual_seed(experts)).tolist()
    empty = [-INF] * experts
    rows = [fine, *broken, empty, fine]
    logits = torch.tensor(rows).to(dtype).cuda()
    bias = torch.zeros(experts, device="cuda") if biased else None
    w, ids = ops.route_topk(logits, topk, "softmax", bias, groups, topk_groups, renormalize, 2.5)
    for i, row in enumerate(broken, 1):
        assert ids[i].tolist() == order(row, topk, biased, groups, topk_groups), i
        assert bool(torch.isnan(w[i]).all()), (i, w[i])
    assert ids[-2].tolist() == list(range(topk)) and w[-2].tolist() == [0.0] * topk       # nothing but -infinity: no weight
    alone_w, alone_ids = ops.route_topk(logits[:1], topk, "softmax", bias, groups, topk_groups, renormalize, 2.5)
    for i in (0, -1):                                                                      # the rows around them are as they were
        assert torch.equal(w[i], alone_w[0]) and torch.equal(ids[i], alone_ids[0]) and bool(torch.isfinite(w[i]).all())


def test_a_number_beside_a_nan(ops):
    """Where a number is left a NaN ranks last: without a bias the weights of the chosen are those without it (renormalized), all
    scores of the row are NaN otherwise."""
    row = torch.tensor([[NAN, 1.0, -INF, 3.0, 2.0, -INF, NAN, 0.0]]).cuda()
    w, ids = ops.route_topk(row, 3)
    p = [math.exp(v) for v in (3.0, 2.0, 1.0)]
    assert ids[0].tolist() == [3, 4, 1] and max(abs(a - b / sum(p)) for a, b in zip(w[0].tolist(), p)) < 48 * 2.0 ** -24
    for bias, renormalize in ((None, False), (torch.zeros(8, device="cuda"), True), (torch.zeros(8, device="cuda"), False)):
        w, ids = ops.route_topk(row, 3, "softmax", bias, renormalize=renormalize)
        assert bool(torch.isnan(w).all()) and ids[0].tolist() == ([3, 4, 1] if bias is None else [0, 1, 2])


@pytest.mark.parametrize("experts,groups", [(8, 1), (64, 1), (64, 8), (300, 1), (1024, 32)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_a_nan_that_a_bias_does_not_choose(ops, experts, groups, renormalize):
    """With a bias every key of the row is a NaN, so the ids say nothing: no weight may look like one, wherever the NaN is."""
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn((4, experts), generator=g)
    logits[1, experts - 1] = logits[3, 5] = NAN
    bias = torch.randn(experts, generator=g).cuda()
    w, ids = ops.route_topk(logits.cuda(), 3, "softmax", bias, groups, groups, renormalize)
    assert ids[1].tolist() == ids[3].tolist() == [0, 1, 2]
    assert bool(torch.isnan(w[1]).all()) and bool(torch.isnan(w[3]).all())
    for i in (0, 2):
        alone = ops.route_topk(logits[i:i + 1].cuda(), 3, "softmax", bias, groups, groups, renormalize)
        assert torch.equal(w[i], alone[0][0]) and torch.equal(ids[i], alone[1][0]) and bool(torch.isfinite(w[i]).all())
