"""A mixture-of-experts block as it is used: norm, router, plan, routed experts, combine, shared expert added on top, the next
norm.  Every step is held to its 64-bit form on the inputs that the device gave it; the whole is captured and replayed."""
import pytest
import torch

import dense_reference as ref
from test_gpu_norm import F32, check_codes

pytestmark = pytest.mark.gpu

EXPERTS, HIDDEN, INTER, TOPK, SHARED = 16, 512, 256, 4, 384


@pytest.fixture(scope="module")
def block():
    import paired_nvfp4_kernels as pnk
    return Block(torch.ops.paired_nvfp4, pnk)


class Block:
    def __init__(self, ops, pnk):
        self.ops = ops
        g = torch.Generator(device="cuda").manual_seed(0)

        def w(n, k):
            return (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).to(torch.bfloat16)

        from paired_nvfp4_kernels import reference

        def experts(n, k):
            dense = torch.randn((EXPERTS, n, k), generator=g, device="cuda") * k ** -0.5
            codes, scales, _ = reference.quantize_weight(reference.prune_paired_4of8(dense))
            return ops.compress(codes, scales, k)

        self.norm = 1 + 0.1 * torch.randn(HIDDEN, generator=g, device="cuda")
        self.router, self.bias = w(EXPERTS, HIDDEN), 0.05 * torch.randn(EXPERTS, generator=g, device="cuda")
        self.w13, self.w2 = experts(2 * INTER, HIDDEN), experts(HIDDEN, INTER)
        self.shared13 = w(2 * SHARED, HIDDEN)[pnk.interleave_gate_up_rows(SHARED, "cuda")].contiguous()
        self.shared2 = w(HIDDEN, SHARED)
        self.q13, self.q2 = ops.quant_mx8(self.shared13), ops.quant_mx8(self.shared2)
        self.g1 = torch.full((EXPERTS,), 6 * 448 / 16.0, device="cuda")
        self.g2 = torch.full((EXPERTS,), 6 * 448 / 16.0, device="cuda")

    def __call__(self, x, residual):
        """All intermediate results of one pass, by name."""
        ops, cap = self.ops, x.size(0)
        y, res, q, sf = ops.add_rms_norm(x, residual, self.norm, 1e-6, True, True)
        logits = ops.linear(y, self.router, float_out=True)
        weights, ids = ops.route_topk(logits, TOPK, "sigmoid", self.bias, 4, 2, True, 2.5)
        counts, dest, src_tok, src_route = ops.dispatch_plan(ids, 0, EXPERTS, cap)
        b, sfb = ops.scatter_quant_act_planned(y, src_tok, src_route, None, self.g1, counts, cap)
        h, sfh = ops.group_mm_swiglu_quant(*self.w13, b, sfb, 1 / self.g1, counts, self.g2, 2 * INTER, HIDDEN, 0, 2, 1)
        expert_out = torch.zeros((EXPERTS, cap, HIDDEN), dtype=torch.bfloat16, device="cuda")
        ops.group_mm(expert_out, *self.w2, h, sfh, 1 / self.g2, counts, HIDDEN, INTER)
        routed = torch.empty_like(x)
        ops.moe_finalize(routed, expert_out, dest, weights)
        mid = ops.linear_mx8(q, sf, *self.q13, activation="silu", gated=True)
        out = ops.linear_mx8(*ops.quant_mx8(mid), *self.q2, residual=routed)
        y2, res2, _, _ = ops.add_rms_norm(out, res, self.norm)
        return dict(y=y, res=res, q=q, sf=sf, logits=logits, weights=weights, ids=ids, counts=counts, expert_out=expert_out, dest=dest,
                    routed=routed, mid=mid, out=out, y2=y2, res2=res2)


def make(tokens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple((torch.randn((tokens, HIDDEN), generator=g, device="cuda") * s).to(torch.bfloat16) for s in (1.0, 3.0))


@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_every_step_against_its_formula(block, tokens):
    x, residual = make(tokens, tokens)
    r = block(x, residual)
    v, n = ref.norm(x.cpu(), residual.cpu(), block.norm.cpu(), 1e-6)
    assert bool(((r["y"].cpu().double() - n).abs() <= n.abs() * (ref.BF16 + 2 * F32)).all())
    check_codes(r["q"], r["sf"], n, tokens, HIDDEN)
    want, bound = ref.linear(r["y"], block.router, None, None, "none", False, chunk=512, out_eps=2.0 ** -24)
    assert bool(((r["logits"].double() - want).abs() <= bound).all())
    want_w, want_ids = ref.route(r["logits"], TOPK, "sigmoid", block.bias.cpu(), 4, 2, True, 2.5)
    assert torch.equal(r["ids"].cpu(), want_ids)
    assert bool(((r["weights"].cpu().double() - want_w).abs() <= want_w * 48 * 2.0 ** -24).all())
    assert r["counts"].cpu().tolist() == torch.bincount(want_ids.flatten().long(), minlength=EXPERTS).tolist()
    # the combine: bf16 weights and products as moe_finalize defines them, half a unit each, and its own rounding
    rows = r["expert_out"].view(-1, HIDDEN)[r["dest"].long()].double()
    w = r["weights"].to(torch.bfloat16).double().unsqueeze(-1)
    want = (rows * w).sum(1)
    bound = (rows * w).abs().sum(1) * (ref.BF16 + 2.0 ** -22) + want.abs() * ref.BF16
    assert bool(((r["routed"].double() - want).abs() <= bound + 1e-30).all())

    def values(pair, rows, k):
        return ref.decode(pair[0], ref.scale_rows(pair[1], rows, k)[:rows, :k // 32]).cuda()

    want, bound = ref.linear(values((r["q"], r["sf"]), tokens, HIDDEN), values(block.q13, 2 * SHARED, HIDDEN), None, None, "silu", True, k_step=32)
    assert bool(((r["mid"].double() - want).abs() <= bound).all())
    mid = block.ops.quant_mx8(r["mid"])
    want, bound = ref.linear(values(mid, tokens, SHARED), values(block.q2, HIDDEN, SHARED), None, r["routed"], "none", False, k_step=32)
    assert bool(((r["out"].double() - want).abs() <= bound).all())
    v, n = ref.norm(r["out"].cpu(), r["res"].cpu(), block.norm.cpu(), 1e-6)
    assert bool(((r["y2"].cpu().double() - n).abs() <= n.abs() * (ref.BF16 + 2 * F32)).all())
    assert torch.equal(r["res2"].cpu(), v.float().to(torch.bfloat16))


def same(a, b):
    return all(torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)) for k in a)


@pytest.mark.parametrize("tokens", [1, 64, 301])
def test_captured_and_replayed(block, tokens):
    """Two graphs of the block and eager passes between their replays, each on inputs of its own."""
    a, b = make(tokens, 1), make(tokens, 2)
    want_a, want_b = block(*a), block(*b)
    held, graphs, got = [tuple(t.clone() for t in a), tuple(t.clone() for t in a)], [], []
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(block(*h))
        graphs.append(graph)
    for src, dst in zip(b, held[1]):
        dst.copy_(src)
    for _ in range(3):
        graphs[0].replay()
        eager = block(*b)
        graphs[1].replay()
    torch.cuda.synchronize()
    assert same(got[0], want_a) and same(got[1], want_b) and same(eager, want_b)


def test_on_two_streams_at_once(block):
    inputs = [make(90, 3), make(90, 4)]
    want = [block(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for k in range(12):
        with torch.cuda.stream(streams[k % 2]):
            got.append(block(*inputs[k % 2]))
    torch.cuda.synchronize()
    assert all(same(g, want[k % 2]) for k, g in enumerate(got))


def test_padded_batch(block):
    """Rows of padding change nothing in the rows of tokens."""
    x, residual = make(50, 5)
    padded = [torch.cat([t, torch.zeros((14, HIDDEN), dtype=t.dtype, device="cuda")]) for t in (x, residual)]
    r, p = block(x, residual), block(*padded)
    for k in ("y", "res", "q", "logits", "weights", "ids", "mid", "res2"):
        assert torch.equal(r[k].view(torch.uint8), p[k][:50].view(torch.uint8)), k
