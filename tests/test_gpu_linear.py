"""linear and linear_mx8 against products in 64 bits, within the bound that dense_reference.linear derives."""
import pytest
import torch

import dense_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from paired_nvfp4_kernels import ops as module
    yield torch.ops.paired_nvfp4
    assert module.linear_device_status() == 0            # no bounded wait gave up


def rows(n, k, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, k), generator=g, device="cuda") * scale
    x[:, ::61] *= 8
    return x.to(torch.bfloat16)


def check(out, want, bound):
    off = (out.double() - want).abs()
    assert out.shape == want.shape and bool((off <= bound).all()), (float((off / bound).max()), (off > bound).nonzero()[:4].tolist())


def run(ops, t, n, k, mx8=False, bias=None, residual=False, activation="none", gated=False, float_out=False, beta=1.0, linear_beta=-1.0, seed=0):
    x, w = rows(t, k, seed), rows(n, k, seed + 1, k ** -0.5)
    n_out = n // 2 if gated else n
    b = None if bias is None else torch.randn(n, generator=torch.Generator().manual_seed(seed + 2)).to(bias).cuda()
    r = rows(t, n_out, seed + 3) if residual else None
    more = dict(activation=activation, gated=gated, beta=beta, linear_beta=linear_beta)
    if mx8:
        q, sf = ops.quant_mx8(x)
        wq, wsf = ops.quant_mx8(w)
        out = ops.linear_mx8(q, sf, wq, wsf, b, r, **more)
        x = ref.decode(q, ref.scale_rows(sf, t, k)[:t, :k // 32]).cuda()
        w = ref.decode(wq, ref.scale_rows(wsf, n, k)[:n, :k // 32]).cuda()
    else:
        out = ops.linear(x, w, b, r, float_out=float_out, **more)
    assert out.dtype == (torch.float32 if float_out else torch.bfloat16)
    want, bound = ref.linear(x, w, b, r, activation, gated, beta, linear_beta, 32 if mx8 else 16, 512 if float_out else None,
                             2.0 ** -24 if float_out else ref.BF16)
    check(out, want, bound)


# tokens: each tile width and both sides of its border; K: one instruction, less, more than one stage, no multiple of a stage;
# features: one, odd, around a tile, several
@pytest.mark.parametrize("t", [1, 2, 16, 17, 32, 33, 64, 65, 128, 129])
@pytest.mark.parametrize("n,k", [(1, 8), (7, 64), (128, 16), (129, 200), (256, 1024), (320, 72), (1000, 2880)])
def test_small_and_odd_sizes(ops, t, n, k):
    run(ops, t, n, k, seed=t * n + k)
    run(ops, t, n, k, float_out=True, seed=t * n + k + 1)


@pytest.mark.parametrize("t", [1, 15, 31, 64, 100, 128, 200])
@pytest.mark.parametrize("n,k", [(1, 32), (7, 64), (128, 96), (130, 160), (256, 1024), (384, 4128)])
def test_small_and_odd_sizes_mx8(ops, t, n, k):
    run(ops, t, n, k, mx8=True, seed=t * n + k)


# the pair kernel: tokens and features around its 256 x 256 tiles, K of one stage, odd stages, more than the ring
@pytest.mark.parametrize("t,n,k", [(3000, 2048, 64), (2049, 2304, 72), (2500, 2571, 512), (4000, 2000, 1000), (2200, 4096, 2880), (8192, 1031, 256),
                                   (257, 20000, 512), (5000, 2560, 104)])
@pytest.mark.parametrize("mx8", [False, True])
def test_large_sizes(ops, t, n, k, mx8):
    run(ops, t, n, k // 32 * 32 if mx8 else k, mx8=mx8, bias=torch.bfloat16, residual=True, seed=n)


# a K long enough for clusters of two, four and eight CTAs to share it, and one that leaves some a stage less
@pytest.mark.parametrize("t,n,k", [(1, 128, 256), (1, 256, 7168), (3, 2048, 7168), (16, 4096, 4096), (20, 6144, 1096), (64, 8192, 4168), (100, 1024, 14336),
                                   (128, 256, 520), (128, 2048, 2056), (700, 256, 7168)])
@pytest.mark.parametrize("mx8", [False, True])
def test_shared_k(ops, t, n, k, mx8):
    k = k // 32 * 32 if mx8 else k
    run(ops, t, n, k, mx8=mx8, bias=torch.float32, seed=k)
    if not mx8:
        run(ops, t, n, k, float_out=True, seed=k)


@pytest.mark.parametrize("t", [1, 33, 100, 3000])
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float32])
def test_activations(ops, t, activation, bias):
    n = 2304 if t == 3000 else 200
    run(ops, t, n, 320, activation=activation, bias=bias, seed=5)
    run(ops, t, n, 320, activation=activation, bias=bias, residual=True, mx8=True, seed=6)
    run(ops, t, n, 320, activation=activation, bias=bias, residual=True, float_out=True, seed=7)


@pytest.mark.parametrize("t", [1, 40, 128, 2600])
@pytest.mark.parametrize("n", [64, 192, 2304, 2368])
@pytest.mark.parametrize("activation,beta,linear_beta", [("silu", 1.0, -1.0), ("situ", 1.702, 1.0), ("situ", 0.5, -1.0)])
def test_gated(ops, t, n, activation, beta, linear_beta):
    more = dict(activation=activation, gated=True, beta=beta, linear_beta=linear_beta)
    run(ops, t, n, 640, seed=8, **more)
    run(ops, t, n, 640, mx8=True, bias=torch.bfloat16, seed=9, **more)
    run(ops, t, n, 640, bias=torch.float32, residual=True, seed=10, **more)
    run(ops, t, n, 640, float_out=True, seed=11, **more)


def test_gated_layout_is_that_of_the_grouped_gemm(ops):
    """Rows in the order of interleave_gate_up_rows: the gated product equals the ungated one followed by gated_act."""
    from paired_nvfp4_kernels import interleave_gate_up_rows
    x, w = rows(70, 256, 12), rows(2 * 192, 256, 13, 0.0625)
    got = ops.linear(x, w[interleave_gate_up_rows(192, "cuda")], activation="silu", gated=True)
    plain = ops.linear(x, w, float_out=True).double()
    want = torch.nn.functional.silu(plain[:, :192]) * plain[:, 192:]
    assert bool(((got.double() - want).abs() <= want.abs() * (ref.BF16 + 1e-5) + 1e-6).all())


def test_strided_operands(ops):
    x, r = rows(300, 640, 14), rows(300, 401, 15)
    w = rows(200, 512, 16, 0.05)
    for view in (x[:, 64:64 + 512], x[::2, 8:520]):
        t = view.size(0)
        res = r[:t, 1:201]
        assert torch.equal(ops.linear(view, w, None, res), ops.linear(view.contiguous(), w, None, res.contiguous()))


def test_infinities_and_nan_stay_in_their_row(ops):
    x, w = rows(300, 256, 17), rows(300, 256, 18, 0.06)
    want = ops.linear(x, w)
    bad = x.clone()
    bad[7, 3], bad[290, 255] = float("nan"), float("inf")
    got = ops.linear(bad, w)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[7, 290]] = False
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[7]).all()) and not bool(torch.isfinite(got[290]).any())
    q, sf = ops.quant_mx8(bad)
    wq, wsf = ops.quant_mx8(w)
    q0, sf0 = ops.quant_mx8(x)
    got, want = ops.linear_mx8(q, sf, wq, wsf), ops.linear_mx8(q0, sf0, wq, wsf)
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[7]).all()) and bool(torch.isnan(got[290]).all())
    relu = ops.linear(bad, w, activation="relu")
    assert bool(torch.isnan(relu[7]).all())


@pytest.mark.parametrize("t,k", [(5, 160), (130, 96), (2600, 2144)])
def test_scales_in_the_slop_do_not_matter(ops, t, k):
    n = 2368 if t > 2000 else 200
    x, w = rows(t, k, 19), rows(n, k, 20, 0.1)
    (q, sf), (wq, wsf) = ops.quant_mx8(x), ops.quant_mx8(w)
    want = ops.linear_mx8(q, sf, wq, wsf)
    dirty = [ref.scale_buffer(ref.scale_rows(s, m, k)[:m, :k // 32], m, k).cuda() for s, m in ((sf, t), (wsf, n))]
    got = ops.linear_mx8(q.view(torch.uint8), dirty[0], wq.view(torch.uint8), dirty[1])       # 1-byte types are taken as they are
    assert torch.equal(got, want)


@pytest.mark.parametrize("t,n", [(5, 200), (130, 64), (2600, 2368)])
@pytest.mark.parametrize("float_out", [0, 1])
@pytest.mark.parametrize("gated", [0, 1])
def test_nothing_is_written_outside_the_output(ops, t, n, float_out, gated):
    from paired_nvfp4_kernels import _cabi
    n = n // 64 * 64 if gated else n - 1
    x, w, size = rows(t, 128, 21), rows(n, 128, 22), t * (n // 2 if gated else n)
    buf = torch.full((size + 512,), 7.0, dtype=torch.float32 if float_out else torch.bfloat16, device="cuda")
    rc = _cabi.lib.pnv_linear(buf[256:].data_ptr(), float_out, x.data_ptr(), 128, w.data_ptr(), None, 0, None, 0, t, n, 128, 0 if gated else 2, gated,
                              1.0, -1.0, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    want = ops.linear(x, w, float_out=bool(float_out), gated=bool(gated), activation="silu" if gated else "none")
    assert torch.equal(buf[256:256 + size].view(want.shape), want) and bool((buf[:256] == 7).all()) and bool((buf[256 + size:] == 7).all())


def test_output_and_bias_at_odd_elements(ops):
    """What vector accesses cannot take goes element by element."""
    from paired_nvfp4_kernels import _cabi
    for t, n in ((9, 256), (2600, 2304)):
        x, w, b = rows(t, 128, 23), rows(n, 128, 24), rows(1, n + 1, 25)[0]
        want = ops.linear(x, w, b[1:].clone())
        assert torch.equal(ops.linear(x, w, b[1:]), want)
        buf = torch.zeros(t * n + 1, dtype=torch.bfloat16, device="cuda")
        rc = _cabi.lib.pnv_linear(buf[1:].data_ptr(), 0, x.data_ptr(), 128, w.data_ptr(), b[1:].data_ptr(), 0, None, 0, t, n, 128, 2, 0, 1.0, -1.0, 0,
                                  torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(buf[1:].view(t, n), want)


def test_no_rows(ops):
    w = rows(64, 64, 26)
    assert ops.linear(w[:0], w).shape == (0, 64)
    q, sf = ops.quant_mx8(w)
    assert ops.linear_mx8(q[:0], sf[:0], q, sf, gated=True, activation="silu").shape == (0, 32)


@pytest.mark.parametrize("t,n,k", [(1, 256, 7168), (64, 4096, 2048), (3000, 2304, 512)])
def test_same_bits_every_time_and_in_a_graph(ops, t, n, k):
    """Partial sums are added in a fixed order; a captured call replays on new contents of its inputs; two streams at once."""
    x, w = rows(t, k, 27), rows(n, k, 28, 0.02)
    want = ops.linear(x, w)
    q, sf = ops.quant_mx8(x)
    wq, wsf = ops.quant_mx8(w)
    want8 = ops.linear_mx8(q, sf, wq, wsf)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append((ops.linear(x, w), ops.linear_mx8(q, sf, wq, wsf)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, want8) for a, b in got)
    other = rows(t, k, 29)
    want = ops.linear(other, w)
    x0, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear(x0, w)
        y8 = ops.linear_mx8(*ops.quant_mx8(x0), wq, wsf)
    x0.copy_(other)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(y8, ops.linear_mx8(*ops.quant_mx8(other), wq, wsf))


def test_refusals(ops):
    x, w = rows(4, 64, 30), rows(128, 64, 31)
    q, sf = ops.quant_mx8(x)
    wq, wsf = ops.quant_mx8(w)
    for call, what in ((lambda: ops.linear(x, w[:, :56]), "contiguous"), (lambda: ops.linear(x, w[:, :32].contiguous()), "share K"),
                       (lambda: ops.linear(x[:, :60], w[:, :60].contiguous()), "multiple of 8"), (lambda: ops.linear(x.float(), w), "bf16"),
                       (lambda: ops.linear(x, w, activation="tanh"), "activation"), (lambda: ops.linear(x, w, activation="relu", gated=True), "activation"),
                       (lambda: ops.linear(x, w[:96], activation="silu", gated=True), "multiple of 64"),
                       (lambda: ops.linear(x, w, activation="situ", gated=True, beta=0.0), "beta"),
                       (lambda: ops.linear(x, w, torch.zeros(127, device="cuda")), "bias"), (lambda: ops.linear(x, w, torch.zeros(128)), "device"),
                       (lambda: ops.linear(x, w, None, x), "residual"), (lambda: ops.linear(x, w.cpu()), "device"),
                       (lambda: ops.linear(rows(4, 68, 1)[:, :64], w), "16 bytes"), (lambda: ops.linear(rows(4, 72, 1)[:, 4:68], w), "aligned"),
                       (lambda: ops.linear_mx8(q, sf[:256], wq, wsf), "q_sf is smaller"), (lambda: ops.linear_mx8(q, sf, wq, wsf[:256]), "weight_sf is smaller"),
                       (lambda: ops.linear_mx8(x, sf, wq, wsf), "e4m3"), (lambda: ops.linear_mx8(q, sf.float(), wq, wsf), "e8m0"),
                       (lambda: ops.linear_mx8(q[:, :32], sf, wq, wsf), "contiguous")):
        with pytest.raises(RuntimeError, match=what):
            call()
