"""add_rms_norm and quant_mx8 against their 64-bit forms."""
import pytest
import torch

import dense_reference as ref
from dense_reference import BF16

pytestmark = pytest.mark.gpu

# 32 bits ahead of the rounding: at most 90 additions in a row of squares (2^-24 each, halved by the root), root, quotient and
# products 2^-23 each
F32 = 45 * 2.0 ** -24 + 5 * 2.0 ** -23


@pytest.fixture(scope="module")
def ops():
    import paired_nvfp4_kernels  # noqa: F401
    return torch.ops.paired_nvfp4


def make(rows, width, seed, scale=1.0, pad=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, width + pad), generator=g) * scale).to(torch.bfloat16).cuda()
    return x[:, offset:offset + width]


def check_codes(q, sf, n, rows, width):
    """8-bit outputs against n (float64): slop, scales (an amax within the 32-bit error of a border may go either way), codes
    off by half a step of four significant bits or of the subnormal numbers."""
    all_sf = ref.scale_rows(sf, rows, width)
    assert sf.numel() == all_sf.numel()
    assert bool((all_sf[rows:] == ref.SLOP).all()) and bool((all_sf[:, width // 32:] == ref.SLOP).all())
    got = all_sf[:rows, :width // 32]
    low, high = ref.block_scales(n * (1 - F32)), ref.block_scales(n * (1 + F32))
    assert bool(((got == low) | (got == high)).all())
    scale = torch.ldexp(torch.ones(got.shape, dtype=torch.float64), got.int() - 127).repeat_interleave(32, 1)
    off = (ref.decode(q, got) - n).abs()
    assert bool((off <= n.abs() * (2.0 ** -4 + 2 * F32) + scale * 2.0 ** -10).all())


# widths: one element, odd, just past a vector, the repository's hidden sizes, the largest; rows around atoms of 128
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 33), (5, 264), (129, 1023), (64, 2048), (31, 2880), (300, 2880), (1, 7168),
                                        (2, 4096), (700, 4104), (130, 7168), (3, 16384), (400, 5120), (1, 32768), (301, 32768),
                                        (300, 4097), (9, 8191), (33, 2881), (5, 32761), (3, 32767), (40, 12), (2000, 1), (700, 9)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight_type", [torch.bfloat16, torch.float32])
def test_norm_matches_64_bits(ops, rows, width, residual, weight_type):
    x = make(rows, width, 1)
    r = make(rows, width, 2, 3.0) if residual else None
    w = (1 + 0.3 * torch.randn(width, generator=torch.Generator().manual_seed(3))).to(weight_type).cuda()
    mx8 = width % 32 == 0
    y, res, q, sf = ops.add_rms_norm(x, r, w, 1e-6, True, mx8)
    v, n = ref.norm(x.cpu(), r.cpu() if residual else None, w.cpu(), 1e-6)
    assert y.shape == x.shape and y.dtype == torch.bfloat16
    assert bool(((y.cpu().double() - n).abs() <= n.abs() * (BF16 + 2 * F32) + 1e-38).all())
    if residual:
        assert torch.equal(res.cpu(), (x.cpu().float() + r.cpu().float()).to(torch.bfloat16))
    else:
        assert res is None
    if mx8:
        check_codes(q, sf, n, rows, width)
        only, _, q2, sf2 = ops.add_rms_norm(x, r, w, 1e-6, False, True)
        assert only is None and torch.equal(q2.view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(sf2.view(torch.uint8), sf.view(torch.uint8))
    else:
        assert q is None and sf is None


# slices of wider rows at element offsets that 16-byte accesses cannot take, and at ones they can
@pytest.mark.parametrize("pad,offset", [(8, 8), (3, 1), (64, 32), (5, 4)])
@pytest.mark.parametrize("rows,width", [(5, 64), (200, 2880), (1, 96)])
def test_strided_rows(ops, rows, width, pad, offset):
    x, r = make(rows, width, 4, 1.0, pad, offset), make(rows, width, 5, 1.0, pad + 2, offset)
    w = make(1, width, 6)[0].contiguous()
    got = ops.add_rms_norm(x, r, w, 1e-5, True, True)
    want = ops.add_rms_norm(x.contiguous(), r.contiguous(), w, 1e-5, True, True)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# odd widths whose rows lie alike within 16 bytes in every buffer, and ones where they do not
@pytest.mark.parametrize("pad,offset", [(8, 8), (64, 16), (1, 0), (8, 3)])
@pytest.mark.parametrize("rows,width", [(5, 63), (200, 2881), (1, 97), (300, 4094)])
@pytest.mark.parametrize("weight_type", [torch.bfloat16, torch.float32])
def test_strided_rows_of_odd_widths(ops, rows, width, pad, offset, weight_type):
    x, r = make(rows, width, 4, 1.0, pad + offset, offset), make(rows, width, 5, 1.0, pad + offset + 8, offset)
    w = make(1, width, 6)[0].to(weight_type).contiguous()
    got = ops.add_rms_norm(x, r, w, 1e-5)
    want = ops.add_rms_norm(x.contiguous(), r.contiguous(), w, 1e-5)
    v, n = ref.norm(x.cpu(), r.cpu(), w.cpu(), 1e-5)
    for t in (got, want):
        assert bool(((t[0].cpu().double() - n).abs() <= n.abs() * (BF16 + 2 * F32) + 1e-38).all())
        assert torch.equal(t[1].cpu(), v.float().to(torch.bfloat16))


def test_nothing_is_written_outside_of_odd_rows(ops):
    """C entry on pieces of larger buffers: rows of 4097 elements, outputs with a guard on either side."""
    from paired_nvfp4_kernels import _cabi
    rows, width = 37, 4097
    x, w = make(rows, width, 7).contiguous(), make(1, width, 8)[0].contiguous()
    for lead in (8, 3):
        bufs = [torch.full((rows * width + 64,), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        y, res = (b[lead:lead + rows * width].view(rows, width) for b in bufs)
        rc = _cabi.lib.pnv_add_rms_norm(x.data_ptr(), width, x.data_ptr(), width, w.data_ptr(), 0, 1e-6, rows, width, y.data_ptr(), res.data_ptr(),
                                        None, None, 0, torch.cuda.current_stream().cuda_stream)
        want = ops.add_rms_norm(x, x, w)
        off = (y.double() - want[0].double()).abs()            # (another grouping of the sum: a unit at most)
        assert rc == 0 and bool((off <= want[0].double().abs() * 2 * BF16).all()) and torch.equal(res, want[1])
        assert all(bool((b[:lead] == 7).all()) and bool((b[lead + rows * width:] == 7).all()) for b in bufs)


def test_weight_at_an_odd_element(ops):
    x, w = make(4, 256, 7), make(1, 257, 8)[0]
    got = ops.add_rms_norm(x, x, w[1:], 1e-6, True, True)
    want = ops.add_rms_norm(x, x, w[1:].clone(), 1e-6, True, True)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_zero_rows_infinities_and_nan(ops):
    x = make(6, 256, 9)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 70] = float("nan")
    x[4] = torch.finfo(torch.bfloat16).max
    w = torch.ones(256, device="cuda")
    y, _, q, sf = ops.add_rms_norm(x, None, w, 1e-6, True, True)
    y, q, sf = y.cpu().float(), q.view(torch.uint8).cpu(), ref.scale_rows(sf, 6, 256)[:6, :8]
    assert bool((y[1] == 0).all()) and bool((q[1] & 0x7F == 0).all()) and bool((sf[1] == ref.SLOP).all())
    # an infinity: 1 / sqrt(inf) = 0, so zeros and 0 * inf
    assert bool(torch.isnan(y[2, 5])) and bool((y[2, :5] == 0).all()) and sf[2, 0] == 0xFF and bool((sf[2, 1:] == ref.SLOP).all())
    assert bool((q[2, :32] == 0x7F).all())
    assert bool(torch.isnan(y[3]).all()) and bool((sf[3] == 0xFF).all()) and bool((q[3] == 0x7F).all())
    assert bool((y[4] == 0).all())                       # the squares overflow 32 bits, as in the formula in 32 bits
    for row in (0, 5):
        assert bool(torch.isfinite(y[row]).all())
    y0, _, _, _ = ops.add_rms_norm(torch.zeros_like(x), None, w, 0.0)
    assert bool(torch.isnan(y0).all())                   # 0 / 0 without eps


def test_no_rows(ops):
    w = torch.ones(64, device="cuda")
    x = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    y, r, q, sf = ops.add_rms_norm(x, x, w, 1e-6, True, True)
    assert y.shape == r.shape == q.shape == (0, 64) and sf.numel() == 0
    q, sf = ops.quant_mx8(x)
    assert q.shape == (0, 64) and sf.numel() == 0


@pytest.mark.parametrize("rows,k", [(1, 32), (1, 7168), (3, 96), (127, 128), (128, 160), (129, 2880), (1000, 2048), (257, 14336), (40, 4128)])
def test_quantizer_finds_the_nearest_codes(ops, rows, k):
    g = torch.Generator().manual_seed(rows + k)
    x = torch.randn((rows, k), generator=g) * torch.exp(8 * torch.randn((rows, 1), generator=g))
    x = x.to(torch.bfloat16)
    x.view(-1)[::37] = 0
    q, sf = ops.quant_mx8(x.cuda())
    code, want = ref.encode(x.double())
    all_sf = ref.scale_rows(sf, rows, k)
    assert torch.equal(all_sf[:rows, :k // 32], want)
    assert bool((all_sf[rows:] == ref.SLOP).all()) and bool((all_sf[:, k // 32:] == ref.SLOP).all())
    assert torch.equal(q.view(torch.uint8).cpu(), code)


def test_quantizer_on_every_bf16_magnitude(ops):
    """Every finite bf16 number as the largest of its block, with borders of the scale's choice among them."""
    bits = torch.arange(0x7F80, dtype=torch.int32).to(torch.int16)
    x = torch.zeros((0x7F80, 32), dtype=torch.bfloat16)
    x[:, 3] = bits.view(torch.bfloat16)
    x[:, 4] = -x[:, 3] * 0.37
    q, sf = ops.quant_mx8(x.cuda())
    code, want = ref.encode(x.double())
    assert torch.equal(ref.scale_rows(sf, 0x7F80, 32)[:0x7F80, :1], want)
    got = q.view(torch.uint8).cpu()
    assert torch.equal(torch.where(got == 0x80, 0, got), torch.where(code == 0x80, 0, code))


def test_quantizer_marks_blocks_that_are_not_finite(ops):
    x = make(2, 128, 11).clone()
    x[0, 40], x[1, 127] = float("nan"), float("-inf")
    q, sf = ops.quant_mx8(x)
    sf, q = ref.scale_rows(sf, 2, 128)[:2, :4], q.view(torch.uint8).cpu()
    assert (sf == 0xFF).tolist() == [[False, True, False, False], [False, False, False, True]]
    assert bool((q[0, 32:64] == 0x7F).all()) and bool((q[1, 96:] == 0x7F).all()) and bool((q[0, :32] & 0x7F != 0x7F).all())


def test_quantizer_takes_strided_rows(ops):
    wide = make(70, 512, 12)
    for x in (wide[:, 8:8 + 256], wide[:, 16:16 + 96], wide[::2, :64]):
        for a, b in zip(ops.quant_mx8(x), ops.quant_mx8(x.contiguous())):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals(ops):
    x, w = make(4, 64, 13), torch.ones(64, device="cuda")
    with pytest.raises(RuntimeError, match="at least one"):
        ops.add_rms_norm(x, None, w, 1e-6, False, False)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        ops.add_rms_norm(x[:, :40], None, w[:40], 1e-6, True, True)
    with pytest.raises(RuntimeError, match="shaped like x"):
        ops.add_rms_norm(x, x[:3], w)
    with pytest.raises(RuntimeError, match="weight"):
        ops.add_rms_norm(x, None, w[:63])
    with pytest.raises(RuntimeError, match="contiguous rows"):
        ops.add_rms_norm(x.t(), None, torch.ones(4, device="cuda"))
    with pytest.raises(RuntimeError, match="bf16"):
        ops.add_rms_norm(x.float(), None, w)
    with pytest.raises(RuntimeError, match="eps"):
        ops.add_rms_norm(x, None, w, -1.0)
    with pytest.raises(RuntimeError, match="must be on the device"):
        ops.add_rms_norm(x, x.cpu(), w)
    with pytest.raises(RuntimeError, match="hidden must be"):
        ops.add_rms_norm(make(1, 32769, 1), None, torch.ones(32769, device="cuda"))
    with pytest.raises(RuntimeError, match="multiple of 32"):
        ops.quant_mx8(x[:, :48])
    with pytest.raises(RuntimeError, match="16 bytes"):
        ops.quant_mx8(make(4, 66, 14)[:, :64])
    with pytest.raises(RuntimeError, match="aligned"):
        ops.quant_mx8(make(1, 72, 14)[:, 4:68])
