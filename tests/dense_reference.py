"""Plain 64-bit forms of the operators around the grouped GEMM (norm, 8-bit quantizer, dense layers, routing) and the bounds
that their results are held to."""
import math

import torch

BF16 = torch.finfo(torch.bfloat16).eps / 2           # a rounding to bf16 is off by this much, relative
SLOP = 127                                           # scale byte of 1.0


def scale_rows(buf, rows, k):
    """Scale bytes [rows, ceil(k / 128) * 4] of a buffer in the layout of 512-byte atoms of 128 rows x 4 blocks, one by one."""
    buf = buf.view(torch.uint8).cpu()
    n_kt = -(-k // 128)
    r, kb = torch.arange(-(-rows // 128) * 128).view(-1, 1), torch.arange(n_kt * 4).view(1, -1)
    return buf[((r // 128) * n_kt + kb // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + kb % 4]


def scale_buffer(bytes_, rows, k):
    """The inverse: [rows, k / 32] bytes to a buffer whose slop holds 0xFF."""
    n_kt = -(-k // 128)
    buf = torch.full((-(-rows // 128) * n_kt * 512,), 0xFF, dtype=torch.uint8)
    r, kb = torch.arange(rows).view(-1, 1), torch.arange(k // 32).view(1, -1)
    buf[((r // 128) * n_kt + kb // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + kb % 4] = bytes_.cpu()
    return buf


def block_scales(v):
    """Scale bytes [rows, k / 32] of v (float64 [rows, k]), block by block from the definition: the smallest power of two 2^e,
    e >= -127, with amax <= 448 * 2^e."""
    amax = v.view(v.size(0), -1, 32).abs().amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m * 2 <= 1.75, e - 9, e - 8)      # amax = (2 m) 2^(e - 1), 448 = 1.75 * 2^8
    byte = (e.clamp(min=-127) + 127).to(torch.uint8)
    byte = torch.where(amax == 0, torch.full_like(byte, SLOP), byte)
    return torch.where(torch.isfinite(amax), byte, torch.full_like(byte, 0xFF))


def decode(q, sf_bytes):
    """float64 values of codes [rows, k] with scale bytes [rows, k / 32]."""
    v = q.view(torch.float8_e4m3fn).cpu().double()
    scale = torch.ldexp(torch.ones(sf_bytes.shape, dtype=torch.float64), sf_bytes.int() - 127)
    return v * scale.repeat_interleave(32, 1)


def encode(v):
    """Codes and scale bytes of v (float64), each code the nearest of all (ties to the even one), found by search."""
    sf = block_scales(v)
    scaled = v / torch.ldexp(torch.ones(sf.shape, dtype=torch.float64), sf.int() - 127).repeat_interleave(32, 1)
    table = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()        # 0 .. 448, ascending
    mag = scaled.abs()
    hi = torch.searchsorted(table, mag).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    below, above = mag - table[lo], table[hi] - mag
    code = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi).to(torch.uint8)
    return code | ((torch.signbit(scaled)).to(torch.uint8) << 7), sf


def norm(x, residual, weight, eps):
    v = x.double() + (residual.double() if residual is not None else 0)
    return v, v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * weight.double()


def activation(v, kind):
    if kind == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if kind == "silu":
        return v * torch.sigmoid(v)
    if kind == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    return v


def gated(v, kind, beta, linear_beta):
    g, u = v.unflatten(1, (-1, 2, 32)).unbind(2)
    if kind == "silu":
        y = g * torch.sigmoid(g) * u
    else:
        y = beta * torch.tanh(g / beta) * torch.sigmoid(g) * (linear_beta * torch.tanh(u / linear_beta) if linear_beta > 0 else u)
    return y.flatten(1)


def linear(x, w, bias, residual, kind, is_gated, beta=1.0, linear_beta=-1.0, k_step=16, chunk=None, out_eps=BF16):
    """(result, bound) in 64 bits.  The bound: an instruction of k_step products adds to the accumulator with an error of at
    most 2^-22 of the sum of magnitudes seen (it truncates to 24 bits, and its products among each other); `chunk`: the sum
    restarts every so many K and the pieces are added with 2^-24 each.  Then the bias's addition, the activation's slope and
    own error, the residual's addition, each 2^-24 or a few times that; last the rounding of the result."""
    x, w = x.double(), w.double()
    k = x.size(1)
    steps = -(-(chunk or k) // k_step)
    pieces = -(-k // chunk) if chunk else 1
    v, mag = x @ w.T, x.abs() @ w.abs().T
    err = mag * (steps * 2.0 ** -22 + (pieces + 8) * 2.0 ** -24)
    if bias is not None:
        v = v + bias.double()
        err = err + v.abs() * 2.0 ** -24
    if is_gated:
        y = gated(v, kind, beta, linear_beta)
        g, u = v.unflatten(1, (-1, 2, 32)).unbind(2)
        dg, du = err.unflatten(1, (-1, 2, 32)).unbind(2)
        if kind == "silu":
            e = 1.1 * dg * (u.abs() + du) + du * (g.abs() + dg)
        else:
            up = linear_beta if linear_beta > 0 else u.abs() + du
            e = (1 + beta / 4) * dg * up + beta * du
        # exponentials whose argument was rounded: 2^-24 of |g| log2(e), a few units more for reciprocal and products
        e = e.flatten(1) + y.abs() * (8 * 2.0 ** -23 + g.flatten(1).abs() * 2.0 ** -22)
    else:
        y = activation(v, kind)
        e = 1.2 * err + y.abs() * (8 * 2.0 ** -23 + (v.abs() * 2.0 ** -22 if kind == "silu" else 0)) + (v.abs() * 2.0 ** -21 if kind == "gelu" else 0)
    if residual is not None:
        y = y + residual.double()
        e = e + y.abs() * 2.0 ** -24
    return y, e * (1 + out_eps) + y.abs() * out_eps + 1e-37


def route(logits, topk, scoring, bias=None, groups=1, topk_groups=1, renormalize=True, scale=1.0):
    """Expert by expert in 64 bits: Python's stable sort on (key, index)."""
    weights, ids = [], []
    for row in logits.double().cpu():
        if scoring == "softmax":
            mx = max([v for v in row.tolist() if v == v], default=-math.inf)
            p = [0.0 if mx == -math.inf else 1.0 if v == mx else math.exp(v - mx) for v in row.tolist()]
            score = [v / sum(p) if sum(p) else 0.0 for v in p]
        else:
            score = [1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0 for v in row.tolist()]
        key = [s + b for s, b in zip(score, bias.double().tolist())] if bias is not None else row.tolist()
        key = [-math.inf if k != k else k for k in key]
        nan = [v != v for v in row.tolist()]
        n = len(key) // groups
        best = []
        for g in range(groups):
            top = sorted(key[g * n:(g + 1) * n], reverse=True)
            best.append(sum(top[:2]) if bias is not None and n > 1 else top[0])
        keep = set(sorted(range(groups), key=lambda g: (-best[g], g))[:topk_groups])
        order = sorted((e for e in range(len(key)) if e // n in keep), key=lambda e: (-key[e], nan[e], e))[:topk]
        w = [score[e] for e in order]
        if renormalize:
            w = [v / sum(w) if sum(w) else 0.0 for v in w]
        ids.append(order)
        weights.append([v * scale for v in w])
    return torch.tensor(weights, dtype=torch.float64), torch.tensor(ids, dtype=torch.int32)
