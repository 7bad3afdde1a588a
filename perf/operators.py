"""The operators either side of the grouped GEMM in a mixture-of-experts block, as cases that can be timed and compared:

  norm    add_rms_norm: the residual's addition and the root-mean-square norm, as bf16 and as 8-bit codes with block scales
  quant   quant_mx8: rows to 8-bit codes with block scales (activations between two products, weights at load time)
  linear  linear: dense product with bias, activation (gated ones included) and residual; "mx8" operands: linear_mx8
  route   route_topk: router logits to the top-k expert ids and weights that dispatch_plan and moe_finalize take

`own` chooses between the plain form (elementary torch operations) and the calls of torch.ops.paired_nvfp4.

The 8-bit format: e4m3 codes; one power-of-two scale (e8m0 byte, 2^(byte - 127)) per 32 elements, the smallest that leaves
the block's largest magnitude at 448 or below; scales in the package's scale layout (512-byte atoms of 128 rows x 4 blocks).
8-bit outputs are returned as float8_e4m3fn codes and float8_e8m0fnu scales.
"""
import math
import os
import sys

import torch

own = False

_RANDOM_WIDTHS = (2048, 2880, 4096, 5120, 7168)      # hidden sizes that this repository's workloads have


def _norm(tokens, hidden, residual=True, bf16=True, mx8=False, weight="bf16", strided=False):
    return dict(kind="norm", tokens=tokens, hidden=hidden, residual=residual, bf16=bf16, mx8=mx8, weight=weight, strided=strided)


def _quant(tokens, hidden):
    return dict(kind="quant", tokens=tokens, hidden=hidden)


def _linear(tokens, features, hidden, mx8=False, bias=False, residual=False, activation="none", gated=False,
            float_out=False, strided=False):
    return dict(kind="linear", tokens=tokens, features=features, hidden=hidden, mx8=mx8, bias=bias, residual=residual,
                activation=activation, gated=gated, float_out=float_out, strided=strided)


def _route(tokens, experts, topk, scoring="softmax", bias=False, groups=1, topk_groups=1, renormalize=True, scale=1.0,
           logits="float32"):
    return dict(kind="route", tokens=tokens, experts=experts, topk=topk, scoring=scoring, bias=bias, groups=groups,
                topk_groups=topk_groups, renormalize=renormalize, scale=scale, logits=logits)


def listed():
    return [
        # the norm ahead of an MoE block in one user's decode step: latency; bf16 for the router, codes for the shared expert
        dict(_norm(1, 7168, mx8=True), name="norm_one_token"),
        # the same for a short prompt of a model whose width is no power of two, float32 norm weights, bf16 alone
        dict(_norm(777, 2880, weight="float32"), name="norm_odd"),
        # prefill: memory traffic; both outputs
        dict(_norm(16384, 7168, mx8=True), name="norm_prefill"),
        # activations of a decode batch on their way into an 8-bit product
        dict(_quant(128, 2048), name="quant_decode"),
        # activations of a long prefill between the two products of a wide dense block
        dict(_quant(8192, 14336), name="quant_prefill"),
        # router logits of a small decode batch, in float32
        dict(_linear(16, 256, 7168, float_out=True), name="router_decode"),
        # an output projection with bias and residual on an odd number of tokens, width no power of two
        dict(_linear(777, 2880, 2880, bias=True, residual=True), name="linear_odd"),
        # gate and up projection of a dense block over a prefill, SiLU and the product in the epilogue
        dict(_linear(8192, 28672, 4096, activation="silu", gated=True), name="gated_prefill"),
        # the shared expert's gate and up projection of a decode batch, 8-bit operands: the weights' bytes
        dict(_linear(64, 4096, 7168, mx8=True, activation="silu", gated=True), name="shared_decode"),
        # the shared expert's down projection over a prefill, 8-bit operands, added to the routed experts' output
        dict(_linear(8192, 7168, 2048, mx8=True, residual=True), name="shared_prefill"),
        # routing of a decode batch: sigmoid scores, selection bias, groups of experts
        dict(_route(64, 256, 8, "sigmoid", True, 8, 4, True, 2.5), name="route_decode"),
        # routing of a prefill over 128 experts, softmax
        dict(_route(16384, 128, 8), name="route_prefill"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quant", "linear", "linear", "linear", "linear", "route", "route"])
    tokens = _log_int(rng, 1, 16384)
    if kind == "norm":
        mx8 = rng.random() < 0.5
        hidden = rng.choice([rng.choice(_RANDOM_WIDTHS), 32 * _log_int(rng, 4, 256), _log_int(rng, 64, 8192) if not mx8 else 32 * rng.randint(60, 250)])
        return _norm(tokens, hidden, rng.random() < 0.8, not mx8 or rng.random() < 0.5, mx8, rng.choice(["bf16", "bf16", "float32"]),
                     rng.random() < 0.25)
    if kind == "quant":
        return _quant(_log_int(rng, 1, 8192), 32 * _log_int(rng, 4, 448))
    if kind == "route":
        experts = rng.choice([8, 16, 32, 64, 128, 256, 256, rng.randint(3, 500)])
        topk = rng.randint(1, min(8, experts))
        if rng.random() < 0.5:
            return _route(tokens, experts, topk, "softmax", False, 1, 1, rng.random() < 0.7, 1.0, rng.choice(["float32", "bf16"]))
        fit = [g for g in (1, 2, 4, 8) if experts % g == 0 and experts // g >= topk and experts // g >= 2]
        groups = rng.choice(fit or [1])
        return _route(tokens, experts, topk, "sigmoid", rng.random() < 0.7, groups, rng.randint(1, groups), rng.random() < 0.8,
                      rng.choice([1.0, 2.5]))
    mx8 = rng.random() < 0.5
    gated = rng.random() < 0.4
    hidden = rng.choice([rng.choice(_RANDOM_WIDTHS), 32 * _log_int(rng, 2, 448), 8 * _log_int(rng, 8, 1792) if not mx8 else 32 * rng.randint(16, 300)])
    features = 128 * _log_int(rng, 1, 224) if gated else rng.choice([8 * _log_int(rng, 1, 2000), _log_int(rng, 1, 16384), rng.choice((128, 256))])
    tokens = _log_int(rng, 1, max(16, min(16384, int(1.9e12 / (2.0 * features * hidden)))))
    float_out = not gated and not mx8 and rng.random() < 0.4
    if float_out:
        features = min(features, 1024)               # router logits
    activation = rng.choice(["silu", "silu", "situ"]) if gated else rng.choice(["none", "none", "relu", "silu", "gelu"])
    return _linear(tokens, features, hidden, mx8, rng.random() < 0.4, rng.random() < 0.4, activation, gated, float_out,
                   not mx8 and rng.random() < 0.25)


# ------------------------------------------------------------------------------------------------ inputs

SITU = (1.702, 1.0)    # beta and linear_beta of the SiTU activation, as the workloads of this repository use it
EPS = 1e-6


def _atoms(rows, k):
    return -(-rows // 128), -(-k // 128)


def _scale_layout(sf, k):
    """Scale bytes [rows, k / 32] in the order of the package's scale buffers: atoms of 128 rows x 4 blocks, 512 bytes,
    blocks innermost; what no block owns holds 1.0."""
    rows, kb = sf.shape
    rt, kt = _atoms(rows, k)
    full = torch.full((rt * 128, kt * 4), 127, dtype=torch.uint8, device=sf.device)
    full[:rows, :kb] = sf
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _scale_rows(buf, rows, k):
    """The inverse of _scale_layout: [rows, k / 32]."""
    rt, kt = _atoms(rows, k)
    return buf.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :k // 32]


def _scale_bytes(v):
    """The scale byte of every 32 elements of v (float32 [rows, k]), from the exponent and mantissa of the largest
    magnitude: the smallest power of two that brings it to 448 = 1.75 * 2^8 or below."""
    amax = v.view(v.size(0), -1, 32).abs().amax(-1)
    m, e = torch.frexp(amax)                         # amax = m 2^e, m in [0.5, 1)
    byte = (e - 9 + (m > 0.875).int() + 127).clamp(0, 254)
    return torch.where(amax > 0, byte, torch.full_like(byte, 127)).to(torch.uint8)


def _encode(v):
    """Codes and scale buffer of v (float32 [rows, k])."""
    sf = _scale_bytes(v)
    scaled = torch.ldexp(v.view(v.size(0), -1, 32), (127 - sf.int()).unsqueeze(-1))
    return scaled.to(torch.float8_e4m3fn).view(v.shape), _scale_layout(sf, v.size(1)).view(torch.float8_e8m0fnu)


def _decode(q, buf):
    """float32 values of codes [rows, k] with their scale buffer."""
    rows, k = q.shape
    sf = _scale_rows(buf.view(torch.uint8), rows, k)
    return torch.ldexp(q.float().view(rows, -1, 32), (sf.int() - 127).unsqueeze(-1)).view(rows, k)


def _rows(g, tokens, width, strided, scale=1.0):
    """bf16 activations with a few large channels, as hidden states have; a view of wider rows where strided."""
    wide = width + (64 if strided else 0)
    x = torch.randn((tokens, wide), generator=g, device="cuda") * scale
    x[:, ::61] *= 8.0
    x = x.to(torch.bfloat16)
    return x[:, 32:32 + width] if strided else x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    t = case["tokens"]
    if own:                                          # (the inputs are the same either way: this registers the operators)
        path = os.path.abspath("grouped-sparse-gemm_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import paired_nvfp4_kernels  # noqa: F401
    if case["kind"] == "norm":
        h = case["hidden"]
        s["x"] = _rows(g, t, h, case["strided"])
        s["residual"] = _rows(g, t, h, case["strided"], 3.0) if case["residual"] else None
        w = 1.0 + 0.2 * torch.randn((h,), generator=g, device="cuda")
        s["weight"] = w if case["weight"] == "float32" else w.to(torch.bfloat16)
    elif case["kind"] == "quant":
        s["x"] = _rows(g, t, case["hidden"], False)
    elif case["kind"] == "linear":
        n, k = case["features"], case["hidden"]
        x = _rows(g, t, k, case["strided"])
        w = (torch.randn((n, k), generator=g, device="cuda") * k ** -0.5).to(torch.bfloat16)
        if case["mx8"]:
            s["x"], s["x_sf"] = _encode(x.float())
            s["w"], s["w_sf"] = _encode(w.float())
        else:
            s["x"], s["w"] = x, w
        s["bias"] = torch.randn((n,), generator=g, device="cuda").to(torch.bfloat16) if case["bias"] else None
        n_out = n // 2 if case["gated"] else n
        s["residual"] = _rows(g, t, n_out, False) if case["residual"] else None
    else:
        logits = 1.5 * torch.randn((t, case["experts"]), generator=g, device="cuda")
        s["logits"] = logits if case["logits"] == "float32" else logits.to(torch.bfloat16)
        s["bias"] = 0.1 * torch.randn((case["experts"],), generator=g, device="cuda") if case["bias"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass

def _rounded(v, float_out):
    return v if float_out else v.to(torch.bfloat16)


def _norm_plain(s, c):
    v = s["x"].float()
    if c["residual"]:
        v = v + s["residual"].float()
    n = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    q, sf = _encode(n) if c["mx8"] else (None, None)
    return n.to(torch.bfloat16) if c["bf16"] else None, v.to(torch.bfloat16) if c["residual"] else None, q, sf


def _situ(g, u):
    beta, linear_beta = SITU
    return 0.5 * beta * torch.tanh(g / beta) * (1 + torch.tanh(g / 2)) * linear_beta * torch.tanh(u / linear_beta)


def _activate(v, c):
    """Activation of the product v [tokens, features]; gated: features interleaved in blocks of 32 gates and 32 ups."""
    if c["gated"]:
        g, u = v.view(v.size(0), -1, 2, 32).unbind(2)
        y = g * torch.sigmoid(g) * u if c["activation"] == "silu" else _situ(g, u)
        return y.reshape(v.size(0), -1)
    if c["activation"] == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if c["activation"] == "silu":
        return v * torch.sigmoid(v)
    if c["activation"] == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _linear_plain(s, c):
    x, w = (_decode(s["x"], s["x_sf"]), _decode(s["w"], s["w_sf"])) if c["mx8"] else (s["x"].float(), s["w"].float())
    v = x @ w.T
    if c["bias"]:
        v = v + s["bias"].float()
    v = _activate(v, c)
    if c["residual"]:
        v = v + s["residual"].float()
    return _rounded(v, c["float_out"])


def _select(keys, rank, c):
    """Ids of the top-k experts of each row, best first, ties to the lower index.  keys rank the experts; rank scores the
    groups where there are several (the sum of a group's two best with a bias, its best without)."""
    t, e = keys.shape
    if c["groups"] > 1:
        best = rank.view(t, c["groups"], -1).sort(dim=-1, descending=True).values
        score = best[..., 0] + best[..., 1] if c["bias"] else best[..., 0]
        order = score.sort(dim=-1, descending=True, stable=True).indices[:, :c["topk_groups"]]
        keep = torch.zeros_like(score, dtype=torch.bool).scatter_(1, order, True)
        keys = keys.masked_fill(~keep.repeat_interleave(e // c["groups"], 1), -math.inf)
    return keys.sort(dim=-1, descending=True, stable=True).indices[:, :c["topk"]]


def _route_plain(s, c):
    logits = s["logits"].double()                    # 64 bits: the order of nearly equal scores decides the ids
    if c["scoring"] == "softmax":
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        scores = p / p.sum(-1, keepdim=True)
    else:
        scores = 1.0 / (1.0 + torch.exp(-logits))
    keys = scores + s["bias"].double() if c["bias"] else logits
    ids = _select(keys, keys, c)
    w = scores.gather(1, ids)
    if c["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    return (w * c["scale"]).float(), ids.to(torch.int32)


def run(s):
    c = s["case"]
    if c["kind"] == "norm":
        if own:
            y, r, q, sf = torch.ops.paired_nvfp4.add_rms_norm(s["x"], s["residual"], s["weight"], EPS, c["bf16"], c["mx8"])
            return y if c["bf16"] else None, r if c["residual"] else None, q if c["mx8"] else None, sf if c["mx8"] else None
        return _norm_plain(s, c)
    if c["kind"] == "quant":
        return torch.ops.paired_nvfp4.quant_mx8(s["x"]) if own else _encode(s["x"].float())
    if c["kind"] == "linear":
        if not own:
            return _linear_plain(s, c)
        more = dict(activation=c["activation"], gated=c["gated"])
        if c["activation"] == "situ":
            more.update(beta=SITU[0], linear_beta=SITU[1])
        if c["mx8"]:
            return torch.ops.paired_nvfp4.linear_mx8(s["x"], s["x_sf"], s["w"], s["w_sf"], s["bias"], s["residual"], **more)
        return torch.ops.paired_nvfp4.linear(s["x"], s["w"], s["bias"], s["residual"], float_out=c["float_out"], **more)
    if own:
        return torch.ops.paired_nvfp4.route_topk(s["logits"], c["topk"], c["scoring"], s["bias"], c["groups"], c["topk_groups"],
                                                 c["renormalize"], c["scale"])
    return _route_plain(s, c)


# ------------------------------------------------------------------------------------------------ in 64 bits

def _exact_mx8(v):
    """Codes and scales of v (float64 [rows, k]) as the values they stand for, in 64 bits, scales in the buffer's order."""
    rows, k = v.shape
    blocks = v.view(rows, k // 32, 32)
    amax = blocks.abs().amax(-1)

    def power(e):                                    # exact, where pow() may be off by its rounding
        return torch.ldexp(torch.ones_like(e), e.int())

    e = torch.ceil(torch.log2(amax / 448.0)).clamp(min=-1000)
    e = e + (amax > 448.0 * power(e)).double()
    e = (e - (amax <= 224.0 * power(e)).double()).clamp(min=-127)              # (the logarithm may be off by its rounding)
    scale = torch.where(amax > 0, power(e), torch.ones_like(amax))
    scaled = blocks / scale.unsqueeze(-1)
    step = torch.ldexp(torch.ones_like(scaled), (torch.frexp(scaled).exponent - 4).clamp(min=-9))   # four significant bits
    codes = torch.round(scaled / step) * step
    buf = torch.ones((-(-rows // 128) * 128, -(-k // 128) * 4), dtype=torch.float64, device=v.device)
    buf[:rows, :k // 32] = scale
    buf = torch.cat([band.view(4, 32, -1, 4).permute(2, 1, 0, 3).reshape(-1) for band in buf.split(128)])
    return codes.view(rows, k), buf


def exact(case, seed):
    s, f64 = prepare(case, seed), torch.float64
    kind = case["kind"]
    if kind == "quant":
        return _exact_mx8(s["x"].to(f64))
    if kind == "norm":
        v = s["x"].to(f64) + (s["residual"].to(f64) if case["residual"] else 0.0)
        rms = torch.sqrt((v * v).sum(-1, keepdim=True) / v.size(1) + EPS)
        n = v / rms * s["weight"].to(f64)
        q, sf = _exact_mx8(n) if case["mx8"] else (None, None)
        return n if case["bf16"] else None, v if case["residual"] else None, q, sf
    if kind == "linear":
        if case["mx8"]:
            def values(q, buf):
                rows, k = q.shape
                sf = buf.view(torch.uint8).view(-1, -(-k // 128), 32, 4, 4).transpose(2, 3).transpose(1, 2).transpose(2, 3)
                sf = sf.reshape(-1, -(-k // 128) * 4)[:rows, :k // 32].to(f64)     # [band, quarter, row, atom, block]
                return q.to(f64) * (2.0 ** (sf - 127)).repeat_interleave(32, 1)
            x, w = values(s["x"], s["x_sf"]), values(s["w"], s["w_sf"])
        else:
            x, w = s["x"].to(f64), s["w"].to(f64)
        v = torch.matmul(x, w.t())
        if case["bias"]:
            v += s["bias"].to(f64)
        act = case["activation"]
        if case["gated"]:
            pairs = v.unflatten(1, (-1, 64))
            g, u = pairs[..., :32], pairs[..., 32:]
            if act == "situ":
                b, l = SITU
                y = b / (1 + torch.exp(-g)) * torch.tanh(g / b) * (l * torch.tanh(u / l))
            else:
                y = g / (1 + torch.exp(-g)) * u
            v = y.flatten(1)
        elif act == "relu":
            v = v.clamp(min=0)
        elif act == "silu":
            v = v / (1 + torch.exp(-v))
        elif act == "gelu":
            v = v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
        return v + s["residual"].to(f64) if case["residual"] else v
    # routing: the weights of the experts that the definition picks; ids are whole numbers and have to be equal anyway
    z = s["logits"].to(f64)
    p = torch.softmax(z, -1) if case["scoring"] == "softmax" else torch.sigmoid(z)
    key = p + s["bias"].to(f64) if case["bias"] else z
    if case["groups"] > 1:
        top = key.unflatten(1, (case["groups"], -1)).topk(2, -1).values
        top = top.sum(-1) if case["bias"] else top[..., 0]
        cut = top.topk(case["topk_groups"], -1).values[:, -1:]
        key = key.masked_fill((top < cut).repeat_interleave(z.size(1) // case["groups"], 1), -math.inf)
    ids = torch.argsort(key, dim=-1, descending=True, stable=True)[:, :case["topk"]]
    w = torch.gather(p, 1, ids)
    if case["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    return w * case["scale"], ids.to(torch.int32)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    t, kind = case["tokens"], case["kind"]
    if kind == "norm":
        h = case["hidden"]
        per = 2 + (4 if case["residual"] else 0) + (2 if case["bf16"] else 0) + (1 + 1 / 32 if case["mx8"] else 0)
        return dict(bytes=t * h * per + h * (4 if case["weight"] == "float32" else 2), flops=6 * t * h)
    if kind == "quant":
        return dict(bytes=t * case["hidden"] * (2 + 1 + 1 / 32), flops=3 * t * case["hidden"])
    if kind == "linear":
        n, k = case["features"], case["hidden"]
        n_out = n // 2 if case["gated"] else n
        per = 1 + 1 / 32 if case["mx8"] else 2
        out = t * n_out * ((4 if case["float_out"] else 2) + (2 if case["residual"] else 0))
        return dict(bytes=(t + n) * k * per + out + (2 * n if case["bias"] else 0), flops=2.0 * t * n * k)
    e = case["experts"]
    return dict(bytes=t * e * (4 if case["logits"] == "float32" else 2) + t * case["topk"] * 8 + (4 * e if case["bias"] else 0),
                flops=t * e * 4)
