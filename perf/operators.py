"""What is measured of the operators around the quantised products: layer norm (forward, backward, and fused with
the quantiser), the quantiser for each token, and a whole mixture-of-experts layer for a few tokens.

``run`` computes an operator in its plain form (elementary torch operations) or, where ``own`` is true, through the
package's entry points.  ``exact`` states the same from the definitions in 64 bits.
"""
import functools
import math

import torch

own = False

TOP_CODE = {"int4": 7, "int8": 127}
EPS = 1e-5


def listed():
    return [
        # a few decoded tokens on their way into a 4-bit projection: latency
        {"name": "norm_int4_decode", "op": "layer_norm_quantize", "rows": 8, "cols": 2048, "dtype": "int4", "sub": 0},
        # the input of a SwiGLU up-projection with a scale for each 256 values
        {"name": "norm_int4_sc256", "op": "layer_norm_quantize", "rows": 4096, "cols": 4096, "dtype": "int4", "sub": 256},
        # the norm of a training step over 32768 tokens, and a ragged float32 one
        {"name": "norm_train", "op": "layer_norm", "rows": 32768, "cols": 2048, "dtype": "bf16"},
        {"name": "norm_odd_f32", "op": "layer_norm", "rows": 1001, "cols": 1407, "dtype": "f32"},
        # their backward passes: many rows of a model's width, few rows of a feed-forward's width
        {"name": "norm_bwd_train", "op": "layer_norm_bwd", "rows": 32768, "cols": 2048, "dtype": "bf16"},
        {"name": "norm_bwd_wide_f32", "op": "layer_norm_bwd", "rows": 517, "cols": 14336, "dtype": "f32"},
        # the operand of a grouped product of 32768 tokens, and an odd batch in 8 bits
        {"name": "tokens_int4", "op": "quantize_tokens", "rows": 32768, "cols": 2048, "dtype": "int4", "sub": 0},
        {"name": "tokens_int8_odd", "op": "quantize_tokens", "rows": 129, "cols": 1405, "dtype": "int8", "sub": 0},
        # experts at decoding: one token; a small batch; 8-bit experts; a full batch over few large experts
        {"name": "moe_one_token", "op": "moe", "tokens": 1, "experts": 64, "top_k": 8, "hidden": 2048, "inner": 1408,
         "dtype": "int4", "sub": 0, "layout": "nt"},
        {"name": "moe_batch_sc128", "op": "moe", "tokens": 13, "experts": 64, "top_k": 6, "hidden": 2048, "inner": 1408,
         "dtype": "int4", "sub": 128, "layout": "nn"},
        {"name": "moe_int8", "op": "moe", "tokens": 5, "experts": 16, "top_k": 2, "hidden": 1024, "inner": 2816,
         "dtype": "int8", "sub": 0, "layout": "nt"},
        {"name": "moe_full_batch", "op": "moe", "tokens": 64, "experts": 8, "top_k": 2, "hidden": 4096, "inner": 14336,
         "dtype": "int4", "sub": 0, "layout": "nn"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["layer_norm_quantize", "layer_norm", "layer_norm_bwd", "quantize_tokens", "moe", "moe"])
    if op == "moe":
        tokens, experts = _log(rng, 1, 64), _log(rng, 4, 128)
        hidden = 32 * _log(rng, 8, 128)
        most = (8 * 4096 * 14336) // (experts * hidden)
        inner = 32 * _log(rng, 4, max(5, min(448, most // 32)))
        dtype = rng.choice(["int4", "int4", "int8"])
        if dtype == "int8":
            inner = max(32, inner // 64 * 32)
        return {"op": op, "tokens": tokens, "experts": experts, "top_k": rng.randint(1, min(8, experts)), "hidden": hidden,
                "inner": inner, "dtype": dtype, "sub": rng.choice([0, 0, 32, 64, 128, 256]), "layout": rng.choice(["nt", "nn"])}
    rows = _log(rng, 1, 32768)
    cols = _log(rng, 64, min(16384, 32768 * 2048 // rows))
    if rng.random() < 0.7:
        cols = (cols + 7) // 8 * 8
    case = {"op": op, "rows": rows, "cols": cols}
    if op in ("layer_norm", "layer_norm_bwd"):
        case["dtype"] = rng.choice(["bf16", "f32"])
        if case["dtype"] == "f32":
            case["rows"] = max(1, rows // 2)
    else:
        case["dtype"] = rng.choice(["int4", "int8"])
        case["sub"] = rng.choice([0, 32, 64, 128, 256])
    return case


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _activations(rows, cols, g):
    """A residual stream: every token has its own offset and size, a few channels are far larger than the others."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    channel = 1.0 + 7.0 * (torch.rand(cols, device="cuda", generator=g) < 0.01)
    token = 0.5 + torch.rand(rows, 1, device="cuda", generator=g)
    return x * channel * token + 0.2 * torch.randn(rows, 1, device="cuda", generator=g)


def _codes(shape, dtype, g):
    if dtype == "int4":  # two codes of -8..7 a byte
        return torch.randint(0, 256, shape, device="cuda", dtype=torch.uint8, generator=g)
    return torch.randint(-127, 128, shape, device="cuda", dtype=torch.int8, generator=g)


def _weight_scales(shape, fan_in, dtype, g):
    spread = 4.6 if dtype == "int4" else 73.5  # of the codes: the weights get a variance of about 1 / fan_in
    return ((0.5 + torch.rand(shape, device="cuda", generator=g)) / (spread * fan_in ** 0.5)).to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "moe":
        t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inner"]
        kb = 2 if case["dtype"] == "int4" else 1
        s["x"] = _activations(t, h, g).to(torch.bfloat16)
        s["router"] = (torch.randn(e, h, device="cuda", generator=g) / h ** 0.5).to(torch.bfloat16)
        up, down = ((e, h // kb, 2 * i), (e, i // kb, h)) if case["layout"] == "nn" else ((e, 2 * i, h // kb), (e, h, i // kb))
        s["w_up_gate"], s["w_down"] = _codes(up, case["dtype"], g), _codes(down, case["dtype"], g)
        sub = case["sub"]
        s["up_gate_scale"] = _weight_scales((e, -(-h // sub), 2 * i) if sub else (e, 2 * i), h, case["dtype"], g)
        s["down_scale"] = _weight_scales((e, -(-i // sub), h) if sub else (e, h), i, case["dtype"], g)
        return s
    rows, cols = case["rows"], case["cols"]
    kind = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    s["x"] = _activations(rows, cols, g).to(kind)
    if case["op"] != "quantize_tokens":
        s["weight"] = (1.0 + 0.1 * torch.randn(cols, device="cuda", generator=g)).to(kind)
        s["bias"] = (0.1 * torch.randn(cols, device="cuda", generator=g)).to(kind)
    if case["op"] == "layer_norm_bwd":  # what the forward pass left
        x = s["x"].float()
        mean = x.mean(-1)
        s["mean"], s["rstd"] = mean, torch.rsqrt((x - mean[:, None]).square().mean(-1) + EPS)
        s["dy"] = (torch.randn(rows, cols, device="cuda", generator=g) / rows).to(kind)
    return s


# ---------------------------------------------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _package():
    import strix_halo_int4_gemms_b200 as pkg

    return pkg


@functools.lru_cache(maxsize=None)
def _spec(sub):
    pkg = _package()
    return pkg.ScaleSpec(pkg.ScaleMode.SUBCHANNEL, sub) if sub else pkg.ScaleSpec(pkg.ScaleMode.PER_CHANNEL)


def _values(pkg, s, codes):
    """Codes of 4 bits as the whole numbers they stand for, through the package's own unpacking."""
    return codes if s["dtype"] == "int8" else pkg.unpack_int4_on_device(codes)[:, : s["cols"]]


def _run_own(s):
    pkg = _package()
    op = s["op"]
    if op == "layer_norm":
        y, mean, rstd = pkg.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "layer_norm_bwd":
        dx, dweight, dbias = pkg.layer_norm_bwd(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
        return {"dx": dx, "dweight": dweight, "dbias": dbias}
    dtype = pkg.OperandDType.INT4 if s["dtype"] == "int4" else pkg.OperandDType.INT8
    if op == "layer_norm_quantize":
        codes, scales = pkg.layer_norm_quantize(s["x"], s["weight"], s["bias"], eps=EPS, dtype=dtype, scale=_spec(s["sub"]))
        return {"codes": _values(pkg, s, codes), "scales": scales}
    if op == "quantize_tokens":
        codes, scales = pkg.quantize_tokens(s["x"], dtype=dtype, scale=_spec(s["sub"]))
        return {"codes": _values(pkg, s, codes), "scales": scales}
    return {"out": pkg.moe_swiglu(
        s["x"], s["w_up_gate"], s["w_down"], up_gate_scale=s["up_gate_scale"], down_scale=s["down_scale"],
        router_weight=s["router"], top_k=s["top_k"], dtype=dtype,
        layout=pkg.GemmLayout.NN if s["layout"] == "nn" else pkg.GemmLayout.NT, scale=_spec(s["sub"]))}


# ---------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------
def _round_bf16(x):
    """float64 -> bfloat16 with one rounding: to float32 with the last bit set where bits were lost, then to nearest."""
    f = x.to(torch.float32)
    back = f.to(torch.float64)
    bits = f.view(torch.int32) - (back.abs() > x.abs()).to(torch.int32)
    return (bits | (back != x).to(torch.int32)).view(torch.float32).to(torch.bfloat16)


def _quantize(x, dtype, sub):
    """Codes and scales of rows, one scale for a row or for each ``sub`` values: scale = bf16(amax / top code), a zero
    scale counts as one; code = round to even(x / scale).  64 bits, since a quotient may lie next to a border."""
    x = x.to(torch.float64)
    cols = x.shape[-1]
    size = sub or cols
    groups = -(-cols // size)
    blocks = torch.nn.functional.pad(x, (0, groups * size - cols)).unflatten(-1, (groups, size))
    scales = _round_bf16(blocks.abs().amax(-1) / TOP_CODE[dtype])
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    codes = torch.round(blocks / scales[..., None].to(torch.float64)).flatten(-2)[..., :cols]
    return codes.to(torch.int8), scales if sub else scales[..., 0]


def _norm(x, weight, bias):
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    return (x - mean) * rstd * weight + bias, mean[..., 0], rstd[..., 0]


def _unpack(w, dtype, axis, kind):
    """Weight codes along K as numbers of ``kind``."""
    if dtype == "int8":
        return w.to(kind)
    low = ((w & 15) ^ 8).to(torch.int8) - 8
    high = ((w >> 4) ^ 8).to(torch.int8) - 8
    return torch.stack((low, high), axis + 1).flatten(axis, axis + 1).to(kind)


def _scaled_product(codes, scales, w, w_scale, case):
    """[B, T, K] codes with their scales times [B, ...] weight codes with theirs -> [B, T, N] in 64 bits.  The products
    of the codes are exact: 4-bit ones, and groups of up to 256 8-bit ones, stay below 2^24 in 32 bits."""
    nn, sub = case["layout"] == "nn", case["sub"]
    kind = torch.float32 if case["dtype"] == "int4" or sub else torch.float64
    w = _unpack(w, case["dtype"], 1 if nn else 2, kind)
    w = w if nn else w.transpose(1, 2)                      # [B, K, N]
    if not sub:
        return torch.bmm(codes.to(kind), w).to(torch.float64) * scales.to(torch.float64)[..., None] * w_scale.to(torch.float64)[:, None, :]
    k = codes.shape[-1]
    groups = -(-k // sub)
    pad = groups * sub - k
    a = torch.nn.functional.pad(codes.to(kind), (0, pad)).unflatten(-1, (groups, sub)).transpose(1, 2)   # [B, S, T, sub]
    b = torch.nn.functional.pad(w, (0, 0, 0, pad)).unflatten(1, (groups, sub))                            # [B, S, sub, N]
    part = torch.matmul(a, b).to(torch.float64)
    return (part * scales.to(torch.float64).transpose(1, 2)[..., None] * w_scale.to(torch.float64)[:, :, None, :]).sum(1)


def _moe(s):
    x, e, k = s["x"], s["experts"], s["top_k"]
    t = x.shape[0]
    logits = x.to(torch.float64) @ s["router"].to(torch.float64).t()      # 64 bits: two experts may be close
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids, best = order.indices[:, :k], order.values[:, :k]
    share = torch.softmax(best, dim=-1)
    codes, scales = _quantize(x, s["dtype"], s["sub"])
    if t * k <= e:   # the experts of each (token, choice)
        which = ids.flatten()
        pick = lambda w: w[which]  # noqa: E731
        codes, scales = codes.repeat_interleave(k, 0)[:, None], scales.repeat_interleave(k, 0)[:, None]
    else:            # every expert on every token
        pick = lambda w: w  # noqa: E731
        codes, scales = codes.expand(e, *codes.shape), scales.expand(e, *scales.shape)
    both = _scaled_product(codes, scales, pick(s["w_up_gate"]), pick(s["up_gate_scale"]), s)
    up, gate = both.chunk(2, dim=-1)
    act_codes, act_scales = _quantize(up * gate / (1 + torch.exp(-gate)), s["dtype"], s["sub"])
    y = _scaled_product(act_codes, act_scales, pick(s["w_down"]), pick(s["down_scale"]), s).to(torch.float32)
    y = y.view(t, k, -1) if t * k <= e else y[ids, torch.arange(t, device=x.device)[:, None]]
    return (y * share.to(torch.float32)[..., None]).sum(1).to(torch.bfloat16)


def run(state):
    s = state
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "layer_norm":
        y, mean, rstd = _norm(s["x"].float(), s["weight"].float(), s["bias"].float())
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    if op == "layer_norm_bwd":
        dy = s["dy"].float()
        hat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * s["weight"].float()
        dx = s["rstd"][:, None] * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
        return {"dx": dx.to(s["x"].dtype), "dweight": (dy * hat).sum(0), "dbias": dy.sum(0)}
    if op == "layer_norm_quantize":  # 64 bits: a value may lie next to the border of two codes
        codes, scales = _quantize(_norm(s["x"].double(), s["weight"].double(), s["bias"].double())[0], s["dtype"], s["sub"])
        return {"codes": codes, "scales": scales}
    if op == "quantize_tokens":
        codes, scales = _quantize(s["x"], s["dtype"], s["sub"])
        return {"codes": codes, "scales": scales}
    return {"out": _moe(s)}


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "moe":
        t, e, k, h, i = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "inner"))
        used = e * (1 - (1 - k / e) ** t)                 # experts that at least one token goes to, on average
        weights = 3 * h * i * (0.5 if case["dtype"] == "int4" else 1.0)
        scales = 2.0 * (2 * i * (-(-h // case["sub"]) if case["sub"] else 1) + h * (-(-i // case["sub"]) if case["sub"] else 1))
        return {"bytes": used * (weights + scales) + 2.0 * e * h + 4.0 * t * h, "flops": 2.0 * t * (e * h + 3 * k * h * i)}
    n, cols = case["rows"] * case["cols"], case["cols"]
    if case["op"] in ("layer_norm", "layer_norm_bwd"):
        size = 4 if case["dtype"] == "f32" else 2
        if case["op"] == "layer_norm":
            return {"bytes": 2.0 * n * size + 2 * cols * size + 8 * case["rows"], "flops": 8.0 * n}
        return {"bytes": 3.0 * n * size + cols * (size + 8) + 8 * case["rows"], "flops": 14.0 * n}
    scales = 2.0 * case["rows"] * (-(-cols // case["sub"]) if case["sub"] else 1)
    codes = n * (0.5 if case["dtype"] == "int4" else 1.0)
    norm = case["op"] == "layer_norm_quantize"
    return {"bytes": 2.0 * n + codes + scales + (4 * cols if norm else 0), "flops": (11.0 if norm else 3.0) * n}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_bf16(v):
    """The bfloat16 number nearest to each float64, ties to even, as float64."""
    exponent = torch.frexp(v)[1].clamp_min(-125).to(torch.float64)      # |v| in [2^(e-1), 2^e); the least normal is 2^-126
    step = torch.exp2(exponent - 8)
    return torch.round(v / step) * step


def _exact_row_codes(v, top, sub):
    v = v.double()
    parts, scales = [], []
    for at in range(0, v.shape[-1], sub or v.shape[-1]):
        block = v[..., at: at + (sub or v.shape[-1])]
        scale = _exact_bf16(block.abs().max(-1, keepdim=True).values / top)
        scale = torch.where(scale == 0, 1.0, scale)
        parts.append(torch.round(block / scale))
        scales.append(scale)
    return torch.cat(parts, -1), torch.cat(scales, -1)


def _exact_expert(codes, scales, w, w_scale, nn, packed, sub):
    """Rows of codes through one expert's matrix in 64 bits."""
    w = w if nn else w.t()
    if packed:
        wide = w.to(torch.int16)
        signed = torch.stack(((wide & 15), (wide >> 4)), 1)             # [K/2, 2, N]
        w = torch.where(signed > 7, signed - 16, signed).reshape(-1, w.shape[1])
    if not sub:
        return (codes * scales) @ (w.double() * w_scale.double())
    rep = torch.arange(w.shape[0], device=w.device) // sub
    return (codes * scales[:, rep]) @ (w.double() * w_scale.double()[rep])


def exact(case, seed):
    s = prepare(case, seed)
    op, x = s["op"], s["x"].double()
    if op == "moe":
        top, sub, nn = TOP_CODE[s["dtype"]], s["sub"], s["layout"] == "nn"
        logits = (x[:, None, :] * s["router"].double()[None]).sum(-1) if x.shape[0] * s["router"].numel() < 2 ** 27 else x @ s["router"].double().t()
        ids = torch.argsort(-logits, dim=-1, stable=True)[:, : s["top_k"]]
        share = torch.exp(logits.gather(1, ids) - logits.max(-1, keepdim=True).values)
        share = share / share.sum(-1, keepdim=True)
        codes, scales = _exact_row_codes(x, top, sub)
        out = torch.zeros_like(x)
        for e in range(s["experts"]):
            rows, choice = torch.nonzero(ids == e, as_tuple=True)
            if not rows.numel():
                continue
            both = _exact_expert(codes[rows], scales[rows], s["w_up_gate"][e], s["up_gate_scale"][e], nn, s["dtype"] == "int4", sub)
            up, gate = both[:, : s["inner"]], both[:, s["inner"]:]
            a, sa = _exact_row_codes(up * gate * torch.sigmoid(gate), top, sub)
            y = _exact_expert(a, sa, s["w_down"][e], s["down_scale"][e], nn, s["dtype"] == "int4", sub)
            out.index_add_(0, rows, y * share[rows, choice][:, None])
        return {"out": out}
    if op == "quantize_tokens":
        codes, scales = _exact_row_codes(x, TOP_CODE[s["dtype"]], s["sub"])
        return {"codes": codes.to(torch.int8), "scales": scales if s["sub"] else scales[:, 0]}
    w, rows = s["weight"].double(), x.shape[0]
    if op == "layer_norm_bwd":
        dy, r = s["dy"].double(), s["rstd"].double()
        centred = x - s["mean"].double()[:, None]
        a = (dy * w).sum(-1) / x.shape[1]
        c = torch.einsum("rc,rc,c->r", dy, centred, w) / x.shape[1] * r * r
        dx = r[:, None] * (dy * w - a[:, None] - centred * c[:, None])
        return {"dx": dx, "dweight": torch.einsum("rc,rc,r->c", dy, centred, r), "dbias": torch.ones(rows, device=x.device, dtype=x.dtype) @ dy}
    var, mean = torch.var_mean(x, dim=-1, unbiased=False)
    rstd = 1 / torch.sqrt(var + EPS)
    y = torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], w)
    if op == "layer_norm":
        return {"y": y, "mean": mean, "rstd": rstd}
    codes, scales = _exact_row_codes(y, TOP_CODE[s["dtype"]], s["sub"])
    return {"codes": codes.to(torch.int8), "scales": scales if s["sub"] else scales[:, 0]}
