"""Plain 64-bit statements of the row operators (quantiser for each token, layer norm and its backward pass), on the
CPU, written from the formulas."""
import torch

TOP = {4: 7.0, 8: 127.0}


def round_bf16(v):
    """float64 -> the nearest bfloat16 number, ties to even, in one rounding."""
    v = v.double()
    exponent = torch.frexp(v)[1].clamp_min(-125).double()
    step = torch.exp2(exponent - 8)
    out = torch.round(v / step) * step
    return torch.where(torch.isfinite(v), out, v)


def quantize_rows(v, bits, sub=0):
    """(codes int8 [R, K], scales float64 [R] or [R, S], distance of each quotient from the nearest border)."""
    v = v.double()
    cols = v.shape[-1]
    codes, scales, border = [], [], []
    for at in range(0, cols, sub or cols):
        block = v[:, at:at + (sub or cols)]
        amax = block.abs().amax(-1, keepdim=True)          # NaN stays NaN
        s = round_bf16(amax / TOP[bits])
        s = torch.where(s == 0, torch.ones_like(s), s)
        q = block / s
        code = torch.where(torch.isfinite(s).expand_as(q), torch.round(q).clamp(-TOP[bits], TOP[bits]), torch.zeros_like(q))
        codes.append(code)
        scales.append(s)
        border.append(((q - torch.floor(q)) - 0.5).abs())
    scales = torch.cat(scales, -1)
    return torch.cat(codes, -1).to(torch.int8), scales if sub else scales[:, 0], torch.cat(border, -1)


def norm(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = (x - mean) * rstd * weight.double()
    return (y if bias is None else y + bias.double()), mean[:, 0], rstd[:, 0]


def norm_bwd(dy, x, weight, mean, rstd):
    dy, x, w = dy.double(), x.double(), weight.double()
    mean, rstd = mean.double()[:, None], rstd.double()[:, None]
    h = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx, (dy * h).sum(0), dy.sum(0)
