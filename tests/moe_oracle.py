"""The expert layer from its formulas in 64 bits, on the CPU."""
import torch

import row_oracle


def unpack(w, bits, axis):
    """Codes along ``axis`` as float64."""
    if bits == 8:
        return w.double()
    wide = w.to(torch.int16)
    both = torch.stack((wide & 15, wide >> 4), axis + 1).flatten(axis, axis + 1)
    return torch.where(both > 7, both - 16, both).double()


def route(x, router, top_k, renormalize=True):
    logits = x.double() @ router.double().t()
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids, best = order.indices[:, :top_k], order.values[:, :top_k]
    share = torch.exp(best - best[:, :1])
    total = share.sum(-1, keepdim=True) if renormalize else torch.exp(logits - best[:, :1]).sum(-1, keepdim=True)
    return ids, share / total


def _product(codes, scales, w, w_scale, sub):
    """[R, K] codes x [K, N] codes, scaled."""
    if not sub:
        return (codes.double() @ w) * scales[:, None] * w_scale.double()[None, :]
    out = torch.zeros(codes.shape[0], w.shape[1], dtype=torch.float64)
    for s in range(w_scale.shape[0]):
        part = codes[:, s * sub:(s + 1) * sub].double() @ w[s * sub:(s + 1) * sub]
        out += part * scales[:, s:s + 1] * w_scale[s].double()[None, :]
    return out


def layer(x, w_up_gate, w_down, s_up_gate, s_down, ids, share, *, bits, nn, sub):
    """(out, sum of the sizes of the terms): float64 [T, H]."""
    codes, scales, _ = row_oracle.quantize_rows(x, bits, sub)
    out, size = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    inner = w_up_gate.shape[2 if nn else 1] // 2
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if not 0 <= e < w_up_gate.shape[0]:
                continue
            up_gate = unpack(w_up_gate[e], bits, 0) if nn else unpack(w_up_gate[e], bits, 1).t()
            down = unpack(w_down[e], bits, 0) if nn else unpack(w_down[e], bits, 1).t()
            both = _product(codes[t:t + 1], scales[t:t + 1], up_gate, s_up_gate[e], sub)
            up, gate = both[:, :inner], both[:, inner:]
            act = up * gate / (1 + torch.exp(-gate))
            a, sa, _ = row_oracle.quantize_rows(act, bits, sub)
            y = _product(a, sa, down, s_down[e], sub)[0] * share[t, j].double()
            out[t] += y
            size[t] += y.abs()
    return out, size
