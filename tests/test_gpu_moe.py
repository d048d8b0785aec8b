"""The expert layer for a few tokens on a B200 against its formulas in 64 bits.

The integer sums, codes and scales are exact on both sides, so the result differs by the roundings at the end alone:
each expert's share is rounded to float32, multiplied with a rounded weight and added up in float32 (at most top_k + 4
roundings of 2^-24 of the sum of the sizes of the shares), and the sum is rounded to bfloat16 (2^-8)."""
import pytest
import torch

import moe_oracle
import row_oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _case(pkg, *, tokens, experts, hidden, inner, bits, layout, sub, seed, router_type=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    nn = layout == "nn"
    per = 2 if bits == 4 else 1
    c = dict(bits=bits, nn=nn, sub=sub)
    c["x"] = (torch.randn(tokens, hidden, generator=g) * (1 + 5 * (torch.rand(hidden, generator=g) < 0.03))).bfloat16()
    c["router"] = (torch.randn(experts, hidden, generator=g) / hidden ** 0.5).to(router_type)

    def codes(k, n):
        shape = (experts, k // per, n) if nn else (experts, n, k // per)
        return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) if bits == 4 else torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)

    def scales(k, n):
        shape = (experts, -(-k // sub), n) if sub else (experts, n)
        return ((torch.rand(shape, generator=g) + 0.5) / ((4.6 if bits == 4 else 74) * k ** 0.5)).bfloat16()

    c["w_up_gate"], c["w_down"] = codes(hidden, 2 * inner), codes(inner, hidden)
    c["s_up_gate"], c["s_down"] = scales(hidden, 2 * inner), scales(inner, hidden)
    c["call"] = dict(up_gate_scale=c["s_up_gate"].cuda(), down_scale=c["s_down"].cuda(), layout=pkg.GemmLayout.NN if nn else pkg.GemmLayout.NT,
                     dtype=pkg.OperandDType.INT4 if bits == 4 else pkg.OperandDType.INT8,
                     scale=pkg.ScaleSpec(pkg.ScaleMode.SUBCHANNEL, sub) if sub else pkg.ScaleSpec(pkg.ScaleMode.PER_CHANNEL))
    c["device"] = (c["x"].cuda(), c["w_up_gate"].cuda(), c["w_down"].cuda())
    return c


def _check(c, got, ids, share):
    want, size = moe_oracle.layer(c["x"], c["w_up_gate"], c["w_down"], c["s_up_gate"], c["s_down"], ids, share,
                                  bits=c["bits"], nn=c["nn"], sub=c["sub"])
    off = (ids.shape[1] + 4) * U * size
    bound = 1.01 * off + 2.0 ** -8 * (want.abs() + off)
    worst = ((got.cpu().double() - want).abs() / bound.clamp_min(1e-300)).max()
    assert worst <= 1, float(worst)


def _routed(pkg, c, top_k, **more):
    out, ids, weights = pkg.moe_swiglu(c["x"].cuda(), *c["device"][1:], router_weight=c["router"].cuda(), top_k=top_k, return_routing=True, **c["call"], **more)
    assert out.dtype == torch.bfloat16 and out.shape == c["x"].shape and ids.dtype == torch.int32 and weights.dtype == torch.float32
    want_ids, want_share = moe_oracle.route(c["x"], c["router"], top_k, more.get("renormalize", True))
    assert torch.equal(ids.cpu().long(), want_ids)
    assert ((weights.cpu().double() - want_share).abs() <= 1.01 * U * want_share + 1e-14).all()
    _check(c, out, want_ids, want_share)
    return out


@pytest.mark.parametrize("sub", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
def test_layer(pkg, bits, layout, sub):
    for tokens, experts, top_k, hidden, inner in ((1, 8, 2, 256, 128), (3, 5, 3, 160, 96), (17, 4, 2, 320, 224), (9, 1, 1, 32, 32), (2, 40, 16, 64, 32)):
        c = _case(pkg, tokens=tokens, experts=experts, hidden=hidden, inner=inner, bits=bits, layout=layout, sub=sub, seed=tokens * 100 + sub + bits)
        _routed(pkg, c, top_k)


@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
def test_model_sizes(pkg, bits, layout):
    c = _case(pkg, tokens=2, experts=6, hidden=2048, inner=1408, bits=bits, layout=layout, sub=0, seed=5)
    _routed(pkg, c, 4)
    c = _case(pkg, tokens=1, experts=3, hidden=1024, inner=2816, bits=bits, layout=layout, sub=256, seed=6, router_type=torch.float32)
    _routed(pkg, c, 2, renormalize=False)


@pytest.mark.parametrize("layout,sub", [("nt", 0), ("nn", 0), ("nt", 64), ("nn", 128)])
def test_all_tokens_on_the_same_experts(pkg, layout, sub):
    """64 rows an expert: several passes over the weights."""
    c = _case(pkg, tokens=64, experts=4, hidden=128, inner=64, bits=4, layout=layout, sub=sub, seed=11)
    c["router"][:] = 0
    c["x"][:, 0] = 3.0
    c["router"][2, 0], c["router"][0, 0] = 2.0, 1.0
    _routed(pkg, c, 2)


def test_ties_go_to_the_lowest_expert(pkg):
    c = _case(pkg, tokens=5, experts=70, hidden=64, inner=32, bits=4, layout="nt", sub=0, seed=12)
    c["router"] = c["router"][:7].repeat(10, 1)          # every logit ten times
    _routed(pkg, c, 11)
    c["router"][:] = 0
    _routed(pkg, c, 3, renormalize=False)


@pytest.mark.parametrize("ids_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("layout", ["nt", "nn"])
def test_given_routing(pkg, layout, ids_type):
    c = _case(pkg, tokens=6, experts=5, hidden=96, inner=64, bits=4, layout=layout, sub=0, seed=13)
    g = torch.Generator().manual_seed(14)
    ids = torch.randint(0, 5, (6, 4), generator=g)       # an expert may be given twice to a token
    ids[1, 2], ids[2, 0], ids[3, :] = -1, 5, -1          # no expert: a hole, out of range, a whole token
    ids[4, :] = 3
    share = torch.rand(6, 4, generator=g) - 0.3
    if ids_type is torch.int64:
        ids[5, 1] = 2 ** 40
    out = pkg.moe_swiglu(*c["device"], topk_ids=ids.to(ids_type).cuda(), topk_weights=share.cuda(), **c["call"])
    _check(c, out, ids, share)
    assert not out[3].any()
    none = pkg.moe_swiglu(*c["device"], topk_ids=torch.full((6, 2), -1, dtype=ids_type).cuda(), topk_weights=share[:, :2].contiguous().cuda(), **c["call"])
    assert not none.any()


@pytest.mark.parametrize("sub", [0, 64])
@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tokens,experts,top_k", [(12, 64, 2), (20, 4, 1), (40, 4, 1), (64, 2, 1), (64, 70, 3)])
def test_more_rows_than_a_pass(pkg, tokens, experts, top_k, bits, layout, sub):
    """Routings that are as uneven as can be: an expert has more rows than a pass over its weights is laid out for."""
    c = _case(pkg, tokens=tokens, experts=experts, hidden=160, inner=96, bits=bits, layout=layout, sub=sub, seed=51)
    g = torch.Generator().manual_seed(52)
    ids = torch.randint(0, experts, (tokens, top_k), generator=g)
    ids[:, 0] = 1
    share = torch.rand(tokens, top_k, generator=g)
    out = pkg.moe_swiglu(*c["device"], topk_ids=ids.cuda(), topk_weights=share.cuda(), **c["call"])
    _check(c, out, ids, share)
    none = pkg.moe_swiglu(*c["device"], topk_ids=torch.full_like(ids, experts).cuda(), topk_weights=share.cuda(), **c["call"])
    assert not none.any()


@pytest.mark.parametrize("layout,sub", [("nt", 0), ("nn", 0), ("nt", 32), ("nn", 128)])
def test_an_expert_given_many_times_to_a_token(pkg, layout, sub):
    c = _case(pkg, tokens=8, experts=20, hidden=96, inner=64, bits=4, layout=layout, sub=sub, seed=53)
    g = torch.Generator().manual_seed(54)
    for ids in (torch.full((8, 16), 3), torch.randint(2, 5, (8, 16), generator=g), torch.arange(128).view(8, 16) % 23 - 1):
        share = torch.rand(8, 16, generator=g)
        out = pkg.moe_swiglu(*c["device"], topk_ids=ids.int().cuda(), topk_weights=share.cuda(), **c["call"])
        _check(c, out, torch.where(ids < 20, ids, -1), share)


@pytest.mark.parametrize("tokens,experts,top_k", [(8, 256, 16), (3, 257, 8), (9, 1024, 16), (64, 130, 5)])
def test_many_experts(pkg, tokens, experts, top_k):
    c = _case(pkg, tokens=tokens, experts=experts, hidden=64, inner=32, bits=4, layout="nn", sub=0, seed=55)
    for renormalize in (True, False):
        _routed(pkg, c, top_k, renormalize=renormalize)


@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_that_the_quantiser_reads_twice(pkg, bits, layout):
    c = _case(pkg, tokens=2, experts=2, hidden=64, inner=14368, bits=bits, layout=layout, sub=0, seed=56)
    _routed(pkg, c, 2)


@pytest.mark.parametrize("sub", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
def test_ends_of_k_inside_a_step(pkg, bits, layout, sub):
    for tokens, hidden, inner in ((3, 416, 608), (11, 608, 1056), (1, 1056, 32), (18, 32, 2080)):
        c = _case(pkg, tokens=tokens, experts=3, hidden=hidden, inner=inner, bits=bits, layout=layout, sub=sub, seed=hidden + sub)
        _routed(pkg, c, 2)


@pytest.mark.parametrize("layout", ["nt", "nn"])
def test_special_tokens(pkg, layout):
    c = _case(pkg, tokens=6, experts=4, hidden=128, inner=64, bits=4, layout=layout, sub=0, seed=15)
    clean = pkg.moe_swiglu(*c["device"], router_weight=c["router"].cuda(), top_k=2, **c["call"])
    x = c["x"].clone()
    x[1] = 0
    x[2, 7], x[4, 3] = float("nan"), float("inf")
    out = pkg.moe_swiglu(x.cuda(), *c["device"][1:], router_weight=c["router"].cuda(), top_k=2, **c["call"])
    assert not out[1].any() and not torch.isfinite(out[2]).any() and not torch.isfinite(out[4]).any()
    assert torch.equal(out[[0, 3, 5]], clean[[0, 3, 5]])
    assert pkg.moe_swiglu(x.cuda()[:0], *c["device"][1:], router_weight=c["router"].cuda(), top_k=2, **c["call"]).shape == (0, 128)


def test_a_token_alone_and_in_a_batch(pkg):
    """What other tokens are in the call changes no bit of a token's result."""
    for bits, layout, sub in ((4, "nt", 0), (4, "nn", 0), (8, "nn", 64), (4, "nt", 32)):
        c = _case(pkg, tokens=40, experts=6, hidden=256, inner=160, bits=bits, layout=layout, sub=sub, seed=16)
        router = c["router"].cuda()
        whole = pkg.moe_swiglu(*c["device"], router_weight=router, top_k=3, **c["call"])
        again = pkg.moe_swiglu(*c["device"], router_weight=router, top_k=3, **c["call"])
        assert torch.equal(whole, again)
        for t in (0, 17, 39):
            assert torch.equal(pkg.moe_swiglu(c["device"][0][t:t + 1], *c["device"][1:], router_weight=router, top_k=3, **c["call"])[0], whole[t])


@pytest.mark.parametrize("layout", ["nt", "nn"])
def test_offsets_beyond_32_bits(pkg, layout):
    """Experts whose weights start more than 2^32 bytes into the tensor: the same as those experts alone."""
    hidden, inner, experts = 4096, 8192, 134              # 2 * 8192 * 2048 bytes an expert: 4.5e9 in all
    g = torch.Generator(device="cuda").manual_seed(1)
    nn = layout == "nn"
    up = torch.empty((experts, hidden // 2, 2 * inner) if nn else (experts, 2 * inner, hidden // 2), device="cuda", dtype=torch.uint8)
    down = torch.empty((experts, inner // 2, hidden) if nn else (experts, hidden, inner // 2), device="cuda", dtype=torch.uint8)
    up[-2:].random_(generator=g)
    down[-2:].random_(generator=g)
    su = (torch.rand(experts, 2 * inner, device="cuda", generator=g) * 0.004).bfloat16()
    sd = (torch.rand(experts, hidden, device="cuda", generator=g) * 0.004).bfloat16()
    x = torch.randn(3, hidden, device="cuda", generator=g).bfloat16()
    ids = torch.tensor([[experts - 1, experts - 2], [experts - 2, experts - 1], [experts - 1, -1]], device="cuda", dtype=torch.int32)
    weights = torch.rand(3, 2, device="cuda", generator=g)
    kind = dict(layout=pkg.GemmLayout.NN if nn else pkg.GemmLayout.NT)
    out = pkg.moe_swiglu(x, up, down, up_gate_scale=su, down_scale=sd, topk_ids=ids, topk_weights=weights, **kind)
    few = torch.where(ids >= 0, ids - (experts - 2), ids)
    want = pkg.moe_swiglu(x, up[-2:], down[-2:], up_gate_scale=su[-2:], down_scale=sd[-2:], topk_ids=few, topk_weights=weights, **kind)
    assert torch.equal(out, want) and out.float().abs().max() > 0


def test_refusals_on_a_gpu(pkg):
    c = _case(pkg, tokens=2, experts=4, hidden=64, inner=32, bits=4, layout="nn", sub=0, seed=1)
    x, up, down = c["device"]
    router = c["router"].cuda()
    ok = dict(router_weight=router, top_k=2, **c["call"])
    ids, weights = torch.zeros(2, 2, device="cuda", dtype=torch.int32), torch.zeros(2, 2, device="cuda")
    bad = [
        ((x.float(), up, down), ok, "x must have dtype"), ((x[0], up, down), ok, "x must have shape"),
        ((x.repeat(33, 1), up, down), ok, "at most 64 tokens"), ((x.t().contiguous().t(), up, down), ok, "x must be contiguous"),
        ((x, up.to(torch.int8), down), ok, "w_up_gate must have dtype"), ((x, up[0], down), ok, "grouped tensor"),
        ((x, up[:, :-1].contiguous(), down), ok, "does not match"), ((x, up, down[:, :, :32].contiguous()), ok, "w_down must have shape"),
        ((x, up[:3], down), ok, "w_down must have shape"), ((x, up, down), {**ok, "top_k": 0}, "top_k must be in"),
        ((x, up, down), {**ok, "top_k": 5}, "top_k must be in"), ((x, up, down), {**ok, "topk_ids": ids}, "not both"),
        ((x, up, down), {**ok, "router_weight": None}, "give either"), ((x, up, down), {**ok, "router_weight": router[:, :32].contiguous()}, "router_weight must have shape"),
        ((x, up, down), {**ok, "up_gate_scale": ok["up_gate_scale"][:, :32].contiguous()}, "up_gate_scale must have shape"),
        ((x, up, down), {**ok, "down_scale": ok["down_scale"].float()}, "down_scale must have dtype"),
        ((x, up, down), {**ok, "scale": pkg.ScaleSpec(pkg.ScaleMode.SUBCHANNEL, 32)}, "up_gate_scale must have shape"),
        ((x, up, down), {**c["call"], "topk_ids": ids[:1], "topk_weights": weights[:1]}, "topk_ids must have shape"),
        ((x, up, down), {**c["call"], "topk_ids": ids.short(), "topk_weights": weights}, "topk_ids must have dtype"),
        ((x, up, down), {**c["call"], "topk_ids": ids, "topk_weights": weights[:, :1].contiguous()}, "topk_weights must have shape"),
        ((x, up, down), {**c["call"], "topk_ids": ids, "topk_weights": weights, "top_k": 3}, "has 2 columns"),
        ((x[:, :48].contiguous(), up, down), ok, "multiples of 32"),
    ]
    for args, kw, why in bad:
        with pytest.raises(ValueError, match=why):
            pkg.moe_swiglu(*args, **kw)
    with pytest.raises(TypeError, match="top_k must be a Python int"):
        pkg.moe_swiglu(x, up, down, **{**ok, "top_k": 2.0})
    shifted = torch.empty(x.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view_as(x)
    with pytest.raises(ValueError, match="multiple of 16 bytes"):
        pkg.moe_swiglu(shifted, up, down, **ok)


@pytest.mark.parametrize("tokens", [12, 3])
def test_streams_and_graphs(pkg, tokens):
    """Two calls at once on two streams, and two graphs replayed at once on new inputs: each has its own scratch."""
    c = _case(pkg, tokens=tokens, experts=16, hidden=512, inner=256, bits=4, layout="nn", sub=128, seed=21)
    x, up, down = c["device"]
    kw = dict(router_weight=c["router"].cuda(), top_k=4, **c["call"])
    flipped = x.flip(0).contiguous()
    want = [pkg.moe_swiglu(t, up, down, **kw) for t in (x, flipped)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(pkg.moe_swiglu((x, flipped)[i], up, down, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])
    held = [x.clone(), x.clone()]
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pkg.moe_swiglu(held[i], up, down, **kw))
        graphs.append(graph)
    held[1].copy_(flipped)
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_a_decoding_block(pkg):
    """Norm and quantiser into a 4-bit projection, residual, norm, experts: each step against its statement, on what
    the step before it left on the device."""
    tokens, hidden = 32, 512
    c = _case(pkg, tokens=tokens, experts=8, hidden=hidden, inner=256, bits=4, layout="nn", sub=0, seed=31)
    g = torch.Generator().manual_seed(32)
    gamma, beta = [(1 + 0.2 * torch.randn(hidden, generator=g)).bfloat16() for _ in range(2)]
    w = torch.randint(0, 256, (hidden // 2, hidden), generator=g, dtype=torch.uint8)
    ws = ((torch.rand(hidden, generator=g) + 0.5) * 0.01).bfloat16()
    x = c["x"].cuda()
    codes, scales = pkg.layer_norm_quantize(x, gamma.cuda(), beta.cuda())
    attn = pkg.mm(codes, w.cuda(), a_scale=scales, b_scale=ws.cuda())
    h = x + attn
    y, _, _ = pkg.layer_norm(h, gamma.cuda(), beta.cuda())
    out, ids, weights = pkg.moe_swiglu(y, *c["device"][1:], router_weight=c["router"].cuda(), top_k=2, return_routing=True, **c["call"])
    want_codes, want_scales, _ = row_oracle.quantize_rows(row_oracle.norm(c["x"], gamma, beta, 1e-5)[0], 4)
    assert torch.equal(pkg.unpack_int4_k_major(codes.cpu()), want_codes) and torch.equal(scales.cpu().double(), want_scales)
    exact = (want_codes.double() @ moe_oracle.unpack(w, 4, 0)) * want_scales[:, None] * ws.double()
    assert ((attn.cpu().double() - exact).abs() <= (2.0 ** -8 + 4 * U) * exact.abs()).all()
    c["x"] = y.cpu()
    want_ids, want_share = moe_oracle.route(c["x"], c["router"], 2)
    assert torch.equal(ids.cpu().long(), want_ids)
    _check(c, out, want_ids, want_share)


def test_a_training_step_around_grouped_products(pkg):
    """Norm, quantiser, grouped product forward and backward, norm backward: shapes and formats fit together, and the
    products see exactly the quantised rows."""
    sizes = [48, 0, 80, 32]
    rows, hidden, inner = sum(sizes), 256, 512
    g = torch.Generator().manual_seed(41)
    x = torch.randn(rows, hidden, generator=g).bfloat16()
    gamma = (1 + 0.2 * torch.randn(hidden, generator=g)).bfloat16()
    w = torch.randint(0, 256, (4, hidden // 2, inner), generator=g, dtype=torch.uint8)
    ws = ((torch.rand(4, inner, generator=g) + 0.5) * 0.01).bfloat16()
    sizes_d = torch.tensor(sizes).cuda()
    y, mean, rstd = pkg.layer_norm(x.cuda(), gamma.cuda())
    codes, scales = pkg.quantize_tokens(y)
    z = pkg.ragged_dot_int4(codes, w.cuda(), sizes_d, a_scale=scales, b_scale=ws.cuda())
    want_codes, want_scales, _ = row_oracle.quantize_rows(y.cpu(), 4)
    starts = [0, 48, 48, 128, 160]
    for e in range(4):
        part = slice(starts[e], starts[e + 1])
        exact = (want_codes[part].double() @ moe_oracle.unpack(w[e], 4, 0)) * want_scales[part, None] * ws[e].double()
        assert ((z[part].cpu().double() - exact).abs() <= (2.0 ** -8 + 4 * U) * exact.abs()).all()
    dz = (torch.randn(rows, inner, generator=g) / rows).bfloat16().cuda()
    dz_codes, dz_scales = pkg.quantize_tokens(dz)
    # the weight gradient's scales are one for each group and column: codes of the whole batch with one constant
    ones = torch.ones(4, hidden, device="cuda", dtype=torch.bfloat16), torch.ones(4, inner, device="cuda", dtype=torch.bfloat16)
    dw = pkg.ragged_dot_int4_bwd_flat(pkg.repack_int4_tokens(codes), pkg.repack_int4_tokens(dz_codes), sizes_d, a_scale=ones[0], b_scale=ones[1])
    dz_exact = row_oracle.quantize_rows(dz.cpu(), 4)
    assert torch.equal(dz_scales.cpu().double(), dz_exact[1])
    for e in range(4):
        part = slice(starts[e], starts[e + 1])
        assert torch.equal(dw[e].cpu().double(), want_codes[part].double().t() @ dz_exact[0][part].double())
    dy = (torch.randn(rows, hidden, generator=g) / rows).bfloat16().cuda()
    dx, dgamma, dbeta = pkg.layer_norm_bwd(dy, x.cuda(), gamma.cuda(), mean, rstd)
    want = row_oracle.norm_bwd(dy.cpu(), x, gamma, mean.cpu(), rstd.cpu())
    assert ((dx.cpu().double() - want[0]).abs() <= 2.0 ** -8 * want[0].abs() + 1e-5 * rstd.cpu()[:, None] * dy.cpu().abs().max()).all()
    assert (dgamma.cpu().double() - want[1]).abs().max() <= 1e-5 * want[1].abs().max() and (dbeta.cpu().double() - want[2]).abs().max() <= 1e-5 * want[2].abs().max()


# ---------------------------------------------------------------------------------------------------------------
def _given(pkg, c, ids, share, **more):
    call = {**c["call"], "up_gate_scale": c["s_up_gate"].cuda(), "down_scale": c["s_down"].cuda(), **more}
    return pkg.moe_swiglu(c["x"].cuda(), c["w_up_gate"].cuda(), c["w_down"].cuda(), topk_ids=ids.cuda(), topk_weights=share.cuda(), **call)


@pytest.mark.parametrize("sub", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
def test_scales_of_any_size(pkg, bits, layout, sub):
    """Tokens 2^k times smaller and scales of the first product 2^k times larger, and the same with the second product's scales
    and the experts' weights: powers of two that cancel, so that no bit of the result changes, up to the largest scales that
    bfloat16 has."""
    c = _case(pkg, tokens=11, experts=4, hidden=512, inner=768, bits=bits, layout=layout, sub=sub, seed=61)
    g = torch.Generator().manual_seed(62)
    ids, share = torch.randint(0, 4, (11, 2), generator=g), torch.rand(11, 2, generator=g) + 0.5
    small = 2.0 ** -122 if bits == 4 else 2.0 ** -117     # the tokens' scales stay normal bfloat16 numbers
    c["x"] = (c["x"].double() * small).bfloat16().double().div(small).bfloat16()      # no digits that the small tokens do not have
    want = _given(pkg, c, ids, share)
    _check(c, want, ids, share)
    scaled = {**c, "x": (c["x"].double() * small).bfloat16(), "s_up_gate": (c["s_up_gate"].double() / small).bfloat16()}
    assert torch.equal(_given(pkg, scaled, ids, share), want)
    scaled = {**c, "s_down": (c["s_down"].double() / small).bfloat16()}
    assert torch.equal(_given(pkg, scaled, ids, share * small), want)


@pytest.mark.parametrize("sub", [0, 64])
@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
def test_columns_of_zeros_with_large_scales(pkg, bits, layout, sub):
    """A sum of zero is zero, whatever its two scales are: their product may be beyond float32."""
    c = _case(pkg, tokens=3, experts=2, hidden=128, inner=64, bits=bits, layout=layout, sub=sub, seed=63)
    nn = layout == "nn"
    for name, s_name, n in (("w_up_gate", "s_up_gate", 128), ("w_down", "s_down", 128)):
        empty = torch.arange(n) % 3 == 1
        w = c[name]
        if nn:
            w[:, :, empty] = 0
        else:
            w[:, empty] = 0
        c[s_name][..., empty] = 2.0 ** 100
    # the other columns: tokens of about 2^40, activations of about 2^60
    c["x"] = (c["x"].double() * 2.0 ** 40).bfloat16()
    c["s_up_gate"][..., torch.arange(128) % 3 != 1] *= 2.0 ** -10
    c["s_down"][..., torch.arange(128) % 3 != 1] *= 2.0 ** -60
    ids, share = torch.tensor([[0, 1], [1, 0], [0, 0]]), torch.tensor([[0.5, 0.5], [0.25, 0.75], [1.0, 2.0]])
    out = _given(pkg, c, ids, share)
    assert torch.isfinite(out).all() and not out[:, torch.arange(128) % 3 == 1].any()
    _check(c, out, ids, share)


@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("sub", [0, 128])
@pytest.mark.parametrize("bits", [4, 8])
def test_products_of_scales_below_float32(pkg, bits, sub, layout):
    """The product of two scales has sixteen significant bits however small it is; the sum that it multiplies brings the
    result back into range.  (Tokens of 2^-20, up scales of 2^-117, gate scales of 2^90; then down scales of 2^-100 behind
    activations of about 2^-35.)"""
    inner = 1024
    c = _case(pkg, tokens=5, experts=2, hidden=512, inner=inner, bits=bits, layout=layout, sub=sub, seed=64)
    c["x"] = (c["x"].double() * 2.0 ** -20).bfloat16()
    c["s_up_gate"][..., :inner] *= 2.0 ** -112
    c["s_up_gate"][..., inner:] *= 2.0 ** 96
    ids, share = torch.tensor([[0, 1], [1, 0], [0, 1], [1, 1], [0, 0]]), torch.ones(5, 2)
    out = _given(pkg, c, ids, share)
    assert out.abs().max() > 0
    _check(c, out, ids, share)
    c["s_down"] *= 2.0 ** -72
    out = _given(pkg, c, ids, share)
    want, size = moe_oracle.layer(c["x"], c["w_up_gate"], c["w_down"], c["s_up_gate"], c["s_down"], ids, share, bits=bits, nn=layout == "nn", sub=sub)
    assert 2.0 ** -126 < want.abs().max() < 2.0 ** -100
    # as _check, and the steps of subnormal numbers: half of 2^-149 a share and a sum, half of 2^-133 at the end
    off = 6 * U * size + 4 * 2.0 ** -150
    assert ((out.cpu().double() - want).abs() <= 1.01 * off + 2.0 ** -8 * (want.abs() + off) + 2.0 ** -134).all()


@pytest.mark.parametrize("layout", ["nn", "nt"])
def test_a_token_alone_and_in_a_batch_where_k_is_divided(pkg, layout):
    """One scale a column: the down product of one token divides K into more parts than that of the batch, and the integer
    sums are the same."""
    from strix_halo_int4_gemms_b200 import native

    tokens, hidden, inner, experts = 40, 2048, 2048, 32
    nn, kind = layout == "nn", dict(layout=pkg.GemmLayout(layout), dtype=pkg.OperandDType.INT8)

    def parts(count):     # by the scratch that they ask for: all of it but the codes and activations, in shares of [pairs, hidden]
        fields = (native.DTYPE_CODES[kind["dtype"]], native.LAYOUT_CODES[kind["layout"]], 0, count, hidden, inner, experts, 2, native.OUT_BF16, 1, 32)
        return (native.moe_problem(*fields)[1] - count * (2 * inner * 9 + hidden)) // (count * 2 * hidden * 4)

    assert parts(1) > parts(tokens) >= 1
    g = torch.Generator(device="cuda").manual_seed(65)
    up, down = [torch.randint(-128, 128, (experts, k, n) if nn else (experts, n, k), generator=g, device="cuda", dtype=torch.int8)
                for k, n in ((hidden, 2 * inner), (inner, hidden))]
    su, sd = [((torch.rand(experts, n, generator=g, device="cuda") + 0.5) / 3300).bfloat16() for n in (2 * inner, hidden)]
    x = torch.randn(tokens, hidden, generator=g, device="cuda").bfloat16()
    router = (torch.randn(experts, hidden, generator=g, device="cuda") / hidden ** 0.5).bfloat16()
    call = dict(up_gate_scale=su, down_scale=sd, router_weight=router, top_k=2, **kind)
    whole = pkg.moe_swiglu(x, up, down, **call)
    assert torch.isfinite(whole).all() and whole.float().abs().max() > 0
    for t in (0, 17, 39):
        assert torch.equal(pkg.moe_swiglu(x[t:t + 1], up, down, **call)[0], whole[t])


@pytest.mark.parametrize("sub", [32, 64, 128, 256])
def test_scales_of_k_groups_into_the_products(pkg, sub):
    """``quantize_tokens`` and ``layer_norm_quantize`` with a scale for each K-group are the A operand and ``a_scale`` of the
    dense products."""
    rows, k, n = 256, 512, 256
    g = torch.Generator().manual_seed(sub)
    x = torch.randn(rows, k, generator=g).bfloat16()
    gamma = (1 + 0.2 * torch.randn(k, generator=g)).bfloat16()
    w = torch.randint(0, 256, (k // 2, 2 * n), generator=g, dtype=torch.uint8)
    ws = ((torch.rand(k // sub, 2 * n, generator=g) + 0.5) * 0.01).bfloat16()
    spec = pkg.ScaleSpec(pkg.ScaleMode.SUBCHANNEL, sub)
    full = moe_oracle.unpack(w, 4, 0)
    for codes_scales, rows64 in ((pkg.quantize_tokens(x.cuda(), scale=spec), x),
                                 (pkg.layer_norm_quantize(x.cuda(), gamma.cuda(), scale=spec), row_oracle.norm(x, gamma, None, 1e-5)[0])):
        codes, scales = codes_scales
        want_codes, want_scales, _ = row_oracle.quantize_rows(rows64, 4, sub)
        parts = torch.stack([(want_codes[:, i * sub:(i + 1) * sub].double() @ full[i * sub:(i + 1) * sub]) * want_scales[:, i:i + 1] * ws[i].double() for i in range(k // sub)])
        exact, size = parts.sum(0), parts.abs().sum(0)
        out = pkg.mm(codes, w.cuda(), a_scale=scales, b_scale=ws.cuda(), scale=spec)
        # a group's integer sum, two scales and the sum over at most 16 groups in float32; bfloat16 at the end
        off = (k // sub + 4) * U * size
        assert ((out.cpu().double() - exact).abs() <= 1.01 * off + 2.0 ** -8 * (exact.abs() + off)).all()
        fused = pkg.fused_swiglu_up_gate(codes, w.cuda(), a_scale=scales, b_scale=ws.cuda(), scale=spec)
        packed = pkg.pack_int4_k_major(want_codes).cuda()
        assert torch.equal(fused, pkg.fused_swiglu_up_gate(packed, w.cuda(), a_scale=want_scales.bfloat16().cuda(), b_scale=ws.cuda(), scale=spec))


@pytest.mark.parametrize("layout", ["nt", "nn"])
def test_as_many_pairs_as_there_can_be(pkg, layout):
    c = _case(pkg, tokens=64, experts=1024, hidden=64, inner=32, bits=4, layout=layout, sub=0, seed=71)
    _routed(pkg, c, 16)


@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hidden,inner", [(131040, 32), (32, 131040)])
def test_largest_sums(pkg, bits, layout, hidden, inner):
    """The longest K with the largest codes of one sign on both sides: the integer sums come within 1 % (int8) of 2^31."""
    c = _case(pkg, tokens=2, experts=2, hidden=hidden, inner=inner, bits=bits, layout=layout, sub=0, seed=72)
    for name in ("w_up_gate", "w_down"):
        c[name][0] = 0x88 if bits == 4 else -128
    c["x"] = torch.full((2, hidden), 1.5).bfloat16()
    c["x"][1] = -2.0
    # up and gate of about +-6, activations of one sign each, and results of the size of one
    lowest = 8.0 if bits == 4 else 128.0
    c["s_up_gate"][0] = 4.0 / (hidden * lowest)
    c["s_down"][0] = 1.0 / (inner * lowest)
    ids, share = torch.tensor([[0], [0]]), torch.ones(2, 1)
    out = _given(pkg, c, ids, share)
    assert torch.isfinite(out).all() and (out != 0).all()
    _check(c, out, ids, share)
