"""The quantiser for each token, layer norm, both in one, and layer norm's backward pass on a B200 against plain
64-bit statements.  Codes and scales have to be equal.  The bounds of the floating results count roundings: one of
float32 is off by 2^-24 of its value, one of bfloat16 by 2^-8, and a sum of n terms in any order by the number of
additions on the longest path times 2^-24 of the sum of their sizes."""
import pytest
import torch

import row_oracle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _depth(cols):
    """Additions on the longest path of a row's sum: what one thread adds up (at most 32 in registers; in the rows that
    are read again, eight for each 4096 columns), and the trees over lanes and warps."""
    return max(32, 8 * -(-cols // 4096)) + 10


def _rows(rows, cols, dtype, seed, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * (1 + 7 * (torch.rand(cols, generator=g) < 0.02)) + offset * torch.randn(rows, 1, generator=g)
    return x.to(dtype)


def _codes(pkg, codes, bits, cols):
    if bits == 8:
        return codes.cpu()
    return pkg.unpack_int4_k_major(codes.cpu())[..., :cols]


def _spec(pkg, sub):
    return pkg.ScaleSpec(pkg.ScaleMode.SUBCHANNEL, sub) if sub else pkg.ScaleSpec(pkg.ScaleMode.PER_CHANNEL)


def _dtype(pkg, bits):
    return pkg.OperandDType.INT4 if bits == 4 else pkg.OperandDType.INT8


def _shifted(t, by=1):
    """The same values, contiguous, at an address that is a multiple of the element size only."""
    flat = torch.empty(t.numel() + by, device="cuda", dtype=t.dtype)
    flat[by:] = t.cuda().flatten()
    return flat[by:].view(t.shape)


COLS = [1, 2, 7, 8, 31, 64, 255, 256, 257, 384, 512, 1000, 1024, 1405, 2048, 2056, 4096, 4104, 7168, 8192, 10000, 16384, 16392, 40001]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("cols", COLS)
def test_quantize_tokens(pkg, cols, bits):
    for sub in (0, 32, 64, 128, 256):
        x = _rows(11, cols, torch.bfloat16, cols + bits + sub)
        x[3] = 0
        x[4] *= 1e-30
        codes, scales = pkg.quantize_tokens(x.cuda(), dtype=_dtype(pkg, bits), scale=_spec(pkg, sub))
        want, want_scales, _ = row_oracle.quantize_rows(x, bits, sub)
        assert torch.equal(scales.cpu().double(), want_scales), sub
        assert torch.equal(_codes(pkg, codes, bits, cols), want), sub
        if bits == 4 and cols % 2:
            assert not (codes.cpu()[:, -1] >> 4).any()        # the padding nibble


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_tokens_ties_and_all_bf16_quotients(pkg, bits):
    """Every significand of x against every significand of the scale, over the exponents that codes come from: ties
    included, and scales at both ends of the range."""
    top = row_oracle.TOP[bits]
    sig = torch.arange(128, 256, dtype=torch.float64)
    for power in (-130, -100, -99, -30, 0, 30, 99, 104):
        amax = round_max = sig * top * 2.0 ** (power - 7)        # a scale near sig * 2^(power - 7)
        head = row_oracle.round_bf16(round_max)
        body = torch.cat([sig * 2.0 ** (power - 7 + e) for e in range(-3, 7)])
        x = torch.cat([head[:, None], body[None, :].expand(128, -1), -body[None, :].expand(128, -1)], 1)
        x = torch.where(x.abs() <= head[:, None], x, torch.zeros_like(x))
        x = torch.where(x.abs() < 3.3e38, x, torch.zeros_like(x)).float().bfloat16()
        codes, scales = pkg.quantize_tokens(x.cuda(), dtype=_dtype(pkg, bits))
        want, want_scales, _ = row_oracle.quantize_rows(x, bits)
        assert torch.equal(scales.cpu().double(), want_scales), power
        assert torch.equal(_codes(pkg, codes, bits, x.shape[1]), want), power
        assert amax.numel() == 128


@pytest.mark.parametrize("sub", [0, 64])
@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_tokens_special_values(pkg, bits, sub):
    x = _rows(8, 200, torch.bfloat16, 5)
    x[0, 3] = float("inf")
    x[1, 70] = -float("inf")
    x[2, 199] = float("nan")
    x[3] = 2.0 ** -133                      # subnormal: the scale rounds to zero or loses bits
    x[4, :] = torch.tensor(3.3895e38).bfloat16()
    x[5] = 0
    x[6, 0] = -0.0
    codes, scales = pkg.quantize_tokens(x.cuda(), dtype=_dtype(pkg, bits), scale=_spec(pkg, sub))
    want, want_scales, _ = row_oracle.quantize_rows(x, bits, sub)
    assert torch.equal(torch.nan_to_num(scales.cpu().double(), nan=-1.0), torch.nan_to_num(want_scales, nan=-1.0))
    assert torch.equal(_codes(pkg, codes, bits, 200), want)


def test_quantize_tokens_shapes_and_alignment(pkg):
    x = _rows(6, 320, torch.bfloat16, 9)
    want, want_scales, _ = row_oracle.quantize_rows(x, 4, 64)
    for t in (x.cuda().view(2, 3, 320), _shifted(x).view(2, 3, 320)):
        codes, scales = pkg.quantize_tokens(t, scale=_spec(pkg, 64))
        assert codes.shape == (2, 3, 160) and scales.shape == (2, 3, 5)
        assert torch.equal(_codes(pkg, codes, 4, 320).view(6, 320), want) and torch.equal(scales.cpu().double().view(6, 5), want_scales)
    codes, scales = pkg.quantize_tokens(torch.zeros(0, 320, device="cuda", dtype=torch.bfloat16))
    assert codes.shape == (0, 160) and scales.shape == (0,)
    codes, scales = pkg.quantize_tokens(x[0].cuda())
    assert codes.shape == (160,) and scales.shape == ()
    with pytest.raises(ValueError, match="contiguous"):
        pkg.quantize_tokens(x.cuda().t())


# ---------------------------------------------------------------------------------------------------------------
def _affine(cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(cols, generator=g)).to(dtype), (0.5 * torch.randn(cols, generator=g)).to(dtype)


def _check_norm(pkg, x, w, b, eps, xd):
    y, mean, rstd = pkg.layer_norm(xd, w.cuda(), None if b is None else b.cuda(), eps=eps)
    assert y.dtype == x.dtype and y.shape == xd.shape and mean.dtype == rstd.dtype == torch.float32
    want, want_mean, want_rstd = row_oracle.norm(x, w, b, eps)
    d = _depth(x.shape[1])
    xs = x.double()
    size = xs.abs().mean(-1)
    off_mean = (d + 2) * U * size                                     # the sum, its division, its storing
    assert ((mean.cpu().double().flatten() - want_mean).abs() <= off_mean).all()
    # the variance: squares of differences that are off by the mean's error and one rounding, their sum
    spread = (xs - want_mean[:, None]).abs()
    off_d = off_mean[:, None] + U * spread
    var = (spread ** 2).mean(-1) + eps
    off_var = ((d + 4) * U * var + (2 * spread * off_d + off_d ** 2).mean(-1)) / var
    off_rstd = off_var / 2 * 1.01 + 4 * U                             # rsqrtf: 2 ulp of 2^-23
    assert ((rstd.cpu().double().flatten() / want_rstd - 1).abs() <= off_rstd).all()
    t = (xs - want_mean[:, None]).abs() * want_rstd[:, None] * w.double().abs()
    bound = off_d * want_rstd[:, None] * w.double().abs() + t * (off_rstd[:, None] + 3 * U) + U * (t + (0 if b is None else b.double().abs()))
    bound = 1.01 * bound + HALF_STEP[x.dtype] * (want.abs() + bound)
    worst = ((y.cpu().double().view(x.shape) - want).abs() / bound.clamp_min(1e-300)).max()
    assert worst <= 1, float(worst)


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm(pkg, cols, xt, wt):
    x = _rows(9, cols, xt, cols)
    w, b = _affine(cols, wt, cols + 1)
    _check_norm(pkg, x, w, b, 1e-5, x.cuda())
    _check_norm(pkg, x, w, None, 1e-3, x.cuda())


def test_layer_norm_shapes_alignment_and_offsets(pkg):
    w, b = _affine(264, torch.bfloat16, 1)
    x = _rows(6, 264, torch.bfloat16, 2)
    _check_norm(pkg, x, w, b, 1e-5, x.cuda().view(3, 2, 264))
    _check_norm(pkg, x, w, b, 1e-5, _shifted(x))
    y, mean, rstd = pkg.layer_norm(x.cuda()[:0], w.cuda(), b.cuda())
    assert y.shape == (0, 264) and mean.shape == rstd.shape == (0,)
    y1 = pkg.layer_norm(x.cuda(), _shifted(w), _shifted(b, 3))[0]
    assert torch.equal(y1, pkg.layer_norm(x.cuda(), w.cuda(), b.cuda())[0])
    y1, mean, _ = pkg.layer_norm(x[0].cuda(), w.cuda(), b.cuda())
    assert y1.shape == (264,) and mean.shape == ()
    # an offset a thousand times the spread: the differences are taken from the mean, not from the squares
    x32 = _rows(5, 1000, torch.float32, 3) + 1000
    w, b = _affine(1000, torch.float32, 4)
    _check_norm(pkg, x32, w, b, 1e-5, x32.cuda())
    # a row that is not finite stays its own affair
    x[2, 5] = float("nan")
    x[4, 0] = float("inf")
    y = pkg.layer_norm(x.cuda(), *[t.cuda() for t in _affine(264, torch.bfloat16, 1)])[0].cpu()
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all() and torch.isfinite(y[[0, 1, 3, 5]]).all()


# ---------------------------------------------------------------------------------------------------------------
def _check_norm_codes(pkg, x, w, b, bits, sub, xd=None, eps=1e-5):
    codes, scales = pkg.layer_norm_quantize(x.cuda() if xd is None else xd, w.cuda(), None if b is None else b.cuda(), eps=eps,
                                            dtype=_dtype(pkg, bits), scale=_spec(pkg, sub))
    want, want_scales, border = row_oracle.quantize_rows(row_oracle.norm(x, w, b, eps)[0], bits, sub)
    assert torch.equal(scales.cpu().double().view(want_scales.shape), want_scales)
    got = _codes(pkg, codes, bits, x.shape[1]).view(x.shape)
    # where the oracle's own float64 arithmetic cannot tell the two codes apart, either may be right
    same = (got == want) | ((border < 1e-11 * row_oracle.TOP[bits]) & ((got.int() - want.int()).abs() == 1))
    assert same.all(), int((~same).sum())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_quantize(pkg, cols, xt, bits):
    for sub, wt, with_bias in ((0, torch.bfloat16, True), (0, torch.float32, False), (32, torch.float32, True), (64, torch.bfloat16, True),
                               (128, torch.bfloat16, False), (256, torch.float32, True)):
        x = _rows(9, cols, xt, cols + sub)
        w, b = _affine(cols, wt, cols + 2)
        _check_norm_codes(pkg, x, w, b if with_bias else None, bits, sub)


@pytest.mark.parametrize("sub", [0, 128])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
def test_layer_norm_quantize_many_values(pkg, xt, sub):
    """Enough values that many of them lie next to a border in float32 (8 bits: a zone of about 10^-4 of a code)."""
    x = _rows(700, 2048, xt, 77, offset=3.0)
    w, b = _affine(2048, torch.float32, 78)
    _check_norm_codes(pkg, x, w, b, 8, sub)
    _check_norm_codes(pkg, x, w, 40 * b, 8, sub)       # a bias much larger than the norm
    _check_norm_codes(pkg, x + 100, w, b, 4, sub)      # a mean much larger than the spread


@pytest.mark.parametrize("sub", [0, 32])
def test_layer_norm_quantize_special_rows(pkg, sub):
    x = _rows(8, 256, torch.bfloat16, 6)
    w, b = torch.ones(256), torch.zeros(256)
    x[0] = 1.5                                       # equal values: the norm is the bias
    x[1] = 0
    _check_norm_codes(pkg, x, w, b, 4, sub)
    b2 = torch.linspace(-3, 3, 256)
    _check_norm_codes(pkg, x, w, b2, 4, sub)
    x3 = x.float()
    x3[0] = 0.1
    _check_norm_codes(pkg, x3, w, torch.arange(256.0) % 15 - 7, 4, sub)   # ties and whole codes, exactly
    _check_norm_codes(pkg, x3 * 1e18, w, b2, 8, sub)
    _check_norm_codes(pkg, x3[2:] * 1e-22, w, None, 8, sub, eps=0.0)
    x[2, 9], x[3, 200] = float("nan"), -float("inf")
    codes, scales = pkg.layer_norm_quantize(x.cuda(), w.cuda(), b.cuda(), scale=_spec(pkg, sub))
    codes, scales = _codes(pkg, codes, 4, 256), scales.cpu().view(8, -1)
    assert not codes[2].any() and not codes[3].any() and torch.isnan(scales[2:4]).all() and torch.isfinite(scales[4:]).all()


@pytest.mark.parametrize("sub", [0, 32])
@pytest.mark.parametrize("bits", [4, 8])
def test_layer_norm_quantize_beyond_float32(pkg, bits, sub):
    """Differences, products and scales that float32 has no room for, or too few digits: the exact values decide."""
    g = torch.Generator().manual_seed(61)
    x = torch.randn(6, 512, generator=g)
    x[1] = torch.where(torch.rand(512, generator=g) < 0.05, 3.3e38, -3.3e38)    # x - mean is beyond float32
    x[2] *= 1e-30
    x[3] *= 1e25
    x[4] = 1e30 + x[4] * 1e24
    w = torch.randn(512, generator=g)
    for weight, bias in ((w, None), (w, w.flip(0)), (w * 1e38, None), (w * 1e-38, None), (w * 1e-42, None), (w * 1e-20, w * 1e18)):
        weight = torch.where(torch.isfinite(weight), weight, torch.ones(()))
        for eps in (0.0, 1e-5):
            _check_norm_codes(pkg, x, weight, bias, bits, sub, eps=eps)


@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [512, 1032, 2040, 4096, 8184, 16384])
def test_many_rows(pkg, cols, xt):
    """Rows enough for the launch shapes with many values a thread."""
    x = _rows(600, cols, xt, cols + 5)
    w, b = _affine(cols, torch.bfloat16, cols + 6)
    _check_norm(pkg, x, w, b, 1e-5, x.cuda())
    _check_norm_codes(pkg, x, w, b, 4, 0)
    if xt is torch.bfloat16:
        for bits, sub in ((4, 0), (8, 64)):
            codes, scales = pkg.quantize_tokens(x.cuda(), dtype=_dtype(pkg, bits), scale=_spec(pkg, sub))
            want, want_scales, _ = row_oracle.quantize_rows(x, bits, sub)
            assert torch.equal(scales.cpu().double(), want_scales) and torch.equal(_codes(pkg, codes, bits, cols), want)


def test_layer_norm_quantize_shapes_and_alignment(pkg):
    x = _rows(6, 320, torch.bfloat16, 9)
    w, b = _affine(320, torch.bfloat16, 10)
    _check_norm_codes(pkg, x, w, b, 4, 0, xd=x.cuda().view(2, 3, 320))
    _check_norm_codes(pkg, x, w, b, 4, 64, xd=_shifted(x))
    codes, scales = pkg.layer_norm_quantize(x.cuda()[:0], w.cuda(), b.cuda())
    assert codes.shape == (0, 160) and scales.shape == (0,)


# ---------------------------------------------------------------------------------------------------------------
def _check_bwd(pkg, x, dy, w, shape=None):
    shape = shape or x.shape
    wd, xd, dyd = w.cuda(), x.cuda().view(shape), dy.cuda().view(shape)
    _, mean, rstd = pkg.layer_norm(xd, wd)
    dx, dw, db = pkg.layer_norm_bwd(dyd, xd, wd, mean, rstd)
    again = pkg.layer_norm_bwd(dyd, xd, wd, mean, rstd)
    assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), again))
    assert dx.dtype == x.dtype and dx.shape == shape and dw.dtype == db.dtype == torch.float32 and dw.shape == (x.shape[1],)
    m, r = mean.cpu().double().flatten(), rstd.cpu().double().flatten()
    want_dx, want_dw, want_db = row_oracle.norm_bwd(dy, x, w, m, r)
    d = _depth(x.shape[1])
    h = ((x.double() - m[:, None]) * r[:, None]).abs()                 # two roundings
    g = (dy.double() * w.double()).abs()                               # one
    mg, mgh = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    off = r[:, None] * U * (5 * g + (d + 6) * mg + (d + 12) * h * mgh)
    bound = 1.01 * off + HALF_STEP[x.dtype] * (want_dx.abs() + off)
    worst = ((dx.cpu().double().view(x.shape) - want_dx).abs() / bound.clamp_min(1e-300)).max()
    assert worst <= 1, float(worst)
    # a block adds at most rows / 148 + 1 of its own rows (or a thread rows / 32), then trees and at most 20 partial sums
    path = x.shape[0] / (148 if x.shape[1] <= 16384 else 32) + 1 + 8 + 20 + 5
    for got, want, terms in ((dw, want_dw, (dy.double().abs() * h).sum(0)), (db, want_db, dy.double().abs().sum(0))):
        worst = ((got.cpu().double() - want).abs() / (1.01 * (path + 4) * U * terms).clamp_min(1e-300)).max()
        assert worst <= 1, float(worst)


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_bwd(pkg, cols, xt, wt):
    for rows in (1, 9, 300):
        if rows * cols > 3_000_000:
            continue
        x = _rows(rows, cols, xt, cols + rows)
        dy = _rows(rows, cols, xt, cols + rows + 1) / 7
        _check_bwd(pkg, x, dy, _affine(cols, wt, cols + 2)[0])


@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(20001, 64), (20001, 250), (11000, 512), (5003, 1000), (3001, 2048), (1501, 4096), (901, 8192)])
def test_layer_norm_bwd_rows_that_wait_their_turn(pkg, rows, cols, xt):
    """Many more rows than are on their way at once."""
    x, dy = _rows(rows, cols, xt, cols + 7), _rows(rows, cols, xt, cols + 8)
    _check_bwd(pkg, x, dy, _affine(cols, torch.bfloat16, cols + 9)[0])


def test_layer_norm_bwd_many_rows_and_shapes(pkg):
    for rows, cols in ((20011, 48), (5000, 320), (3001, 1000)):
        x = _rows(rows, cols, torch.bfloat16, rows)
        _check_bwd(pkg, x, _rows(rows, cols, torch.bfloat16, rows + 1), _affine(cols, torch.float32, 2)[0])
    x, dy = _rows(6, 264, torch.bfloat16, 1), _rows(6, 264, torch.bfloat16, 2)
    w = _affine(264, torch.bfloat16, 3)[0]
    _check_bwd(pkg, x, dy, w, shape=(2, 3, 264))
    _, mean, rstd = pkg.layer_norm(x.cuda(), w.cuda())
    want = pkg.layer_norm_bwd(dy.cuda(), x.cuda(), w.cuda(), mean, rstd)
    got = pkg.layer_norm_bwd(_shifted(dy), _shifted(x, 3), _shifted(w), mean, rstd)
    # the narrow loads of unaligned tensors use another number of threads for no row here: the same sums
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    empty = torch.zeros(0, 264, device="cuda", dtype=torch.bfloat16)
    dx, dw, db = pkg.layer_norm_bwd(empty, empty, w.cuda(), mean[:0], rstd[:0])
    assert dx.shape == (0, 264) and not dw.any() and not db.any() and dw.shape == (264,)
    with pytest.raises(ValueError, match="dy must have"):
        pkg.layer_norm_bwd(dy.cuda().float(), x.cuda(), w.cuda(), mean, rstd)
    with pytest.raises(ValueError, match="dy must have the shape"):
        pkg.layer_norm_bwd(dy.cuda()[:5], x.cuda(), w.cuda(), mean, rstd)
    with pytest.raises(ValueError, match="mean must have shape"):
        pkg.layer_norm_bwd(dy.cuda(), x.cuda(), w.cuda(), mean[:5], rstd)
    with pytest.raises(ValueError, match="rstd must have dtype"):
        pkg.layer_norm_bwd(dy.cuda(), x.cuda(), w.cuda(), mean, rstd.double())


def test_row_operators_on_streams_and_in_graphs(pkg):
    """Two streams at once, and one graph replayed on new inputs: each call has its own scratch."""
    x = _rows(500, 1024, torch.bfloat16, 21).cuda()
    dy = _rows(500, 1024, torch.bfloat16, 22).cuda()
    w, b = [t.cuda() for t in _affine(1024, torch.bfloat16, 23)]

    def step(x, dy):
        y, mean, rstd = pkg.layer_norm(x, w, b)
        return (*pkg.layer_norm_bwd(dy, x, w, mean, rstd), *pkg.quantize_tokens(y), *pkg.layer_norm_quantize(x, w, b))

    want, other = step(x, dy), step(x.flip(0).contiguous(), dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    flipped = x.flip(0).contiguous()
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = step(flipped if i else x, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got[0], want)) and all(torch.equal(a, c) for a, c in zip(got[1], other))
    held_x, held_dy = x.clone(), dy.clone()
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(held_x, held_dy))
        graphs.append(graph)
    held_x.copy_(flipped)
    for stream, graph in zip(streams, graphs):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for result in results:
        assert all(torch.equal(a, c) for a, c in zip(result, other))


# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [1, 7, 255, 1000, 1405, 2040, 2048, 7168, 10000, 20000, 40001])
def test_layer_norm_of_equal_values(pkg, cols, xt):
    """A row of equal values has that value as its mean and no variance: its norm is the bias, or zero without one, and
    the quantiser behind it gives codes of zero, as the two in one pass do."""
    values = torch.tensor([0.0, 0.1, 1.0, -3.3, 100.0, 999.0, 29952.0, -1e6, 1e-20, 3e15]).to(xt)
    w, b = _affine(cols, xt, cols)
    for rows in (10, 650):                                            # few rows and many have launch shapes of their own
        x = values.repeat(rows // 10)[:, None].expand(rows, cols).contiguous()
        y, mean, rstd = pkg.layer_norm(x.cuda(), w.cuda(), b.cuda())
        assert torch.equal(mean.cpu(), x[:, 0].float())
        assert torch.equal(y.cpu(), b.expand(rows, cols))
        assert ((rstd.cpu().double() * 1e-5 ** 0.5 - 1).abs() <= 5 * U).all()      # eps as fp32, the sum, rsqrtf: 2 ulp of 2^-23
        y = pkg.layer_norm(x.cuda(), w.cuda())[0]
        assert not y.any()
        if xt is torch.bfloat16:
            for codes, scales in (pkg.quantize_tokens(y), pkg.layer_norm_quantize(x.cuda(), w.cuda())):
                assert not codes.any() and (scales == 1).all()


@pytest.mark.parametrize("first", [0.0, 30.0, 1e4])
@pytest.mark.parametrize("cols", [255, 1000, 2040, 7168, 20000])
def test_layer_norm_of_nearly_equal_values(pkg, cols, first):
    """The mean's own rounding, and what the sum of large equal parts loses, shift no row: the bound is the spread's, not the
    offset's.  The mean's first part, from d rounded differences from the row's first value x0, is off by at most p =
    U ((d + 5) (S + |x0 - m|) + |m|), S being the mean |x - m|; the second, from d rounded differences from the first, by
    e = U (d + 5) (S + p).  A difference has a rounding of its own, the two products one each, and the correction one."""
    w, b = _affine(cols, torch.float32, cols)
    g = torch.Generator().manual_seed(cols)
    for rows in (9, 620):
        offset = torch.tensor([100.0, 1000.0, -30000.0])[torch.arange(rows) % 3][:, None]
        spread = torch.tensor([1e-1, 1e-2, 1.0])[torch.arange(rows) // 3 % 3][:, None]
        x = torch.randn(rows, cols, generator=g)
        x[:, 0] += first
        x = offset + spread * x
        for bias in (b, None):
            y, mean, rstd = pkg.layer_norm(x.cuda(), w.cuda(), None if bias is None else bias.cuda())
            want, want_mean, want_rstd = row_oracle.norm(x, w, bias, 1e-5)
            d, xs, m, r = _depth(cols), x.double(), want_mean[:, None], want_rstd[:, None]
            apart = (xs - m).abs()
            s, deviation = apart.mean(-1, keepdim=True), (apart ** 2).mean(-1, keepdim=True).sqrt()
            from_first = apart[:, :1]
            p = 1.01 * U * ((d + 5) * (s + from_first) + m.abs())
            off_e = U * (d + 5) * (s + p)
            assert ((mean.cpu().double()[:, None] - m).abs() <= 1.01 * (U * m.abs() + off_e)).all()
            var = 1 / r ** 2
            square = deviation ** 2 + p ** 2                                     # what is added up, before the correction
            off_var = U * ((d + 8) * square + 3 * var) + 2 * (p + off_e) * off_e
            off_r = off_var / var / 2 * 1.01 + 4 * U
            assert ((rstd.cpu().double()[:, None] / r - 1).abs() <= off_r).all()
            size = w.double().abs() * r
            off = size * (U * (apart + p) + off_e + U * (p + off_e) + apart * (off_r + 2 * U))
            off = 1.01 * (off + U * (size * apart + (0 if bias is None else bias.double().abs())))
            worst = ((y.cpu().double() - want).abs() / (off + U * (want.abs() + off))).max()
            assert worst <= 1, float(worst)


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
def test_layer_norm_quantize_where_the_bias_cancels_the_norm(pkg, xt, bits, wt):
    """Rows of +-1 with a bias of the opposite fp32 number, or nearly that: float32 sees zeros in the group (or digits of its own
    rounding alone), the exact norm is what the rounding of rstd leaves.  Whole rows, groups, and a short last group of two values."""
    for cols, sub in ((2, 0), (64, 0), (2048, 0), (34, 32), (130, 64), (258, 256), (1024, 128), (9002, 0), (20000, 64)):
        x = torch.ones(1, cols)
        x[:, 1::2] = -1
        x = x.to(xt)
        for eps in (1e-5, 3e-3, 0.37):
            r = torch.tensor((1 + eps) ** -0.5, dtype=torch.float64).float()
            if wt is torch.bfloat16:           # the product's weight, so that w r is near a bfloat16 number
                r = r.bfloat16().float()
            w = torch.ones(cols).to(wt)
            for part in (slice(0, cols), slice(cols - 2, cols)):
                b = torch.linspace(-2, 2, cols)
                b[part] = -r * x[0, part].float()
                _check_norm_codes(pkg, x, w, b.to(wt), bits, sub, eps=eps)


def test_two_copies_of_the_library_in_one_process(pkg, native_lib, tmp_path):
    """Kernels that need more shared memory than is given unasked get the permission in each copy."""
    import shutil

    from strix_halo_int4_gemms_b200 import native

    copy = tmp_path / "copy_of_the_library.so"
    shutil.copy(native_lib, copy)
    x, dy = [_rows(300, 2048, torch.bfloat16, seed).cuda() for seed in (71, 72)]
    w = _affine(2048, torch.bfloat16, 73)[0].cuda()
    _, mean, rstd = pkg.layer_norm(x, w)
    want = pkg.layer_norm_bwd(dy, x, w, mean, rstd)
    got = native.layer_norm_bwd_on_device(dy, x, w, mean, rstd, library_path=copy)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(2500, 8712), (1203, 14336), (1500, 16500), (700, 20000), (1029, 40000), (1500, 9001), (1200, 20001)])
def test_layer_norm_bwd_of_wide_rows(pkg, rows, cols, xt):
    """Wide rows, read 16 bytes at a time or not, in several parts that the warps of a block share."""
    x, dy, w = _rows(rows, cols, xt, cols).cuda(), (_rows(rows, cols, xt, cols + 1) / 7).cuda(), _affine(cols, torch.float32, 3)[0].cuda()
    _, mean, rstd = pkg.layer_norm(x, w)
    dx, dw, db = pkg.layer_norm_bwd(dy, x, w, mean, rstd)
    m, r = mean.double(), rstd.double()
    want_dx, want_dw, want_db = row_oracle.norm_bwd(dy, x, w, m, r)
    d = _depth(cols)
    h, g = ((x.double() - m[:, None]) * r[:, None]).abs(), (dy.double() * w.double()).abs()
    off = r[:, None] * U * (5 * g + (d + 6) * g.mean(-1, keepdim=True) + (d + 12) * h * (g * h).mean(-1, keepdim=True))   # as in _check_bwd
    assert ((dx.double() - want_dx).abs() <= 1.01 * off + HALF_STEP[xt] * (want_dx.abs() + off)).all()
    # a thread adds the rows of its warp, one in eight of its part; then the warps' eight sums, and at most six parts
    path = rows / 8 + 1 + 8 + 6
    for got, want, terms in ((dw, want_dw, (dy.double().abs() * h).sum(0)), (db, want_db, dy.double().abs().sum(0))):
        assert ((got.double() - want).abs() <= 1.01 * (path + 4) * U * terms).all()


def test_layer_norm_bwd_divides_the_rows_of_wide_rows(pkg):
    """The number of parts, by the scratch that is asked for (16 bytes a row, and 8 bytes a column for each part): enough blocks for
    the device at widths whose strips alone fill half of it, and at most 512 rows to a warp however many there are."""
    from strix_halo_int4_gemms_b200 import native

    size = native.load_dispatch_library().b200_int4_gemms_layer_norm_bwd_workspace_bytes

    def parts(rows, cols, kind):
        return (size(0, rows, cols, kind) - 16 * rows) // (8 * cols)

    for cols, kind in ((20000, native.OUT_F32), (33000, native.OUT_F32), (40000, native.OUT_BF16)):
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        strips = -(-cols // (128 if kind == native.OUT_F32 else 256))
        if sms < strips <= 1.2 * sms:
            assert parts(4096, cols, kind) >= 3, cols
    for cols in (8704, 19200, 65536):
        for kind in (native.OUT_F32, native.OUT_BF16):
            assert parts(32768, cols, kind) >= 8 and 1 <= parts(5, cols, kind) <= 2


@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [7, 264, 2048, 20000])
def test_layer_norm_mean_of_rows_that_are_not_finite(pkg, cols, xt):
    inf, nan = float("inf"), float("nan")
    x = _rows(7, cols, xt, cols)
    x[0, 0], x[1, cols - 1], x[2, 0], x[3, 1], x[4, 2] = inf, inf, -inf, -inf, nan
    x[5, 0], x[5, cols - 1] = inf, -inf
    y, mean, rstd = pkg.layer_norm(x.cuda(), torch.ones(cols, device="cuda"))
    assert mean[:4].tolist() == [inf, inf, -inf, -inf] and torch.isnan(mean[4:6]).all()
    assert torch.isnan(rstd[:6]).all() and torch.isnan(y[:6]).all() and torch.isfinite(y[6]).all() and torch.isfinite(mean[6])


def test_row_operators_beyond_2_31_values(pkg):
    """Rows whose values start more than 2^31 values into the tensor: the same as those rows alone."""
    rows, cols, some = 1_100_000, 2048, 300
    g = torch.Generator(device="cuda").manual_seed(81)
    x, dy = [torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    for t in (x, dy):
        t[-some:] = torch.randn(some, cols, device="cuda", generator=g).bfloat16()
    w, b = [t.cuda() for t in _affine(cols, torch.bfloat16, 82)]
    last = x[-some:].clone()
    y, mean, rstd = pkg.layer_norm(x, w, b)
    # 300 rows have another launch shape and order of sums than many: each side is within its bounds of the exact row.  Those of
    # _check_norm with at most _depth additions, |x - m| below 6 deviations, deviations of about 1 and weights below 3: mean
    # off by (d + 5) U (2 mean |x|), rstd by (d / 2 + 16) U, y by less than 60 * 6 * 3 U = 2^-13 and half a step of bfloat16.
    y1, mean1, rstd1 = [t.double() for t in pkg.layer_norm(last, w, b)]
    d = _depth(cols)
    assert ((mean[-some:].double() - mean1).abs() <= 2 * (d + 5) * U * 2 * last.double().abs().mean(-1)).all()
    assert ((rstd[-some:].double() / rstd1 - 1).abs() <= 2 * (d / 2 + 16) * U).all()
    assert ((y[-some:].double() - y1).abs() <= 2 * (2.0 ** -8 * y1.abs() * 1.01 + 2.0 ** -13)).all()
    dx, dw, db = pkg.layer_norm_bwd(dy, x, w, mean, rstd)
    alone = pkg.layer_norm_bwd(dy[-some:].clone(), last, w, mean[-some:].clone(), rstd[-some:].clone())
    assert torch.equal(dx[-some:], alone[0]) and not dx[:-some].any()
    # the other rows have no gradient: the same sums but for the order of 300 additions, and a rounding or two of each term
    tail = dy[-some:].double().abs()
    h = ((last.double() - mean[-some:, None].double()) * rstd[-some:, None].double()).abs()
    for got, want, terms in ((dw, alone[1], (tail * h).sum(0)), (db, alone[2], tail.sum(0))):
        assert ((got.double() - want.double()).abs() <= 2 * 1.01 * (some + 4) * U * terms).all()
    del y, dx
    for call in (pkg.quantize_tokens, lambda t, **kw: pkg.layer_norm_quantize(t, w, b, **kw)):
        for bits, sub in ((4, 0), (8, 64)):
            kw = dict(dtype=_dtype(pkg, bits), scale=_spec(pkg, sub))
            for got, want in zip(call(x, **kw), call(last, **kw)):
                assert torch.equal(got[-some:], want)


def test_row_operators_from_two_host_threads(pkg):
    import threading

    w, b = [t.cuda() for t in _affine(1000, torch.float32, 91)]
    xs = [_rows(200 + 100 * i, 1000, torch.float32, 92 + i).cuda() for i in range(2)]

    def step(x):
        y, mean, rstd = pkg.layer_norm(x, w, b)
        return (y, *pkg.layer_norm_bwd(x, x, w, mean, rstd), *pkg.quantize_tokens(x.bfloat16()), *pkg.layer_norm_quantize(x, w, b))

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                got = step(xs[i])
                stream.synchronize()
                if not all(torch.equal(a, c) for a, c in zip(got, want[i])):
                    failed.append(i)
                try:                                  # a refusal's message belongs to its thread
                    pkg.layer_norm(xs[i], w[: 999 - i], b)
                    failed.append(i)
                except ValueError as refusal:
                    if "(1000,)" not in str(refusal) or str(999 - i) not in str(refusal):
                        failed.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
