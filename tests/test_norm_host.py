"""Layer norm and the quantiser for each token without a GPU: the oracle against differences, and every refusal of the
Python entry points and of the C ABI (nothing is launched)."""
import ctypes

import pytest
import torch

import row_oracle


def test_oracle_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 7, generator=g, dtype=torch.float64)
    w = torch.randn(7, generator=g, dtype=torch.float64)
    b = torch.randn(7, generator=g, dtype=torch.float64)
    dy = torch.randn(3, 7, generator=g, dtype=torch.float64)
    _, mean, rstd = row_oracle.norm(x, w, b, 1e-5)
    dx, dw, db = row_oracle.norm_bwd(dy, x, w, mean, rstd)

    def loss(x, w, b):
        return float((row_oracle.norm(x, w, b, 1e-5)[0] * dy).sum())

    step = 1e-6   # differences of second order: error about step^2 * third derivative + 1e-16 / step, below 1e-8
    for tensor, grad, place in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        flat = tensor.flatten()
        for i in range(flat.numel()):
            up, down = flat.clone(), flat.clone()
            up[i] += step
            down[i] -= step
            args = [x, w, b]
            args[place] = up.view_as(tensor)
            high = loss(*args)
            args[place] = down.view_as(tensor)
            assert abs((high - loss(*args)) / (2 * step) - float(grad.flatten()[i])) < 1e-7


def test_oracle_rounding_to_bf16():
    v = torch.tensor([1.0, 1.00390625, 1.01171875, 1.00390625 + 1e-12, -3.0078125, 0.0, 2.0 ** -140], dtype=torch.float64)
    want = torch.tensor([1.0, 1.0, 1.015625, 1.0078125, -3.0, 0.0, 0.0], dtype=torch.float64)
    assert torch.equal(row_oracle.round_bf16(v), want)
    some = torch.randn(4096, dtype=torch.float32)      # float32 values are exact in float64: torch rounds them once too
    assert torch.equal(row_oracle.round_bf16(some).float(), some.bfloat16().float())


def test_oracle_codes_of_special_rows():
    inf = float("inf")
    v = torch.tensor([[0.0, 0.0], [inf, 1.0], [float("nan"), 1.0], [7.0, 0.5], [-14.0, 3.0]])
    codes, scales, _ = row_oracle.quantize_rows(v, 4)
    assert codes.tolist() == [[0, 0], [0, 0], [0, 0], [7, 0], [-7, 2]]
    assert scales[0] == 1 and scales[1] == inf and torch.isnan(scales[2]) and scales[3] == 1 and scales[4] == 2


@pytest.mark.parametrize("fn", ["layer_norm", "layer_norm_quantize"])
def test_norm_refusals(pkg, fn):
    call = getattr(pkg, fn)
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        call([1.0], w)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        call(x, w)
    if not torch.cuda.is_available():
        return
    x, w = x.cuda(), w.cuda()
    for bad, why in (((x.half(), w), "dtype"), ((x.t(), w), "contiguous"), ((x, w[:7]), "shape"), ((x, w.half()), "dtype"),
                     ((x, w, w.bfloat16()), "dtype of weight"), ((x, w.cpu()), "CUDA"), ((x[:, :0], w), "at least one"),
                     ((torch.zeros((), device="cuda"), w), "at least one")):
        with pytest.raises(ValueError, match=why):
            call(*bad)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            call(x, w, eps=eps)
    for eps in ("1", True, None):
        with pytest.raises(TypeError, match="eps"):
            call(x, w, eps=eps)


def test_quantize_tokens_refusals(pkg):
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        pkg.quantize_tokens(3)
    with pytest.raises(TypeError, match="OperandDType"):
        pkg.quantize_tokens(x, dtype="int4")
    with pytest.raises(ValueError, match="at least one value"):
        pkg.quantize_tokens(torch.zeros(4, 0, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="CUDA bfloat16"):
        pkg.quantize_tokens(x)


def test_norm_bwd_refusals(pkg):
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        pkg.layer_norm_bwd(x, x, torch.ones(8), torch.zeros(4), torch.zeros(4))


def test_c_entry_points_check_arguments(pkg, native_lib):
    from strix_halo_int4_gemms_b200 import native

    lib = native.load_dispatch_library()

    def said(rc):
        assert rc == 1
        return lib.b200_int4_gemms_last_error().decode()

    p = 4096
    q = lib.b200_int4_gemms_quantize_tokens
    assert said(q(0, 0, p, p, p, -1, 8, 4, 0)) == "rows must be non-negative"
    assert said(q(0, 0, p, p, p, 1, 0, 4, 0)) == "cols must be positive"
    assert said(q(0, 0, p, p, p, 1, 2 ** 31, 4, 0)) == "too many columns for one launch"
    assert said(q(0, 0, p, p, p, 1, 8, 5, 0)) == "bits must be 4 or 8"
    assert "subchannel must be" in said(q(0, 0, p, p, p, 1, 8, 4, 48))
    assert said(q(0, 0, None, p, p, 1, 8, 4, 0)) == "src, codes and scales pointers must be non-null"
    assert said(q(0, 0, p + 1, p, p, 1, 8, 4, 0)) == "src is not aligned to its element size"
    assert said(q(99, 0, p, p, p, 1, 8, 4, 0)) == "device_index out of range"
    assert q(0, 0, None, None, None, 0, 8, 4, 0) == 0
    n = lib.b200_int4_gemms_layer_norm
    assert said(n(0, 0, p, p, p, p, p, p, 1, 8, 2, 0, 1e-5)) == "x and weight types must be bf16 or float32"
    assert said(n(0, 0, p, p, p, p, p, p, 1, 8, 0, 0, -1.0)) == "eps must be non-negative"
    assert said(n(0, 0, p, p, p, p, p, p, 1, 8, 0, 0, float("nan"))) == "eps must be non-negative"
    assert said(n(0, 0, p, None, p, p, p, p, 1, 8, 0, 0, 1e-5)) == "x, weight, y, mean and rstd pointers must be non-null"
    assert said(n(0, 0, p + 2, p, p, p, p, p, 1, 8, 1, 0, 1e-5)) == "x is not aligned to its element size"
    assert n(0, 0, None, None, None, None, None, None, 0, 8, 0, 0, 1e-5) == 0
    nq = lib.b200_int4_gemms_layer_norm_quantize
    assert said(nq(0, 0, p, p, p, p, p, 1, 8, 0, 0, 1e-5, 3, 0)) == "bits must be 4 or 8"
    assert said(nq(0, 0, p, p, p, None, p, 1, 8, 0, 0, 1e-5, 4, 0)) == "x, weight, codes and scales pointers must be non-null"
    b = lib.b200_int4_gemms_layer_norm_bwd
    assert said(b(0, 0, p, p, p, p, p, p, None, p, p, 8, 1, 8, 0, 0)) == "dweight and dbias pointers must be non-null"
    assert said(b(0, 0, None, p, p, p, p, p, p, p, p, 8, 1, 8, 0, 0)) == "dy, x, weight, mean, rstd and dx pointers must be non-null"
    assert lib.b200_int4_gemms_layer_norm_bwd_workspace_bytes(99, 1, 8, 0) == 0


def test_a_failed_size_of_the_backward_scratch_is_not_kept(pkg):
    from strix_halo_int4_gemms_b200 import native

    class Library:
        """What the library answers while the device cannot be asked, and afterwards."""

        def __init__(self):
            self.answers, self.calls = [0, 4096], 0

        def b200_int4_gemms_layer_norm_bwd_workspace_bytes(self, *fields):
            self.calls += 1
            return self.answers[min(self.calls, 2) - 1]

        @staticmethod
        def b200_int4_gemms_last_error():
            return b"the device did not answer"

    library = Library()
    with pytest.raises(RuntimeError, match="the device did not answer"):
        native._layer_norm_bwd_workspace(library, 0, 8, 16, native.OUT_F32)
    assert native._layer_norm_bwd_workspace(library, 0, 8, 16, native.OUT_F32) == 4096
    assert native._layer_norm_bwd_workspace(library, 0, 8, 16, native.OUT_F32) == 4096 and library.calls == 2
    library.answers, library.calls = [0, 0], 0
    assert native._layer_norm_bwd_workspace(library, 0, 0, 16, native.OUT_F32) == 0     # no rows, no scratch


def test_layer_norm_refuses_an_eps_that_float32_has_no_room_for(pkg, native_lib):
    from strix_halo_int4_gemms_b200 import native

    lib = native.load_dispatch_library()
    for eps in (1e-50, 1e300, float("inf")):
        assert lib.b200_int4_gemms_layer_norm(0, 0, 4096, 4096, 4096, 4096, 4096, 4096, 1, 8, 0, 0, eps) == 1
        assert lib.b200_int4_gemms_last_error() == b"eps must be zero or within the range of float32"
    for eps in (0.0, 1e-45, 1e-38, 3e38):
        assert lib.b200_int4_gemms_layer_norm(0, 0, None, None, None, None, None, None, 0, 8, 0, 0, eps) == 0
    if torch.cuda.is_available():
        x, w = torch.zeros(2, 8, device="cuda"), torch.ones(8, device="cuda")
        for eps in (1e-50, 1e300):
            with pytest.raises(ValueError, match="within the range of float32"):
                pkg.layer_norm(x, w, eps=eps)
            pkg.layer_norm_quantize(x, w, eps=eps)        # adds it in float64
        assert not pkg.layer_norm(x, w, eps=1e-45)[0].any()
