"""The expert layer without a GPU: record layout, refusals of the Python entry point and of the C ABI."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

HEADER = Path(__file__).resolve().parent.parent / "include" / "b200_int4_gemms.h"


def test_problem_record_and_limits_match_the_header(pkg):
    from strix_halo_int4_gemms_b200 import moe
    from strix_halo_int4_gemms_b200.native import MoeProblem

    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct b200_moe_problem \{(.*?)\}", text, flags=re.S).group(1)
    assert re.findall(r"int32_t\s+(\w+);", body) == [name for name, _ in MoeProblem._fields_]
    for name, value in (("TOKENS", moe.MOE_MAX_TOKENS), ("TOP_K", moe.MOE_MAX_TOP_K), ("EXPERTS", moe.MOE_MAX_EXPERTS)):
        assert f"#define B200_MOE_MAX_{name} {value}" in text


def test_refusals_before_any_device_work(pkg):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w = torch.zeros(4, 32, 128, dtype=torch.uint8)
    call = dict(up_gate_scale=torch.ones(4, 128), down_scale=torch.ones(4, 64))
    with pytest.raises(TypeError, match="OperandDType"):
        pkg.moe_swiglu(x, w, w, dtype="int4", **call)
    with pytest.raises(TypeError, match="GemmLayout"):
        pkg.moe_swiglu(x, w, w, layout="nn", **call)
    with pytest.raises(ValueError, match="supports layouts nn and nt"):
        pkg.moe_swiglu(x, w, w, layout=pkg.GemmLayout.TN, **call)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        pkg.moe_swiglu(x, w, w, **call)
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        pkg.moe_swiglu(None, w, w, **call)


def test_c_entry_point_checks_arguments(pkg, native_lib):
    from strix_halo_int4_gemms_b200 import native

    lib = native.load_dispatch_library()

    def problem(**changes):
        fields = dict(dtype=0, layout=0, subchannel=0, tokens=2, hidden=64, inner=32, experts=4, top_k=2, router_type=0, renormalize=1, ids_bits=32)
        fields.update(changes)
        return native.MoeProblem(**fields)

    def said(record, pointers=None, workspace=(4096, 1 << 30)):
        a = [4096] * 9 if pointers is None else pointers
        rc = lib.b200_int4_gemms_moe_swiglu(None if record is None else ctypes.byref(record), 0, 0, *a, *workspace)
        return rc, lib.b200_int4_gemms_last_error().decode()

    assert said(None) == (1, "problem must be non-null")
    for changes, why in (
        (dict(dtype=2), "problem.dtype"), (dict(layout=2), "problem.layout must be NN or NT"), (dict(subchannel=16), "problem.subchannel"),
        (dict(tokens=65), "tokens must be at most 64"), (dict(tokens=-1), "tokens must be at most 64"), (dict(experts=0), "experts must be in"),
        (dict(experts=1025), "experts must be in"), (dict(top_k=0), "top_k must be in"), (dict(top_k=5), "top_k must be in"),
        (dict(top_k=17, experts=32), "top_k must be in"), (dict(hidden=48), "multiples of 32"), (dict(inner=0), "multiples of 32"),
        (dict(hidden=131072), "below 131072"), (dict(router_type=2), "router weights"), (dict(ids_bits=16), "ids must have"),
    ):
        rc, message = said(problem(**changes))
        assert rc == 1 and why in message, changes
        assert lib.b200_int4_gemms_moe_swiglu_workspace_bytes(ctypes.byref(problem(**changes))) == 0
    for hole in (0, 4, 5, 6, 7, 8):
        pointers = [4096] * 9
        pointers[hole] = None
        assert said(problem(), pointers) == (1, "x, weight, scale and out pointers must be non-null")
    pointers = [4096, None, None] + [4096] * 6
    assert "either router weights or" in said(problem(), pointers)[1]
    pointers = [4096] * 9
    pointers[4] = 4100
    assert said(problem(), pointers)[1] == "x, weight and scale pointers must be 16-byte aligned"
    assert "written as int32" in said(problem(ids_bits=64))[1]
    assert said(problem(tokens=0), [None] * 9, (None, 0))[0] == 0
    # scratch of the documented size: everything a pair and a token need, each part rounded up to 256 bytes
    need = lib.b200_int4_gemms_moe_swiglu_workspace_bytes(ctypes.byref(problem(tokens=64, hidden=2048, inner=1408, experts=64, top_k=8)))
    pairs = 512
    want = 64 * 1024 + 64 * 64 * 8 + pairs * (1408 * 8 + 704 + 2048 * 4)
    assert want <= need <= want + 16 * 1024
