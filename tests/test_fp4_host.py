"""The 4-bit operators without a GPU: sizes of packed operands, refusals of the C ABI (they come before any CUDA call),
and the 64-bit reference that the GPU tests compare with, pinned by hand-computed values."""
import ctypes

import numpy as np
import pytest

import fp4_reference as ref

P = ctypes.c_void_p
A = 0x1000   # a non-null, aligned address that a refused call never touches


def test_packed_sizes(cuda_lib):
    for k in (1, 15, 16, 31, 32, 33, 64, 1000, 1536):
        assert cuda_lib.vrb_fp4_row_bytes(k) == ref.row_bytes(k)
        for rows in (1, 127, 128, 129, 1000):
            for fmt in (0, 1):
                assert cuda_lib.vrb_fp4_scale_bytes(fmt, rows, k) == ref.scale_bytes(fmt, rows, k)
    assert cuda_lib.vrb_fp4_row_bytes(0) == 0 and cuda_lib.vrb_fp4_row_bytes(-5) == 0
    assert cuda_lib.vrb_fp4_scale_bytes(2, 4, 4) == 0 and cuda_lib.vrb_fp4_scale_bytes(0, 0, 4) == 0
    rows, k = 300, 500   # every (row, block) has a byte of its own inside the buffer
    at = ref.scale_index(np.arange(rows)[:, None], np.arange(32)[None, :], 32)
    assert len(np.unique(at)) == at.size and at.max() < ref.scale_bytes(0, rows, k)


def test_reference_known_values():
    x = np.zeros((1, 32))
    x[0, :9] = [6.0, 5.0, 2.5, -0.25, 0.75, 3.5, -1.25, 0.2, 1.75]
    codes, scales = ref.quantize(x, ref.MXFP4)          # largest magnitude 6: scale 2^(2 - 2) = 1
    assert scales[0] == 127
    got = ref.values(codes, scales, ref.MXFP4, 1, 32)[0, :9]
    assert got.tolist() == [6.0, 4.0, 2.0, 0.0, 1.0, 4.0, -1.0, 0.0, 2.0]   # every border goes to the even code
    codes, scales = ref.quantize(x[:, :16] * 4.5, ref.NVFP4, 0.5)     # 27 / (6 * .5) = 9 = 1.125 * 2^3
    assert ref.E4M3[scales[0]] == 9.0
    assert np.array_equal(ref.values(codes, scales, ref.NVFP4, 1, 16, 0.5)[0, :9], 4.5 * np.array(got))
    codes, scales = ref.quantize(np.full((1, 32), 7.9), ref.MXFP4)    # saturates: scale 1, element 6
    assert scales[0] == 127 and (ref.values(codes, scales, ref.MXFP4, 1, 32) == 6.0).all()


def _status(lib, name, *args):
    return getattr(lib, name)(*args), lib.vrb_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    ({"format": 2}, -1, "unknown 4-bit format"),
    ({"x": None}, -1, "null tensor"),
    ({"codes": None}, -1, "null tensor"),
    ({"scales": None}, -1, "null tensor"),
    ({"dtype": 5}, -2, "dtype must be F32 or BF16"),
    ({"rows": 0}, -1, "must be positive"),
    ({"k": 0}, -1, "must be positive"),
    ({"rows": 1 << 30, "k": 1 << 30}, -1, "at most 2^40"),
    ({"codes": A + 8}, -1, "16-byte aligned"),
    ({"scales": A + 4}, -1, "16-byte aligned"),
    ({"format": 1, "scale": A}, -1, "MXFP4 has no tensor scale"),
    ({"scale": A + 2}, -1, "aligned to their elements"),
    ({"x": A + 1}, -1, "aligned to their elements"),
    ({"x": A + 2, "dtype": 0}, -1, "aligned to their elements"),
])
def test_quantize_refusals(cuda_lib, change, code, text):
    a = {"format": 0, "x": A, "dtype": 2, "scale": None, "codes": A, "scales": A, "rows": 4, "k": 64} | change
    rc, why = _status(cuda_lib, "vrb_fp4_quantize", a["format"], a["x"], a["dtype"], a["scale"], a["codes"], a["scales"], a["rows"], a["k"], None)
    assert rc == code and text in why
    if change.get("x", A) is not None:
        rc, why = _status(cuda_lib, "vrb_fp4_dequantize", a["format"], a["codes"], a["scales"], a["scale"], a["x"], a["dtype"], a["rows"], a["k"], None)
        assert rc == code and text in why


def test_tensor_scale_refusals(cuda_lib):
    for args, code in (((None, 2, 4, A, None), -1), ((A, 2, 4, None, None), -1), ((A, 5, 4, A, None), -2), ((A, 2, 0, A, None), -1),
                       ((A + 1, 2, 4, A, None), -1), ((A, 2, 4, A + 2, None), -1)):
        assert cuda_lib.vrb_fp4_tensor_scale(*args) == code


@pytest.mark.parametrize("change,code,text", [
    ({"format": -1}, -1, "unknown 4-bit format"),
    ({"ac": None}, -1, "null tensor"), ({"as": None}, -1, "null tensor"), ({"bc": None}, -1, "null tensor"),
    ({"bs": None}, -1, "null tensor"), ({"out": None}, -1, "null tensor"),
    ({"odt": 5}, -2, "F32 or BF16"), ({"bias": A, "bdt": 5}, -2, "F32 or BF16"),
    ({"m": 0}, -1, "must be positive"), ({"n": -1}, -1, "must be positive"), ({"k": 0}, -1, "must be positive"),
    ({"m": 1 << 31}, -1, "below 2^31"), ({"n": 1 << 31}, -1, "below 2^31"), ({"k": 1 << 31}, -1, "below 2^31"),
    ({"format": 1, "ag": A}, -1, "MXFP4 has no tensor scale"), ({"format": 1, "bg": A}, -1, "MXFP4 has no tensor scale"),
    ({"act": 5}, -1, "unknown activation"), ({"act": -2}, -1, "unknown activation"),
    ({"ac": A + 8}, -1, "16-byte aligned"), ({"bs": A + 8}, -1, "16-byte aligned"),
    ({"out": A + 1}, -1, "aligned to their elements"), ({"bias": A + 2, "bdt": 0}, -1, "aligned to their elements"),
    ({"ag": A + 1}, -1, "aligned to their elements"), ({"bg": A + 2}, -1, "aligned to their elements"),
    ({"m": 1 << 30, "n": 1 << 30}, -1, "at most 2^40 elements"),
])
def test_linear_refusals(cuda_lib, change, code, text):
    a = {"format": 0, "ac": A, "as": A, "ag": None, "m": 4, "bc": A, "bs": A, "bg": None, "n": 8, "k": 64, "bias": None, "bdt": 0, "act": -1,
         "out": A, "odt": 2} | change
    rc, why = _status(cuda_lib, "vrb_fp4_linear", *[a[n] for n in ("format", "ac", "as", "ag", "m", "bc", "bs", "bg", "n", "k", "bias", "bdt", "act", "out", "odt")], None)
    assert rc == code and text in why


@pytest.mark.parametrize("change,code,text", [
    ({"x": None}, -1, "null tensor"), ({"out": None}, -1, "null tensor"), ({"dtype": 5}, -2, "F32 or BF16"),
    ({"w": A, "wdt": 5}, -2, "F32 or BF16"), ({"b": A, "bdt": 3}, -2, "F32 or BF16"),
    ({"act": 5}, -1, "unknown activation"), ({"act": -2}, -1, "unknown activation"),
    ({"batch": 0}, -1, "shape/groups mismatch"), ({"spatial": 0}, -1, "shape/groups mismatch"), ({"channels": 0}, -1, "shape/groups mismatch"),
    ({"groups": 0}, -1, "shape/groups mismatch"), ({"groups": 3}, -1, "shape/groups mismatch"),
    ({"channels": 1 << 25}, -1, "exceeds CUDA grid capacity"), ({"spatial": 1 << 40}, -1, "exceeds CUDA grid capacity"),
    ({"x": A + 1}, -1, "aligned to their elements"), ({"out": A + 2, "dtype": 0}, -1, "aligned to their elements"),
    ({"w": A + 2}, -1, "aligned to their elements"), ({"b": A + 1, "bdt": 2}, -1, "aligned to their elements"),
    ({"spatial": 1 << 20, "ws": None}, -4, "workspace needs"), ({"spatial": 1 << 20, "size": 16}, -4, "workspace needs"),
    ({"spatial": 1 << 20, "ws": A + 16}, -4, "workspace needs"),
])
def test_group_norm_channels_last_refusals(cuda_lib, change, code, text):
    a = {"x": A, "dtype": 2, "w": None, "wdt": 0, "b": None, "bdt": 0, "out": A, "batch": 2, "spatial": 64, "channels": 64, "groups": 32, "act": -1,
         "ws": A, "size": 1 << 40} | change
    rc, why = _status(cuda_lib, "vrb_group_norm_channels_last", a["x"], a["dtype"], a["w"], a["wdt"], a["b"], a["bdt"], a["out"], a["batch"], a["spatial"],
                      a["channels"], a["groups"], ctypes.c_float(1e-5), a["act"], a["ws"], a["size"], None)
    assert rc == code and text in why
