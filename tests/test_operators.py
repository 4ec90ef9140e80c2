"""CPU tests of the operators' entry points: what they refuse before a GPU is
touched, and the MXFP4 row sizes."""
import ctypes

import pytest

import doantotnghiepmoe_b200 as M
from doantotnghiepmoe_b200 import _lib
from doantotnghiepmoe_b200.layer import mxfp4_strides


def test_mxfp4_row_sizes():
    L = M.lib()
    for k, codes, scales in ((1, 16, 4), (32, 16, 4), (33, 32, 4), (128, 64, 4), (129, 80, 8),
                             (2048, 1024, 64), (0, 0, 0), (-5, 0, 0)):
        assert L.moe_mxfp4_code_stride(k) == codes
        assert L.moe_mxfp4_scale_stride(k) == scales
        assert k < 1 or mxfp4_strides(k) == (codes, scales)


def test_null_arguments_are_refused():
    L, p = M.lib(), ctypes.c_void_p(256)  # never dereferenced
    d, n = _lib.MoeGroupedDesc(), _lib.MoeBlockNormDesc()
    bad = _lib.MOE_ERR_INVALID
    assert L.moe_get_stream(None) is None
    for f in (L.moe_grouped_mm, L.moe_grouped_mm_dgrad, L.moe_grouped_mm_wgrad):
        assert f(None, ctypes.byref(d), p, p, p, p, None) == bad
    assert L.moe_mxfp4_quantize(None, p, 4, 32, 1, None, 1, 32, p, p, None) == bad
    assert L.moe_mxfp4_dequantize(None, p, p, 1, 32, p, 4, 32, None) == bad
    assert L.moe_grouped_mm_mxfp4(None, 1, 1, 1, 32, p, p, p, p, p, p, 4, 1, None) == bad
    assert L.moe_block_norm(None, ctypes.byref(n), p, p, p, p, p, p, p, None) == bad
    assert L.moe_block_norm_backward_workspace(None, 1, 8) == 0
    assert L.moe_block_norm_backward(None, ctypes.byref(n), p, p, p, p, p, p, p, p, p, p, p, p, p,
                                     8, None) == bad


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    eng = M.MoeLayerEngine.__new__(M.MoeLayerEngine)  # no handle: the checks come first
    eng._h, eng.device, eng._dev = None, 0, torch.device("cuda", 0)
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: eng.grouped_mm(x, w, off, x), lambda: eng.grouped_mm_dgrad(x, w, off, x),
                 lambda: eng.grouped_mm_wgrad(x, x, off, w),
                 lambda: eng.mxfp4_quantize(x, x, x), lambda: eng.mxfp4_dequantize(x, x, x),
                 lambda: eng.grouped_mm_mxfp4(x, x, x, x, off, 8, x),
                 lambda: eng.block_norm(x, x, x), lambda: eng.block_norm_backward(x, x, x, None, x)):
        with pytest.raises(M.MoeError) as e:
            call()
        assert e.value.status == _lib.MOE_ERR_INVALID


def test_a_single_row_has_no_stride():
    """The stride that torch gives a one-row tensor addresses nothing: whatever it
    is, it agrees with other tensors' and keeps 16-byte accesses."""
    torch = pytest.importorskip("torch")
    eng = M.MoeLayerEngine.__new__(M.MoeLayerEngine)  # no handle: only the checks run
    eng.device, eng._dev = 0, torch.device("cpu")
    bf = torch.bfloat16
    wide, near = torch.zeros(4, 100)[:1, :33], torch.zeros(1, 33)
    assert wide.stride(0) == 100 and near.stride(0) == 33
    assert eng._norm_kind(1, 33, ("x", wide), ("x_out", near), ("none", None)) == (4, 40)
    with pytest.raises(M.MoeError):
        eng._norm_kind(2, 33, ("x", torch.zeros(4, 100)[:2, :33]), ("x_out", torch.zeros(2, 33)))
    off, out = torch.zeros(3, dtype=torch.int32), torch.zeros(1, 16)
    d = eng._grouped(torch.zeros(4, 101, dtype=bf)[:1, :24], out,
                     torch.zeros(2, 16, 24, dtype=bf), off, out)
    assert (d.rows, d.ld_x, d.ld_w, d.ld_out, d.expert_stride) == (1, 24, 24, 16, 384)
    row = torch.zeros(2, 3, 32, dtype=bf)[:, :1, :24]  # experts of one row
    out = torch.zeros(5, 1)
    d = eng._grouped(torch.zeros(5, 24, dtype=bf), out, row.as_strided((2, 1, 24), (96, 7, 1)),
                     off, out)
    assert (d.n, d.ld_w, d.expert_stride, d.ld_out) == (1, 24, 96, 1)
