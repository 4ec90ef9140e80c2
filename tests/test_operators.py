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
