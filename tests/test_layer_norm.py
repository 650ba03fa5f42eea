"""layer_norm: what is refused, before any launch (no GPU)."""

import ctypes

import pytest
import torch

from model_amd import _lib
from model_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward


@pytest.mark.parametrize("x,scale,bias,residual,match", [
    (torch.zeros(4, 8), torch.zeros(9), torch.zeros(8), None, "scale"),
    (torch.zeros(4, 8), torch.zeros(8), torch.zeros(1, 8), None, "bias"),
    (torch.zeros(4, 8), torch.zeros(8), torch.zeros(8, dtype=torch.float16), None, "bias"),
    (torch.zeros(4, 8, dtype=torch.float16), torch.zeros(8, dtype=torch.bfloat16), torch.zeros(8), None, "scale"),
    (torch.zeros(4, 8, dtype=torch.float64), torch.zeros(8), torch.zeros(8), None, "float32, float16 or bfloat16"),
    (torch.zeros(()), torch.zeros(1), torch.zeros(1), None, "rows of shape"),
    (torch.zeros(4, 0), torch.zeros(0), torch.zeros(0), None, "rows of shape"),
    (torch.zeros(2, 16385), torch.zeros(16385), torch.zeros(16385), None, "at most 16384"),
    (torch.zeros(4, 8), torch.zeros(8), torch.zeros(8), torch.zeros(3, 8), "residual"),
    (torch.zeros(4, 8), torch.zeros(8), torch.zeros(8), torch.zeros(4, 8, dtype=torch.float16), "residual"),
    (torch.zeros(4, 8), torch.zeros(8), torch.zeros(8), None, "on the GPU only"),
])
def test_refused(x, scale, bias, residual, match):
    for f in (layer_norm, layer_norm_forward):
        with pytest.raises(ValueError, match=match):
            f(x, scale, bias, residual=residual)


def test_backward_refused():
    s, w, st = torch.zeros(4, 8), torch.zeros(8), torch.zeros(4)
    with pytest.raises(ValueError, match="g_y"):
        layer_norm_backward(torch.zeros(4, 7), s, w, st, st)
    with pytest.raises(ValueError, match="g_residual"):
        layer_norm_backward(s, s, w, st, st, g_residual=torch.zeros(4, 8, dtype=torch.float16))
    with pytest.raises(ValueError, match="on the GPU only"):
        layer_norm_backward(s, s, w, st, st)


def test_c_entries_validate_before_launch():
    L = _lib.lib()
    one = ctypes.c_void_p(4096)  # never read: every call below is refused

    def fwd(x=one, xp=8, r=None, rp=0, dtype=0, w=one, b=one, pdt=0, rows=4, d=8, y=one, s=None, mean=one, rstd=one):
        return L.mpl_layer_norm(x, xp, r, rp, dtype, w, b, pdt, rows, d, 1e-6, y, s, mean, rstd, None)

    def bwd(dy=one, dyp=8, x=one, xp=8, r=None, rp=0, dtype=0, w=one, pdt=0, mean=one, rstd=one, rows=4, d=8, dx=one,
            ds=one, db=one, ws=one, n=1 << 20):
        return L.mpl_layer_norm_bwd(dy, dyp, x, xp, r, rp, dtype, w, pdt, mean, rstd, rows, d, dx, ds, db, ws, n, None)

    assert fwd(rows=0) == _lib.MPL_OK
    for f in (fwd, bwd):
        assert f(rows=-1) == _lib.MPL_EINVAL and f(d=0) == _lib.MPL_EINVAL and f(dtype=5) == _lib.MPL_EINVAL
        assert f(pdt=1) == _lib.MPL_EINVAL and b"parameters" in L.mpl_last_error()
        assert f(d=16385, xp=16385) == _lib.MPL_EUNSUPPORTED
        assert f(x=None) == _lib.MPL_EINVAL and f(w=None) == _lib.MPL_EINVAL
        assert f(xp=7) == _lib.MPL_EINVAL and b"pitch" in L.mpl_last_error()
        assert f(r=one, rp=3) == _lib.MPL_EINVAL
        assert f(x=ctypes.c_void_p(4098)) == _lib.MPL_EINVAL and b"aligned" in L.mpl_last_error()
    assert fwd(y=None) == _lib.MPL_EINVAL and fwd(rstd=None) == _lib.MPL_EINVAL
    assert fwd(s=one) == _lib.MPL_EINVAL and b"sum without residual" in L.mpl_last_error()
    assert bwd(rows=0) == _lib.MPL_EINVAL and bwd(mean=None) == _lib.MPL_EINVAL
    assert bwd(dx=None, ds=None, db=None) == _lib.MPL_EINVAL
    assert bwd(ws=None) == _lib.MPL_EINVAL and bwd(n=8) == _lib.MPL_EWORKSPACE
    for dtype in (0, 1, 2):
        assert L.mpl_layer_norm_bwd_workspace_bytes(100, 300, dtype) >= 2 * 300 * 4
        assert L.mpl_layer_norm_bwd_workspace_bytes(0, 300, dtype) == 0
        assert L.mpl_layer_norm_bwd_workspace_bytes(4, 16385, dtype) == 0
