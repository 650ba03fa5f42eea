"""clip_global_norm and global_norm_scale: what is refused, before any launch (no GPU)."""

import ctypes

import pytest
import torch

from model_amd import _lib
from model_amd.grad_clip import clip_global_norm, global_norm_scale


@pytest.mark.parametrize("grads,clip,row_sq,match", [
    ([], 1.0, None, "no gradients"),
    ([torch.zeros(4)], -1.0, None, "negative"),
    ([torch.zeros(4)], float("nan"), None, "negative"),
    ([torch.zeros(4), torch.zeros(4, dtype=torch.float64)], 1.0, None, "gradient 1 must be"),
    ([torch.zeros(4, dtype=torch.int32)], 1.0, None, "gradient 0 must be"),
    ([torch.zeros(4).to_sparse()], 1.0, None, "gradient 0 must be"),
    ([torch.zeros(4), torch.zeros(4, device="meta")], 1.0, None, "gradient 1 on meta"),
    ([torch.zeros(4)], 1.0, torch.zeros(4, dtype=torch.float16), "row_sq"),
    ([torch.zeros(4)], 1.0, torch.zeros(4, device="meta"), "row_sq"),
    ([torch.zeros(4)], 1.0, None, "on the GPU only"),
    ([], 1.0, torch.zeros(4), "on the GPU only"),
])
def test_refused(grads, clip, row_sq, match):
    for f in (clip_global_norm, global_norm_scale):
        with pytest.raises(ValueError, match=match):
            f(grads, clip, row_sq=row_sq)


def test_refused_in_place():
    with pytest.raises(ValueError, match="expanded"):
        clip_global_norm([torch.zeros(1).expand(4)], 1.0)
    with pytest.raises(ValueError, match="requires grad"):
        clip_global_norm([torch.zeros(4, requires_grad=True)], 1.0)
    with pytest.raises(ValueError, match="on the GPU only"):
        global_norm_scale([torch.zeros(1).expand(4), torch.zeros(4, requires_grad=True)], 1.0)
    with pytest.raises(TypeError):
        clip_global_norm([None], 1.0)


def test_c_entry_validates_before_launch():
    L = _lib.lib()
    one = 4096  # never read: every call below is refused

    def call(x=(one,), n=(4,), dtype=(0,), count=None, row_sq=None, rows=0, out=one, ws=one, wsb=1 << 20):
        m = len(x)
        return L.mpl_clip_grads((ctypes.c_void_p * m)(*x), (ctypes.c_int64 * m)(*n), (ctypes.c_int * m)(*dtype),
                                m if count is None else count, row_sq, rows, 1.0, 1, out, ws, wsb, None)

    assert call(count=-1) == _lib.MPL_EINVAL and call(rows=-1) == _lib.MPL_EINVAL
    assert call(rows=4) == _lib.MPL_EINVAL and call(row_sq=4098, rows=4) == _lib.MPL_EINVAL
    assert call(out=None) == _lib.MPL_EINVAL
    assert call(dtype=(3,)) == _lib.MPL_EINVAL and b"dtype" in L.mpl_last_error()
    assert call(n=(-1,)) == _lib.MPL_EINVAL and call(x=(None,)) == _lib.MPL_EINVAL
    assert call(x=(4098,)) == _lib.MPL_EINVAL and call(x=(4097,), dtype=(1,)) == _lib.MPL_EINVAL
    assert call(ws=None) == _lib.MPL_EINVAL and call(wsb=4) == _lib.MPL_EWORKSPACE
    assert call(x=(one,) * 400, n=(1 << 30,) * 400, dtype=(1,) * 400, wsb=1 << 14) == _lib.MPL_EWORKSPACE
    assert L.mpl_clip_grads_workspace_bytes(-1) == 0 and L.mpl_clip_grads_workspace_bytes(0) > 0
