"""packed_attention: what is refused, before any launch (no GPU)."""

import ctypes

import pytest
import torch

from model_amd import _lib
from model_amd.attention import packed_attention, packed_attention_backward, packed_attention_forward

I32 = torch.int32


def _args(T=6, S=6, H=4, G=2, hd=32, dtype=torch.float32, **kw):
    a = {"q": torch.zeros(T, H, hd, dtype=dtype), "k": torch.zeros(S, G, hd, dtype=dtype),
         "v": torch.zeros(S, G, hd, dtype=dtype), "starts": torch.tensor([0, 2, T], dtype=I32)}
    a.update(kw)
    return a


BAD = [
    (dict(q=torch.zeros(6, 4, 64)), "do not fit"),
    (dict(q=torch.zeros(6, 128)), "do not fit"),
    (dict(v=torch.zeros(6, 4, 32)), "do not fit"),
    (dict(hd=48), "heads of 48"),
    (dict(hd=0), "heads of 0"),
    (dict(H=4, G=3), "share"),
    (dict(G=0), "share"),
    (dict(dtype=torch.float64), "float32, float16 or bfloat16"),
    (dict(k=torch.zeros(6, 2, 32, dtype=torch.float16)), "float32, float16 or bfloat16"),
    (dict(starts=torch.zeros(3)), "starts"),
    (dict(starts=torch.zeros(0, dtype=I32)), "starts"),
    (dict(starts=torch.zeros(1, 3, dtype=I32)), "starts"),
    (dict(S=9), "need key_starts"),
    (dict(key_lengths=torch.zeros(2, dtype=I32)), "go with key_starts"),
    (dict(key_starts=torch.zeros(4, dtype=I32)), "key_starts"),
    (dict(key_starts=torch.zeros(3, dtype=torch.int64)), "key_starts"),
    (dict(key_starts=torch.zeros(3, dtype=I32), key_lengths=torch.zeros(3, dtype=I32)), "key_lengths"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(), "on the GPU only"),
    (dict(key_starts=torch.zeros(3, dtype=I32), key_lengths=torch.zeros(2, dtype=I32)), "on the GPU only"),
    (dict(starts=torch.zeros(1, dtype=I32), key_starts=torch.zeros(1, dtype=I32), key_lengths=torch.zeros(0, dtype=I32)),
     "on the GPU only"),
]


@pytest.mark.parametrize("kw,match", BAD)
def test_refused(kw, match):
    a = _args(**kw)
    q, k, v, starts = (a.pop(n) for n in ("q", "k", "v", "starts"))
    for f in (packed_attention, packed_attention_forward):
        with pytest.raises(ValueError, match=match):
            f(q, k, v, starts, **a)
    with pytest.raises(ValueError, match=match):
        packed_attention_backward(q, q, k, v, q, torch.zeros(q.shape[:2]), starts, **a)


def test_c_entries_validate_before_launch():
    L = _lib.lib()
    one = 4096  # never read: every call below is refused

    class A(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_void_p) for n in "qkv"]
                    + [(n, ctypes.c_int64) for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head")]
                    + [(n, ctypes.c_int) for n in ("dtype", "heads", "groups", "head_dim")]
                    + [(n, ctypes.c_int64) for n in ("tokens", "keys", "sequences")]
                    + [(n, ctypes.c_void_p) for n in ("starts", "key_starts", "key_lengths")]
                    + [("index_bytes", ctypes.c_int), ("scale", ctypes.c_float)])

    def args(**kw):
        a = dict(q=one, k=one, v=one, q_token=128, q_head=32, k_token=64, k_head=32, v_token=64, v_head=32, dtype=0,
                 heads=4, groups=2, head_dim=32, tokens=10, keys=10, sequences=2, starts=one, key_starts=one,
                 key_lengths=None, index_bytes=4, scale=1.0)
        a.update(kw)
        return ctypes.byref(A(**a))

    def fwd(ws=one, n=1 << 30, out=one, **kw):
        return L.mpl_packed_attention(args(**kw), ws, n, out, one, None)

    def bwd(g=one, gt=128, gh=32, out=one, lse=one, ws=one, n=1 << 30, dq=one, dk=one, dv=one, **kw):
        return L.mpl_packed_attention_bwd(args(**kw), g, gt, gh, out, lse, None, ws, n, dq, dk, dv, None)

    assert fwd(tokens=0) == _lib.MPL_OK
    for f in (fwd, bwd):
        assert f(dtype=3) == _lib.MPL_EINVAL and f(heads=5) == _lib.MPL_EINVAL and f(groups=0) == _lib.MPL_EINVAL
        assert f(head_dim=96) == _lib.MPL_EUNSUPPORTED and b"head_dim" in L.mpl_last_error()
        assert f(tokens=-1) == _lib.MPL_EINVAL and f(sequences=-1) == _lib.MPL_EINVAL and f(keys=-1) == _lib.MPL_EINVAL
        assert f(tokens=1 << 31) == _lib.MPL_EUNSUPPORTED and f(keys=1 << 31) == _lib.MPL_EUNSUPPORTED
        assert f(sequences=1 << 24) == _lib.MPL_EUNSUPPORTED and b"too many" in L.mpl_last_error()
        assert f(index_bytes=2) == _lib.MPL_EINVAL
        assert f(scale=0.0) == _lib.MPL_EINVAL and f(scale=float("nan")) == _lib.MPL_EINVAL
        assert f(scale=float("inf")) == _lib.MPL_EINVAL
        assert f(starts=None) == _lib.MPL_EINVAL and f(starts=one + 2) == _lib.MPL_EINVAL
        assert f(q=None) == _lib.MPL_EINVAL and f(q=one + 4) == _lib.MPL_EINVAL and f(v=None) == _lib.MPL_EINVAL
        assert f(k_token=63) == _lib.MPL_EINVAL and b"aligned" in L.mpl_last_error()
        assert f(q_head=-32) == _lib.MPL_EINVAL and f(dtype=1, v_head=36) == _lib.MPL_EINVAL
    assert fwd(out=None) == _lib.MPL_EINVAL and fwd(out=one + 4) == _lib.MPL_EINVAL
    assert fwd(tokens=2, keys=100000, n=8) == _lib.MPL_EWORKSPACE
    assert fwd(tokens=2, keys=100000, ws=None) == _lib.MPL_EINVAL
    assert bwd(dq=None, dk=None, dv=None) == _lib.MPL_EINVAL and bwd(dq=one + 4) == _lib.MPL_EINVAL
    assert bwd(g=None) == _lib.MPL_EINVAL and bwd(gt=2) == _lib.MPL_EINVAL and bwd(lse=None) == _lib.MPL_EINVAL
    assert bwd(ws=None) == _lib.MPL_EINVAL and bwd(ws=one + 8) == _lib.MPL_EINVAL and bwd(n=8) == _lib.MPL_EWORKSPACE
    W = L.mpl_packed_attention_workspace_bytes
    assert W(args(), 0) > 0 and W(args(), 1) >= 2 * 4 * 40
    assert W(args(head_dim=48), 0) == 0 and W(args(tokens=1 << 31), 1) == 0 and W(None, 0) == 0


def _calls():
    ops = _lib.ops()
    k = torch.zeros(0, 2, 32)
    st = torch.zeros(1, dtype=I32)
    return {
        "packed_attention": lambda q: ops.packed_attention(q, k, k, st, None, None, 1.0, False, False)[0],
        "packed_attention_backward": lambda q: ops.packed_attention_backward(
            q, torch.zeros(0, 4, 32), k, k, torch.zeros(0, 4, 32), torch.zeros(0, 4), st, None, None, 1.0, None)[0],
    }


@pytest.mark.parametrize("name", ["packed_attention", "packed_attention_backward"])
def test_transforms_are_refused(name):
    """Calls of no rows launch nothing, and take the same ways."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    f, x = _calls()[name], torch.zeros(0, 4, 32)
    f(x)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="dual tensor"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, x, check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(f)(x)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.vmap(f)(torch.zeros(3, 0, 4, 32))
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda x: f(x).sum())(x)
    with FakeTensorMode() as mode:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            f(mode.from_tensor(x))
    f(x)


def test_backward_under_capture_is_refused():
    ops = _lib.ops()
    q = torch.zeros(0, 4, 32, requires_grad=True)
    k = torch.zeros(0, 2, 32)
    out, _ = ops.packed_attention(q, k, k, torch.zeros(1, dtype=I32), None, None, 1.0, False, True)
    ops.pretend_capturing(True)
    try:
        with pytest.raises(RuntimeError, match="HIP graph capture"):
            out.sum().backward()
    finally:
        ops.pretend_capturing(False)
