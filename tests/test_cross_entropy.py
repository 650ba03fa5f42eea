"""vocab_cross_entropy: what is refused, before any launch (no GPU)."""

import ctypes

import pytest
import torch

from model_amd import _lib
from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads


def _args(**kw):
    a = dict(hidden=torch.zeros(4, 8), embedding=torch.zeros(10, 8), targets=torch.zeros(4, dtype=torch.int64))
    a.update(kw)
    return a["hidden"], a["embedding"], a["targets"]


@pytest.mark.parametrize("kw,match", [
    (dict(embedding=torch.zeros(10, 9)), "do not fit"),
    (dict(embedding=torch.zeros(10, 2, 4)), "do not fit"),
    (dict(hidden=torch.zeros(())), "do not fit"),
    (dict(embedding=torch.zeros(0, 8)), "empty embedding"),
    (dict(targets=torch.zeros(5, dtype=torch.int64)), "targets"),
    (dict(targets=torch.zeros(4)), "int64 or int32"),
    (dict(embedding=torch.zeros(10, 8, dtype=torch.float16)), "must both be"),
    (dict(hidden=torch.zeros(4, 8, dtype=torch.float64), embedding=torch.zeros(10, 8, dtype=torch.float64)),
     "must both be"),
    (dict(), "on the GPU only"),
])
def test_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        vocab_cross_entropy(*_args(**kw))
    with pytest.raises(ValueError, match=match):
        vocab_cross_entropy_grads(*_args(**kw), torch.zeros(4))


def test_workspace_bytes():
    L = _lib.lib()
    for dtype in (_lib.MPL_F32, _lib.MPL_F16, _lib.MPL_BF16):
        for rows, vocab, d in ((1, 1, 1), (8192, 16384, 256), (1001, 50021, 500), (1 << 20, 131072, 1024)):
            fwd = L.mpl_vocab_cross_entropy_workspace_bytes(rows, vocab, d, dtype, 0)
            bwd = L.mpl_vocab_cross_entropy_workspace_bytes(rows, vocab, d, dtype, 1)
            assert 0 < fwd < rows * vocab * 4 + (64 << 20) + 8 * (rows + vocab) * (d + 64) and bwd > 0
    # a piece's dz stays near 512 MiB whatever the vocabulary
    big = L.mpl_vocab_cross_entropy_workspace_bytes(16384, 1 << 20, 1024, _lib.MPL_F16, 1)
    assert big < (1 << 30)
    for rows, vocab, d, dtype in ((-1, 4, 4, 0), (4, 0, 4, 0), (4, 4, 0, 0), (4, 4, 65537, 0), (4, 4, 4, 3),
                                  ((1 << 31) + 1, 4, 4, 0), (1 << 31, 1 << 20, 64, 0)):
        assert L.mpl_vocab_cross_entropy_workspace_bytes(rows, vocab, d, dtype, 0) == 0


@pytest.mark.parametrize("rows,vocab,d,ok", [
    (1 << 20, 1 << 18, 1024, True),  # 2^22 tiles
    (1 << 20, 1 << 19, 1024, False),  # 2^23: 2^32 threads of the tiles' grid
    (1 << 19, 1 << 19, 16384, False),  # 2^34 elements: 2^32 threads of the sums
    ((1 << 19) - 1, 1 << 19, 16384, True),
    (1 << 29, 1, 1, False)])  # 2^32 threads of the join
def test_largest_sizes(rows, vocab, d, ok):
    L = _lib.lib()
    for dtype in (_lib.MPL_F32, _lib.MPL_F16, _lib.MPL_BF16):
        for backward in (0, 1):
            assert (L.mpl_vocab_cross_entropy_workspace_bytes(rows, vocab, d, dtype, backward) > 0) == ok


def test_width_does_not_wrap():
    d = (1 << 32) + 64
    t = [torch.empty(1, d, device="meta", dtype=torch.float16) for _ in range(2)]
    with pytest.raises(ValueError, match="at most 65536"):
        vocab_cross_entropy(*t, torch.zeros(1, dtype=torch.int64, device="meta"))


def test_c_entries_validate_before_launch():
    L = _lib.lib()
    one = ctypes.c_void_p(4096)  # never read: every call below is refused
    ok = dict(hp=64, ep=64, dtype=_lib.MPL_F16, rows=4, vocab=8, d=64, ws=one, n=1 << 30)

    def fwd(h=one, e=one, t=one, loss=one, lse=one, **kw):
        a = {**ok, **kw}
        return L.mpl_vocab_cross_entropy(h, a["hp"], e, a["ep"], a["dtype"], t, a["rows"], a["vocab"], a["d"], -100,
                                         a["ws"], a["n"], loss, lse, None)

    def bwd(h=one, e=one, t=one, lse=one, gl=one, gs=None, dh=one, de=one, **kw):
        a = {**ok, **kw}
        return L.mpl_vocab_cross_entropy_bwd(h, a["hp"], e, a["ep"], a["dtype"], t, a["rows"], a["vocab"], a["d"],
                                             -100, lse, gl, gs, a["ws"], a["n"], dh, de, None)

    assert fwd(rows=0) == _lib.MPL_OK
    for f in (fwd, bwd):
        assert f(dtype=7) == _lib.MPL_EINVAL and b"bad sizes or type" in L.mpl_last_error()
        assert f(rows=-1) == _lib.MPL_EINVAL and f(vocab=0) == _lib.MPL_EINVAL and f(d=0) == _lib.MPL_EINVAL
        assert f(h=None) == _lib.MPL_EINVAL and f(e=None) == _lib.MPL_EINVAL and f(t=None) == _lib.MPL_EINVAL
        assert f(hp=63) == _lib.MPL_EINVAL and b"pitch" in L.mpl_last_error()
        assert f(ep=68) == _lib.MPL_EINVAL and b"16-byte" in L.mpl_last_error()
        assert f(hp=1 << 23) == _lib.MPL_EUNSUPPORTED and b"2^23" in L.mpl_last_error()
        assert f(rows=1 << 31, vocab=1 << 31) == _lib.MPL_EINVAL
        assert f(h=ctypes.c_void_p(4098)) == _lib.MPL_EINVAL
        assert f(h=ctypes.c_void_p(4097), d=60) == _lib.MPL_EINVAL and b"elements" in L.mpl_last_error()
        assert f(ws=None) == _lib.MPL_EINVAL
        assert f(n=100) == _lib.MPL_EWORKSPACE and b"workspace" in L.mpl_last_error()
    assert fwd(loss=None) == _lib.MPL_EINVAL
    assert bwd(rows=0) == _lib.MPL_EINVAL
    assert bwd(gl=None) == _lib.MPL_EINVAL and bwd(lse=None) == _lib.MPL_EINVAL
    assert bwd(dh=None, de=None) == _lib.MPL_EINVAL


@pytest.mark.parametrize("rows,vocab,d", [(16384, 131072, 1024), (8192, 1 << 18, 512)])
def test_backward_holds_a_piece_of_the_gradients_table(rows, vocab, d):
    """Beside z's operands (fp32: both arrays split, 4 bytes an element) the
    backward holds operands of one piece of the vocabulary: at most 512 MiB of dz
    (2 bytes an element; fp32 4), the piece's table, the weighted rows, and both
    gradients' fp32 sums in at most 8 parts."""
    L = _lib.lib()
    for dtype, size in ((_lib.MPL_F32, 4), (_lib.MPL_F16, 2), (_lib.MPL_BF16, 2)):
        n = L.mpl_vocab_cross_entropy_workspace_bytes(rows, vocab, d, dtype, 1)
        z = (rows + vocab) * d * 4 if dtype == _lib.MPL_F32 else 0
        piece = (512 << 20) // (rows * size)
        most = z + (512 << 20) + (piece + rows) * d * size + rows * d * 4 * 8 + piece * d * 4 * 8 + (16 << 20)
        assert n <= most, (dtype, n, most)
