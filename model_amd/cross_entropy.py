"""Softmax cross entropy of tokens over the vocabulary, from the hidden rows
and the embedding table (the backbone's tied output layer, model.py:125-126,
and the loss that a trainer takes of its logits), with its gradients.  The
logits never lie in memory as a whole: libmpl.so forms them tile by tile
(mpl_vocab_cross_entropy), and again in pieces of the vocabulary for the
gradients (mpl_vocab_cross_entropy_bwd).

  vocab_cross_entropy        the loss of each token, differentiable by torch autograd
  vocab_cross_entropy_grads  loss and gradients in one call without autograd (for captured training steps)
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.MPL_F32, torch.float16: _lib.MPL_F16, torch.bfloat16: _lib.MPL_BF16}


def _rows(t: torch.Tensor, d: int) -> Tuple[torch.Tensor, int]:
    """``t`` [..., d] as rows that the library reads, elements of a row next to
    each other, and the elements from row to row.  Copied only where it does
    not lie so, or where 16-bit rows that are read by tiles as they lie (d a
    multiple of 64) do not start at 16 bytes."""
    pitch = d
    if not t.is_contiguous():
        t = t.reshape(-1, d)
        if d > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < d:
            t = t.contiguous()
        elif t.shape[0] > 1:
            pitch = t.stride(0)
    if t.dtype != torch.float32 and d % 64 == 0 and (t.data_ptr() % 16 or pitch % 8):
        return t.clone(memory_format=torch.contiguous_format), d
    return t, pitch


def _check(hidden: torch.Tensor, embedding: torch.Tensor, targets: torch.Tensor, what: str) -> None:
    if hidden.dim() < 1 or embedding.dim() != 2 or hidden.shape[-1] != embedding.shape[1]:
        raise ValueError(f"{what}: hidden {tuple(hidden.shape)} and embedding {tuple(embedding.shape)} do not fit "
                         "([..., d] and [vocab, d])")
    if embedding.shape[0] == 0 or embedding.shape[1] == 0:
        raise ValueError(f"{what}: an empty embedding {tuple(embedding.shape)}")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"{what}: targets {tuple(targets.shape)} for hidden {tuple(hidden.shape)}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: targets must be int64 or int32, got {targets.dtype}")
    if hidden.dtype not in _DTYPES or embedding.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden {hidden.dtype} and embedding {embedding.dtype} must both be float32, float16 "
                         "or bfloat16")
    if hidden.device.type != "cuda" or embedding.device != hidden.device or targets.device != hidden.device:
        raise ValueError(f"{what} runs on the GPU only (libmpl.so), all arguments on one device: hidden on "
                         f"{hidden.device}, embedding on {embedding.device}, targets on {targets.device}")


def _workspace(rows: int, vocab: int, d: int, code: int, backward: int, device) -> torch.Tensor:
    n = _lib.lib().mpl_vocab_cross_entropy_workspace_bytes(rows, vocab, d, code, backward)
    if n == 0:
        raise ValueError(f"vocab_cross_entropy: {rows} rows, a vocabulary of {vocab} and a width of {d} are out of range")
    return torch.empty(n, dtype=torch.uint8, device=device)


def _ids(targets: torch.Tensor) -> torch.Tensor:
    return (targets if targets.dtype == torch.int64 else targets.to(torch.int64)).contiguous()


def _forward(hidden, embedding, ids, ignore_index: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, lse) of ids' shape; ids contiguous int64."""
    dev, (V, d), R = hidden.device, embedding.shape, ids.numel()
    loss = torch.empty(ids.shape, dtype=torch.float32, device=dev)
    lse = torch.empty(ids.shape, dtype=torch.float32, device=dev)
    if R:
        (h, h_pitch), (e, e_pitch) = _rows(hidden, d), _rows(embedding, d)
        code = _DTYPES[h.dtype]
        with _lib.on_device(dev):
            ws = _workspace(R, V, d, code, 0, dev)
            _lib.check(_lib.lib().mpl_vocab_cross_entropy(
                h.data_ptr(), h_pitch, e.data_ptr(), e_pitch, code, ids.data_ptr(), R, V, d, ignore_index,
                ws.data_ptr(), ws.numel(), loss.data_ptr(), lse.data_ptr(), _lib.stream_ptr(dev)),
                "mpl_vocab_cross_entropy")
    return loss, lse


def _backward(hidden, embedding, ids, ignore_index: int, lse, g_loss, g_lse, want_h: bool, want_e: bool):
    """Gradients of hidden and embedding (None where not wanted); g_loss and g_lse fp32 or None (not both)."""
    dev, (V, d), R = hidden.device, embedding.shape, ids.numel()
    dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if want_h else None
    de = (torch.empty if R else torch.zeros)((V, d), dtype=hidden.dtype, device=dev) if want_e else None
    if R and (want_h or want_e):
        (h, h_pitch), (e, e_pitch) = _rows(hidden, d), _rows(embedding, d)
        code = _DTYPES[h.dtype]
        P = _lib.ptr
        with _lib.on_device(dev):
            ws = _workspace(R, V, d, code, 1, dev)
            _lib.check(_lib.lib().mpl_vocab_cross_entropy_bwd(
                h.data_ptr(), h_pitch, e.data_ptr(), e_pitch, code, ids.data_ptr(), R, V, d, ignore_index,
                lse.data_ptr(), P(g_loss), P(g_lse), ws.data_ptr(), ws.numel(), P(dh), P(de), _lib.stream_ptr(dev)),
                "mpl_vocab_cross_entropy_bwd")
    return dh, de


def _row_grad(g: Optional[torch.Tensor], shape, device, name: str) -> Optional[torch.Tensor]:
    if g is None:
        return None
    if g.shape != shape or g.device != device or not g.is_floating_point():
        raise ValueError(f"{name} {tuple(g.shape)} {g.dtype} on {g.device}: must be floating, {tuple(shape)}, on {device}")
    return g.detach().to(torch.float32).contiguous()


def _capturing() -> bool:
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


_NO_CAPTURE = ("torch autograd through vocab_cross_entropy is not supported under HIP graph capture: use "
               "vocab_cross_entropy_grads, which captures")


class _CrossEntropyFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, embedding, targets, ignore_index):
        ids = _ids(targets)
        loss, lse = _forward(hidden, embedding, ids, ignore_index)
        ctx.save_for_backward(hidden, embedding, ids, lse)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        return loss, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_loss, g_lse):
        if _capturing():
            raise RuntimeError(_NO_CAPTURE)
        if g_loss is None and g_lse is None:
            return None, None, None, None
        hidden, embedding, ids, lse = ctx.saved_tensors
        want_h, want_e = ctx.needs_input_grad[:2]
        dh, de = _backward(hidden, embedding, ids, ctx.ignore_index, lse,
                           _row_grad(g_loss, ids.shape, hidden.device, "the loss's gradient"),
                           _row_grad(g_lse, ids.shape, hidden.device, "the logsumexp's gradient"), want_h, want_e)
        return dh, de, None, None


def vocab_cross_entropy(hidden: torch.Tensor, embedding: torch.Tensor, targets: torch.Tensor, *,
                        ignore_index: int = -100,
                        return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The cross entropy of each token: with z = hidden . embedding^T (embed.attend),
    logsumexp(z) - z[target], fp32 of targets' shape.

    hidden [..., d] and embedding [vocab, d] are fp32, fp16 or bf16 (both the
    same; any strides, any d up to 65,536), targets [...] int64 or int32 word
    ids.  Where the target is ``ignore_index`` the loss is 0 and passes no
    gradient; any other id outside the table gives NaN.  With ``return_lse``
    also the logsumexp of each token's logits (of ignored ones too),
    differentiable as well (a z-loss, or logits' norms).  A mean over the
    counted tokens is loss.sum() / (targets != ignore_index).sum().

    Logits are sums in fp32 of the exact products (fp32 operands are held to
    2^-23 of each).  fp32 rows or table entries that are not finite give NaN.
    The gradients hold dz in fp16 under a power of two (fp32: hi and lo, to
    2^-23), down to 2^-38 of the largest gradient of a token.  For gradients
    inside a captured HIP graph use vocab_cross_entropy_grads."""
    _check(hidden, embedding, targets, "vocab_cross_entropy")
    if torch.is_grad_enabled() and (hidden.requires_grad or embedding.requires_grad):
        if _capturing():
            raise RuntimeError(_NO_CAPTURE)
        loss, lse = _CrossEntropyFunction.apply(hidden, embedding, targets, int(ignore_index))
        return (loss, lse) if return_lse else loss
    loss, lse = _forward(hidden, embedding, _ids(targets), int(ignore_index))
    return (loss, lse) if return_lse else loss


def vocab_cross_entropy_grads(hidden: torch.Tensor, embedding: torch.Tensor, targets: torch.Tensor,
                              g_loss: Optional[torch.Tensor], g_lse: Optional[torch.Tensor] = None, *,
                              ignore_index: int = -100
                              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """vocab_cross_entropy with its gradients in one call, outside autograd:
    (loss, lse, d_hidden, d_embedding) for the gradients g_loss and g_lse of
    each token's loss and logsumexp (targets' shape; either may be None).  It
    may be captured in a HIP graph."""
    _check(hidden, embedding, targets, "vocab_cross_entropy_grads")
    gl = _row_grad(g_loss, targets.shape, hidden.device, "g_loss")
    gs = _row_grad(g_lse, targets.shape, hidden.device, "g_lse")
    if gl is None and gs is None:
        raise ValueError("vocab_cross_entropy_grads: g_loss or g_lse is needed")
    with torch.no_grad():
        ids = _ids(targets)
        loss, lse = _forward(hidden, embedding, ids, int(ignore_index))
        dh, de = _backward(hidden, embedding, ids, int(ignore_index), lse, gl, gs, True, True)
    return loss, lse, dh, de
