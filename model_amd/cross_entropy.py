"""Softmax cross entropy of tokens over the vocabulary, from the hidden rows
and the embedding table (the backbone's tied output layer, model.py:125-126,
and the loss that a trainer takes of its logits), with its gradients.  The
logits never lie in memory as a whole: libmpl.so forms them tile by tile
(mpl_vocab_cross_entropy), and again in pieces of the vocabulary for the
gradients (mpl_vocab_cross_entropy_bwd).  Here arguments are checked; the calls
and the autograd node are csrc/torch/ops.cpp.

  vocab_cross_entropy        the loss of each token, differentiable by torch autograd
  vocab_cross_entropy_grads  loss and gradients in one call without autograd (for captured training steps)
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_WIDTH = 65536


def _check(hidden: torch.Tensor, embedding: torch.Tensor, targets: torch.Tensor, what: str) -> None:
    if hidden.dim() < 1 or embedding.dim() != 2 or hidden.shape[-1] != embedding.shape[1]:
        raise ValueError(f"{what}: hidden {tuple(hidden.shape)} and embedding {tuple(embedding.shape)} do not fit "
                         "([..., d] and [vocab, d])")
    if embedding.shape[0] == 0 or embedding.shape[1] == 0:
        raise ValueError(f"{what}: an empty embedding {tuple(embedding.shape)}")
    if embedding.shape[1] > MAX_WIDTH:
        raise ValueError(f"{what}: rows of {embedding.shape[1]} elements, at most {MAX_WIDTH}")
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


def _check_grad(name: str, g: Optional[torch.Tensor], shape, device) -> None:
    if g is not None and (g.shape != shape or g.device != device or not g.is_floating_point()):
        raise ValueError(f"{name} {tuple(g.shape)} {g.dtype} on {g.device}: must be floating, {tuple(shape)}, on {device}")


def _capturing() -> bool:
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


_NO_CAPTURE = ("torch autograd through vocab_cross_entropy is not supported under HIP graph capture: use "
               "vocab_cross_entropy_grads, which captures")


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

    Logits are sums in fp32 of the exact products (of more than 64 rows fp32
    operands are held to 2^-23 of each and 2^-39 of the largest of their row, 2^-33
    of a table row's).  fp32 rows or table entries that are not finite may give NaN
    where the formula has a logit of -inf.  Up to some 2^39 logits and 2^34
    elements of both arrays.
    The gradients hold dz in fp16 under a power of two a token (fp32: hi and lo,
    to 2^-23), down to 2^-38 of the token's own gradient; the table in d hidden and
    the tokens' weighted rows in d embedding down to 2^-39 of their largest (bf16
    exactly above 2^-29 of it, fp16 tables as they are); those of few tokens (64 in
    fp32) are in fp32.  A row that passes no gradient adds nothing to the table's,
    whatever it holds: padding may be NaN.  For gradients
    inside a captured HIP graph use vocab_cross_entropy_grads.  Dual tensors,
    torch.func's transforms and tracing are refused."""
    _check(hidden, embedding, targets, "vocab_cross_entropy")
    autograd = torch.is_grad_enabled() and (hidden.requires_grad or embedding.requires_grad)
    if autograd and _capturing():
        raise RuntimeError(_NO_CAPTURE)
    loss, lse = _lib.ops().vocab_cross_entropy(hidden, embedding, targets, int(ignore_index), autograd)
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
    _check_grad("g_loss", g_loss, targets.shape, hidden.device)
    _check_grad("g_lse", g_lse, targets.shape, hidden.device)
    if g_loss is None and g_lse is None:
        raise ValueError("vocab_cross_entropy_grads: g_loss or g_lse is needed")
    return _lib.ops().vocab_cross_entropy_grads(hidden, embedding, targets, g_loss, g_lse, int(ignore_index))
