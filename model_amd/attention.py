"""Causal attention over packed sequences of unlike lengths, with grouped heads
and its backward pass (the backbone's attention, model.py:88-95, for documents
packed into one batch, for prompts that continue a cache and for single new
tokens over one), as libmpl.so launches (mpl_packed_attention,
mpl_packed_attention_bwd).  Here arguments are checked; the calls and the
autograd node are csrc/torch/ops.cpp.

  packed_attention            out (and lse), differentiable by torch autograd
  packed_attention_forward    (out, lse) outside autograd, what the backward takes
  packed_attention_backward   its gradients; both may be captured in a HIP graph
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _lib

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
HEAD_DIMS = (32, 64, 128)


def _check_places(what: str, name: str, t: torch.Tensor, numel: Optional[int], like: Optional[torch.Tensor]) -> None:
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64) or t.numel() == 0 and numel != 0:
        raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} must be one-dimensional int32 or int64")
    if like is not None and (t.numel() != numel or t.dtype != like.dtype):
        raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} must be [{numel}] of starts' {like.dtype}")


def _check(what: str, q, k, v, starts, key_starts, key_lengths, scale) -> float:
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit "
                         "([tokens, heads, hd], and twice [keys, key heads, hd])")
    if q.shape[2] not in HEAD_DIMS:
        raise ValueError(f"{what}: heads of {q.shape[2]} elements ({', '.join(map(str, HEAD_DIMS))})")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{what}: {q.shape[1]} heads cannot share {k.shape[1]} key heads alike")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q {q.dtype}, k {k.dtype} and v {v.dtype} must all be float32, float16 or bfloat16")
    _check_places(what, "starts", starts, None, None)
    if key_starts is None:
        if key_lengths is not None:
            raise ValueError(f"{what}: key_lengths go with key_starts")
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"{what}: {k.shape[0]} keys for {q.shape[0]} tokens need key_starts")
    else:
        _check_places(what, "key_starts", key_starts, starts.numel(), starts)
        if key_lengths is not None:
            _check_places(what, "key_lengths", key_lengths, starts.numel() - 1, starts)
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:  # of fp32's normal numbers, with the scores' own range left over
        raise ValueError(f"{what}: scale {scale} must be positive and of ordinary size")
    if q.device.type != "cuda":
        raise ValueError(f"{what} runs on the GPU only (libmpl.so), q is on {q.device}")
    for name, t in (("k", k), ("v", v), ("starts", starts), ("key_starts", key_starts), ("key_lengths", key_lengths)):
        if t is not None and t.device != q.device:
            raise ValueError(f"{what}: {name} on {t.device}, q on {q.device}")
    return scale


def _capturing() -> bool:
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


_NO_CAPTURE = ("torch autograd through packed_attention is not supported under HIP graph capture: use "
               "packed_attention_forward and packed_attention_backward, which capture")


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, *,
                     key_starts: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None,
                     return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of each of several sequences that lie one behind the
    other: softmax(scale q . k) v over the keys that a query sees.

    q [tokens, heads, hd] and k, v [keys, key heads, hd] are fp32, fp16 or bf16,
    hd 32, 64 or 128, any strides (the slices of a fused projection are read as
    they lie); heads is a multiple of key heads, and query head h reads key head
    h // (heads // key heads).  scale is hd^-0.5 unless given, above 0.

    starts [n + 1] (int32 or int64, on the GPU) ascends in [0, tokens]: sequence i
    is q[starts[i]:starts[i + 1]], and its keys are the same rows of k and v.  With
    key_starts [n + 1], ascending in [0, keys], they are
    k[key_starts[i]:key_starts[i + 1]], of which key_lengths [n], where given, says
    how many are in use (a cache with free places).  A sequence's queries are its
    last tokens: of Lq queries and Lk keys query j sees keys 0 .. j + Lk - Lq.  So a
    whole prompt has Lq = Lk, a prompt that continues a cache Lq < Lk, a new token
    Lq = 1.  Sequences may be empty.  A query that sees no key, and one of no
    sequence, gives 0 (lse -inf) and passes no gradient.

    Returns out as q, and with ``return_lse`` also the logsumexp of each query's
    scores, fp32 [tokens, heads], differentiable as well.  Sums, maxima and the
    softmax are fp32; in 16 bits the weights, and their gradients, are rounded to
    the inputs' type for the products with v, k, q and the output's gradient.
    Deterministic: no atomics.  What is not finite in one sequence never reaches
    another; in its own it may reach every row.  The GPU's starts are not read by
    the host: such as do not ascend within the arrays give unspecified rows, never
    an access outside.

    Inside a captured HIP graph use packed_attention_forward and
    packed_attention_backward.  Differentiable once; dual tensors, torch.func's
    transforms and tracing are refused."""
    scale = _check("packed_attention", q, k, v, starts, key_starts, key_lengths, scale)
    autograd = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if autograd and _capturing():
        raise RuntimeError(_NO_CAPTURE)
    out, lse = _lib.ops().packed_attention(q, k, v, starts, key_starts, key_lengths, scale, return_lse, autograd)
    return (out, lse) if return_lse else out


def packed_attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, *,
                             key_starts: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None,
                             scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """packed_attention outside autograd: (out, lse), what
    packed_attention_backward takes."""
    scale = _check("packed_attention_forward", q, k, v, starts, key_starts, key_lengths, scale)
    return _lib.ops().packed_attention(q, k, v, starts, key_starts, key_lengths, scale, True, False)


def packed_attention_backward(g_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                              out: torch.Tensor, lse: torch.Tensor, starts: torch.Tensor, *,
                              key_starts: Optional[torch.Tensor] = None, key_lengths: Optional[torch.Tensor] = None,
                              scale: Optional[float] = None, g_lse: Optional[torch.Tensor] = None
                              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv) from the gradient g_out of out (and g_lse of lse), the
    forward's arguments and what packed_attention_forward returned for them."""
    what = "packed_attention_backward"
    scale = _check(what, q, k, v, starts, key_starts, key_lengths, scale)
    for name, t in (("g_out", g_out), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} on {t.device} must be as q {tuple(q.shape)} "
                             f"{q.dtype}")
    for name, t in (("lse", lse), ("g_lse", g_lse)):
        if t is not None and (t.shape != q.shape[:2] or t.dtype != torch.float32 or t.device != q.device):
            raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} on {t.device} must be fp32 "
                             f"{tuple(q.shape[:2])} on {q.device}")
    return _lib.ops().packed_attention_backward(g_out, q, k, v, out, lse, starts, key_starts, key_lengths, scale, g_lse)
