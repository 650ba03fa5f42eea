"""LayerNorm with its backward pass (nn.LayerNorm of model.py:86-125), with the
residual add before it, as libmpl.so launches (mpl_layer_norm,
mpl_layer_norm_bwd).  Here arguments are checked; the calls and the autograd
node are csrc/torch/ops.cpp.

  layer_norm            y (and x + residual), differentiable by torch autograd
  layer_norm_forward    the same outside autograd, with the statistics that the backward takes
  layer_norm_backward   its gradients; both may be captured in a HIP graph
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

LN_EPS = 1e-6  # flax.linen.LayerNorm default
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
MAX_WIDTH = 16384


def _check(what: str, x: torch.Tensor, params, others) -> None:
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what}: rows of shape {tuple(x.shape)}")
    d = x.shape[-1]
    if d > MAX_WIDTH:
        raise ValueError(f"{what}: rows of {d} elements, at most {MAX_WIDTH}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what}: x must be float32, float16 or bfloat16, got {x.dtype}")
    for name, t in params:
        if t.shape != (d,) or t.dtype not in (torch.float32, x.dtype) or t.dtype != params[0][1].dtype:
            raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} must be [{d}], float32 or x's {x.dtype}, all "
                             "parameters alike")
    for name, t in others:
        if t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} must be as x {tuple(x.shape)} {x.dtype}")
    if x.device.type != "cuda":
        raise ValueError(f"{what} runs on the GPU only (libmpl.so), x is on {x.device}")
    for name, t in (*params, *others):
        if t.device != x.device:
            raise ValueError(f"{what}: {name} on {t.device}, x on {x.device}")


def _capturing() -> bool:
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


_NO_CAPTURE = ("torch autograd through layer_norm is not supported under HIP graph capture: use layer_norm_forward and "
               "layer_norm_backward, which capture")


def layer_norm(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor, eps: float = LN_EPS, *,
               residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """LayerNorm over the last axis of x [..., d] (fp32, fp16 or bf16, any
    strides, d up to 16,384): (x - mean) rstd scale + bias in fp32, rounded
    once to x's type; scale and bias [d] are fp32 or of x's type.  With
    ``residual`` (as x) the norm is that of s = x + residual rounded to x's
    type, and (y, s) are returned: the backbone's residual stream and the
    norm of its next block in one launch, the bits of the add and of
    layer_norm(s).

    Gradients come from mpl_layer_norm_bwd, those of scale and bias as fixed-order
    fp32 sums over the rows; the gradient of s joins that of x in the same pass.
    Inside a captured HIP graph use layer_norm_forward and layer_norm_backward.
    Dual tensors, torch.func's transforms and tracing are refused."""
    others = () if residual is None else (("residual", residual),)
    _check("layer_norm", x, (("scale", scale), ("bias", bias)), others)
    autograd = torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or bias.requires_grad
                                            or residual is not None and residual.requires_grad)
    if autograd and _capturing():
        raise RuntimeError(_NO_CAPTURE)
    return _lib.ops().layer_norm(x, scale, bias, float(eps), residual, autograd)


def layer_norm_forward(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor, eps: float = LN_EPS, *,
                       residual: Optional[torch.Tensor] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """layer_norm outside autograd: (y, s, mean, rstd), what layer_norm_backward
    takes: s is x, or x + residual; mean and rstd are fp32 [rows]."""
    others = () if residual is None else (("residual", residual),)
    _check("layer_norm_forward", x, (("scale", scale), ("bias", bias)), others)
    return _lib.ops().layer_norm_forward(x, scale, bias, float(eps), residual)


def layer_norm_backward(g_y: torch.Tensor, s: torch.Tensor, scale: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor, *, g_residual: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(d_x, d_scale, d_bias) from the gradient g_y of y and what
    layer_norm_forward returned; g_residual, the gradient of s from elsewhere
    (the residual stream's), is added to d_x."""
    others = (("g_y", g_y),) if g_residual is None else (("g_y", g_y), ("g_residual", g_residual))
    _check("layer_norm_backward", s, (("scale", scale),), others)
    rows = s.numel() // s.shape[-1]
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.numel() != rows or t.dtype != torch.float32 or t.device != s.device or not t.is_contiguous():
            raise ValueError(f"layer_norm_backward: {name} {tuple(t.shape)} {t.dtype} must be contiguous fp32 of {rows} "
                             f"rows on {s.device}")
    return _lib.ops().layer_norm_backward(g_y, s, scale, mean, rstd, g_residual)
