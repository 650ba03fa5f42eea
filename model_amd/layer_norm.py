"""LayerNorm with its backward pass (nn.LayerNorm of model.py:86-125), with the
residual add before it, as libmpl.so launches (mpl_layer_norm,
mpl_layer_norm_bwd).

  layer_norm            y (and x + residual), differentiable by torch autograd
  layer_norm_forward    the same outside autograd, with the statistics that the backward takes
  layer_norm_backward   its gradients; both may be captured in a HIP graph
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

LN_EPS = 1e-6  # flax.linen.LayerNorm default
_DTYPES = {torch.float32: _lib.MPL_F32, torch.float16: _lib.MPL_F16, torch.bfloat16: _lib.MPL_BF16}
MAX_WIDTH = 16384


def _rows(t: torch.Tensor, d: int) -> torch.Tensor:
    """``t`` as [rows, d], elements of a row next to each other, rows apart by
    any pitch of at least d; copied only where it does not lie so."""
    t = t.reshape(-1, d)
    if d > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < d:
        return t.contiguous()
    return t


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


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


def _forward(x, scale, bias, eps, residual, stats: bool):
    """(y, sum or None, mean, rstd [rows]) of x [..., d] and its parameters, checked."""
    d, shape = x.shape[-1], x.shape
    x2 = _rows(x, d)
    rows = x2.shape[0]
    y = torch.empty((rows, d), dtype=x.dtype, device=x.device)
    total = None if residual is None else torch.empty((rows, d), dtype=x.dtype, device=x.device)
    st = torch.empty((2, rows), dtype=torch.float32, device=x.device) if stats else None
    mean, rstd = (st[0], st[1]) if stats else (None, None)
    if rows:
        r2 = None if residual is None else _rows(residual, d)
        scale, bias = scale.contiguous(), bias.contiguous()
        P = _lib.ptr
        with _lib.on_device(x.device):
            _lib.check(_lib.lib().mpl_layer_norm(
                x2.data_ptr(), _pitch(x2), P(r2), 0 if r2 is None else _pitch(r2), _DTYPES[x.dtype], scale.data_ptr(),
                bias.data_ptr(), _DTYPES[scale.dtype], rows, d, float(eps), y.data_ptr(), P(total), P(mean), P(rstd),
                _lib.stream_ptr(x.device)), "mpl_layer_norm")
    return y.view(shape), None if total is None else total.view(shape), mean, rstd


def _backward(g_y, s, scale, mean, rstd, g_residual, want_x: bool, want_params: bool):
    """(dx, d_scale, d_bias), None where not wanted."""
    d = s.shape[-1]
    s2, g2 = _rows(s, d), _rows(g_y, d)
    rows = s2.shape[0]
    dx = torch.empty((rows, d), dtype=s.dtype, device=s.device) if want_x else None
    dp = torch.empty((2, d), dtype=scale.dtype, device=s.device) if want_params else None
    if rows == 0:
        if want_params:
            dp.zero_()
    elif want_x or want_params:
        r2 = None if g_residual is None else _rows(g_residual, d)
        scale = scale.contiguous()
        L, P, code = _lib.lib(), _lib.ptr, _DTYPES[s.dtype]
        with _lib.on_device(s.device):
            ws = None
            if want_params:
                ws = torch.empty(L.mpl_layer_norm_bwd_workspace_bytes(rows, d, code), dtype=torch.uint8, device=s.device)
            _lib.check(L.mpl_layer_norm_bwd(
                g2.data_ptr(), _pitch(g2), s2.data_ptr(), _pitch(s2), P(r2), 0 if r2 is None else _pitch(r2), code,
                scale.data_ptr(), _DTYPES[scale.dtype], mean.data_ptr(), rstd.data_ptr(), rows, d, P(dx),
                dp[0].data_ptr() if want_params else None, dp[1].data_ptr() if want_params else None, P(ws),
                ws.numel() if want_params else 0, _lib.stream_ptr(s.device)), "mpl_layer_norm_bwd")
    return (None if dx is None else dx.view(s.shape)), *((dp[0], dp[1]) if want_params else (None, None))


def _capturing() -> bool:
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


_NO_CAPTURE = ("torch autograd through layer_norm is not supported under HIP graph capture: use layer_norm_forward and "
               "layer_norm_backward, which capture")


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, eps, residual):
        y, total, mean, rstd = _forward(x, scale, bias, eps, residual, True)
        # the sum is an output: saved as one, it keeps no cycle
        ctx.save_for_backward(x if residual is None else total, scale, mean, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_y, g_sum=None):
        if _capturing():
            raise RuntimeError(_NO_CAPTURE)
        s, scale, mean, rstd = ctx.saved_tensors
        nx, ns, nb, _, nr = ctx.needs_input_grad
        if g_y is None:  # only the sum was used
            return (g_sum if nx else None), None, None, None, (g_sum if nr else None)
        dx, ds, db = _backward(g_y, s, scale, mean, rstd, g_sum, nx or nr, ns or nb)
        return (dx if nx else None), (ds if ns else None), (db if nb else None), None, (dx if nr else None)


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
    Inside a captured HIP graph use layer_norm_forward and layer_norm_backward."""
    others = () if residual is None else (("residual", residual),)
    _check("layer_norm", x, (("scale", scale), ("bias", bias)), others)
    if torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or bias.requires_grad
                                    or residual is not None and residual.requires_grad):
        if _capturing():
            raise RuntimeError(_NO_CAPTURE)
        return _LayerNormFunction.apply(x, scale, bias, float(eps), residual)
    y, total, _, _ = _forward(x, scale, bias, eps, residual, False)
    return y if residual is None else (y, total)


def layer_norm_forward(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor, eps: float = LN_EPS, *,
                       residual: Optional[torch.Tensor] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """layer_norm outside autograd: (y, s, mean, rstd), what layer_norm_backward
    takes: s is x, or x + residual; mean and rstd are fp32 [rows]."""
    others = () if residual is None else (("residual", residual),)
    _check("layer_norm_forward", x, (("scale", scale), ("bias", bias)), others)
    with torch.no_grad():
        y, total, mean, rstd = _forward(x, scale, bias, eps, residual, True)
    return y, (x if residual is None else total), mean, rstd


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
    with torch.no_grad():
        return _backward(g_y, s, scale, mean, rstd, g_residual, True, True)
