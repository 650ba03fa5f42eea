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


def _rows(t: torch.Tensor, d: int) -> Tuple[torch.Tensor, int]:
    """``t`` as rows of d elements next to each other, and the elements from
    row to row (at least d); copied only where it does not lie so."""
    if t.is_contiguous():
        return t, d
    t = t.reshape(-1, d)
    if d > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < d:
        return t.contiguous(), d
    return t, t.stride(0) if t.shape[0] > 1 else d


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
    """(y, sum or None, statistics [2, rows] or None) of x [..., d] and its parameters, checked."""
    d, dev = x.shape[-1], x.device
    rows = x.numel() // d
    x2, x_pitch = _rows(x, d)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    r2, r_pitch, total = None, 0, None
    if residual is not None:
        r2, r_pitch = _rows(residual, d)
        total = torch.empty(x.shape, dtype=x.dtype, device=dev)
    st = torch.empty((2, rows), dtype=torch.float32, device=dev) if stats else None
    if rows:
        scale, bias = scale.contiguous(), bias.contiguous()
        P = _lib.ptr
        mean = P(st)
        with _lib.on_device(dev):
            _lib.check(_lib.lib().mpl_layer_norm(
                x2.data_ptr(), x_pitch, P(r2), r_pitch, _DTYPES[x.dtype], scale.data_ptr(), bias.data_ptr(),
                _DTYPES[scale.dtype], rows, d, eps, y.data_ptr(), P(total), mean, mean and mean + 4 * rows,
                _lib.stream_ptr(dev)), "mpl_layer_norm")
    return y, total, st


def _backward(g_y, s, scale, mean: int, rstd: int, g_residual, want_x: bool, want_params: bool):
    """(dx, d_scale, d_bias), None where not wanted; mean and rstd are the addresses of fp32 [rows]."""
    d, dev = s.shape[-1], s.device
    rows = s.numel() // d
    dx = torch.empty(s.shape, dtype=s.dtype, device=dev) if want_x else None
    ds = db = ws = None
    if want_params:
        new = torch.empty if rows else torch.zeros
        ds, db = new(d, dtype=scale.dtype, device=dev), new(d, dtype=scale.dtype, device=dev)
    if rows and (want_x or want_params):
        (s2, s_pitch), (g2, g_pitch) = _rows(s, d), _rows(g_y, d)
        r2, r_pitch = (None, 0) if g_residual is None else _rows(g_residual, d)
        scale = scale.contiguous()
        L, P, code, n = _lib.lib(), _lib.ptr, _DTYPES[s.dtype], 0
        with _lib.on_device(dev):
            if want_params:
                n = L.mpl_layer_norm_bwd_workspace_bytes(rows, d, code)
                ws = torch.empty(n, dtype=torch.uint8, device=dev)
            _lib.check(L.mpl_layer_norm_bwd(
                g2.data_ptr(), g_pitch, s2.data_ptr(), s_pitch, P(r2), r_pitch, code, scale.data_ptr(),
                _DTYPES[scale.dtype], mean, rstd, rows, d, P(dx), P(ds), P(db), P(ws), n, _lib.stream_ptr(dev)),
                "mpl_layer_norm_bwd")
    return dx, ds, db


def _capturing() -> bool:
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


_NO_CAPTURE = ("torch autograd through layer_norm is not supported under HIP graph capture: use layer_norm_forward and "
               "layer_norm_backward, which capture")


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, eps, residual):
        y, total, stats = _forward(x, scale, bias, eps, residual, True)
        # the sum is an output: saved as one, it keeps no cycle
        ctx.save_for_backward(x if residual is None else total, scale, stats)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_y, g_sum=None):
        if _capturing():
            raise RuntimeError(_NO_CAPTURE)
        s, scale, stats = ctx.saved_tensors
        nx, ns, nb, _, nr = ctx.needs_input_grad
        if g_y is None:  # only the sum was used
            return (g_sum if nx else None), None, None, None, (g_sum if nr else None)
        mean = stats.data_ptr()
        dx, ds, db = _backward(g_y, s, scale, mean, mean + 2 * stats.numel(), g_sum, nx or nr, ns or nb)
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
    y, total, _ = _forward(x, scale, bias, float(eps), residual, False)
    return y if residual is None else (y, total)


def layer_norm_forward(x: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor, eps: float = LN_EPS, *,
                       residual: Optional[torch.Tensor] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """layer_norm outside autograd: (y, s, mean, rstd), what layer_norm_backward
    takes: s is x, or x + residual; mean and rstd are fp32 [rows]."""
    others = () if residual is None else (("residual", residual),)
    _check("layer_norm_forward", x, (("scale", scale), ("bias", bias)), others)
    with torch.no_grad():
        y, total, stats = _forward(x, scale, bias, float(eps), residual, True)
    return y, (x if residual is None else total), *stats.unbind(0)


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
        return _backward(g_y, s, scale, mean.data_ptr(), rstd.data_ptr(), g_residual, True, True)
