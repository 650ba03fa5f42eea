"""The global norm of many gradients and the clip by it (train.py:395-399,
optax.global_norm over every dense gradient of a model beside the pool's sparse
rows), as libmpl.so launches (mpl_clip_grads); arguments are checked, and the
tables of tensors made, in csrc/torch/ops.cpp.

  clip_global_norm    scales the gradients in place
  global_norm_scale   the scale and the norm alone

rows.clip_scale and rows.sum_squares do the same for up to 7 and 8 fp32 tensors
without the scaling; rows.SparseRowUpdate takes either.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib


def clip_global_norm(grads: Sequence[torch.Tensor], grad_clip: float, *,
                     row_sq: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Scales the gradients in place by scale = min(1, grad_clip / (norm + 1e-6)),
    norm = sqrt(sum of all their squares + sum of row_sq), and returns the
    device tensor [scale, norm] (fp32), as rows.clip_scale does.

    grads are fp32, fp16 or bf16, mixed as they come, any number and any shapes
    on one GPU; such as do not lie in one piece are scaled through a copy.  No
    two may share an element, whatever their layouts, and none may be expanded.
    row_sq (fp32, any shape) are squares that join the norm: MergedRows.row_sq of
    the sparse rows, whose update takes the scale.  Squares are summed in fp64 in
    a fixed order, and x scale is rounded once to x's type; where scale is 1 the
    values stay as they are, and nothing is written but the copies' own.
    A norm that is not finite gives NaN or zero, as the formula does.  No host
    read, no atomics: it may be captured in a HIP graph."""
    return _lib.ops().clip_global_norm(list(grads), float(grad_clip), row_sq)


def global_norm_scale(grads: Sequence[torch.Tensor], grad_clip: float, *,
                      row_sq: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[scale, norm] of clip_global_norm, the gradients left as they are."""
    return _lib.ops().global_norm_scale(list(grads), float(grad_clip), row_sq)
