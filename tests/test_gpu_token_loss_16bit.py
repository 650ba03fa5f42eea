"""MemoryPoolLM.token_loss of 16-bit parameters (no memory layers: the lookup
answers in fp32, and apply() refuses the mix too) and under autocast."""

import pytest
import torch

from model_amd import model as M
from model_amd.cross_entropy import vocab_cross_entropy
from tests.test_gpu_token_loss import _leaves, _setup

pytestmark = pytest.mark.gpu


def _cast(tree, dtype):
    return {k: _cast(v, dtype) if isinstance(v, dict) else v.to(dtype) for k, v in tree.items()}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_parameters(gpu_lib, dtype):
    """The loss is that of the trunk's rows and the table as they are, bit for
    bit, its table's gradient too, and every parameter has a gradient of its type."""
    model, params, tokens, targets = _setup(use_memory=False, memory_layers=())
    params = _cast(params, dtype)
    leaves = {k: v.requires_grad_(True) for k, v in _leaves(params).items()}
    loss, lse, _ = model.token_loss(params, tokens, targets, return_lse=True)
    kw = dict(train=False, pool_off=False, route_through_pool=False, sparse_grad=False, probes=None, positions=None,
              noise_scale=1.0, shuffle_pool=False, cache=None, rngs=None)
    x, _ = model._trunk(params, tokens, M._add_layer_norm, **kw)
    assert x.dtype == dtype and loss.dtype == torch.float32
    want, want_lse = vocab_cross_entropy(x, params["embed"]["embedding"], targets, return_lse=True)
    assert torch.equal(loss, want) and torch.equal(lse, want_lse)
    a = torch.autograd.grad(loss.sum(), list(leaves.values()))
    b = torch.autograd.grad(want.sum(), list(leaves.values()))
    for k, p, q, leaf in zip(leaves, a, b, leaves.values()):
        assert p.dtype == dtype and p.shape == leaf.shape and torch.isfinite(p).all(), k
        if k != "embed/embedding" and k != "pos_embed":  # sums by atomics in torch's gather
            assert torch.equal(p, q), k


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_autocast(gpu_lib, dtype):
    """The products in between are 16-bit, the norms, rows and table stay fp32."""
    model, params, tokens, targets = _setup()
    leaves = {k: v.requires_grad_(True) for k, v in _leaves(params).items() if not k.startswith("pool/")}
    with torch.autocast("cuda", dtype):
        loss, _ = model.token_loss(params, tokens, targets)
    assert loss.dtype == torch.float32 and (loss[targets == -100] == 0).all()
    for k, g in zip(leaves, torch.autograd.grad(loss.sum(), list(leaves.values()), allow_unused=True)):
        assert g is None or (g.dtype == torch.float32 and torch.isfinite(g).all()), k
