"""layer_norm and vocab_cross_entropy under torch's transforms: what no kernel
can follow is refused, never dropped.  No GPU: calls of no rows through the
extension module launch nothing, and take the same ways."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from model_amd import _lib

D = 8


def _calls():
    ops = _lib.ops()
    w, b, e = torch.ones(D), torch.zeros(D), torch.ones(10, D)
    ids = torch.zeros(0, dtype=torch.int64)
    st = torch.zeros(0)
    return {
        "layer_norm": lambda x: ops.layer_norm(x, w, b, 1e-6, None, False),
        "layer_norm residual": lambda x: ops.layer_norm(torch.zeros(0, D), w, b, 1e-6, x, False)[0],
        "layer_norm_forward": lambda x: ops.layer_norm_forward(x, w, b, 1e-6, None)[0],
        "layer_norm_backward": lambda x: ops.layer_norm_backward(x, torch.zeros(0, D), w, st, st, None)[0],
        "vocab_cross_entropy": lambda x: ops.vocab_cross_entropy(x, e, ids, -100, False)[0],
        "vocab_cross_entropy_grads": lambda x: ops.vocab_cross_entropy_grads(x, e, ids, st, None, -100)[2],
    }


NAMES = list(("layer_norm", "layer_norm residual", "layer_norm_forward", "layer_norm_backward", "vocab_cross_entropy",
              "vocab_cross_entropy_grads"))


@pytest.mark.parametrize("name", NAMES)
def test_refused(name):
    f, x = _calls()[name], torch.zeros(0, D)
    f(x)  # no transform: runs
    with forward_ad.dual_level():
        f(x)  # nor has this one a tangent
        with pytest.raises(RuntimeError, match="dual tensor"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, x, check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(f)(x)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.vmap(f)(torch.zeros(3, 0, D))
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda x: f(x).sum())(x)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with FakeTensorMode() as mode:
        with pytest.raises(RuntimeError, match="cannot be traced"):
            f(mode.from_tensor(x))
    with pytest.raises(RuntimeError, match="plain tensors"):
        f(mode.from_tensor(x))
    f(x)


def test_subclasses_without_dispatch_run():
    class Named(torch.Tensor):
        pass

    x = torch.zeros(0, D).as_subclass(Named)
    for f in _calls().values():
        f(x)
    for f in _calls().values():
        f(torch.nn.Parameter(torch.zeros(0, D)))


def test_batched_gradients_are_refused():
    ops = _lib.ops()
    x = torch.zeros(0, D, requires_grad=True)
    y = ops.layer_norm(x, torch.ones(D), torch.zeros(D), 1e-6, None, True)
    loss, _ = ops.vocab_cross_entropy(x, torch.ones(10, D), torch.zeros(0, dtype=torch.int64), -100, True)
    for out in (y, loss):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, x, torch.ones(3, *out.shape), is_grads_batched=True)
