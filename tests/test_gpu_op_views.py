"""layer_norm and vocab_cross_entropy of tensors whose memory is not their value:
negated views, and zeros without memory."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _views(x):
    """x as a negated view of -x, as a conjugate's imaginary part."""
    z = torch.complex(torch.zeros_like(x), -x).conj().imag
    n = torch._neg_view(-x)
    assert z.is_neg() and n.is_neg() and torch.equal(z, x) and torch.equal(n, x)
    return z, n


@pytest.mark.parametrize("rows,d", [(5, 40), (1, 1), (7, 1)])
def test_negated(gpu_lib, rows, d):
    from model_amd.cross_entropy import vocab_cross_entropy_grads
    from model_amd.layer_norm import layer_norm_backward, layer_norm_forward

    x, r, gy = (torch.randn(rows, d, device="cuda") for _ in range(3))
    w, b = torch.randn(d, device="cuda"), torch.randn(d, device="cuda")
    want = layer_norm_forward(x, w, b, residual=r)
    grads = layer_norm_backward(gy, want[1], w, *want[2:], g_residual=r)
    e, t = torch.randn(9, d, device="cuda"), torch.arange(rows, device="cuda")
    gl, gs = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    loss = vocab_cross_entropy_grads(x, e, t, gl, gs)
    for k in range(2):
        got = layer_norm_forward(*(_views(v)[k] for v in (x, w, b)), residual=_views(r)[k])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        got = layer_norm_backward(_views(gy)[k], want[1], _views(w)[k], *want[2:], g_residual=_views(r)[k])
        assert all(torch.equal(p, q) for p, q in zip(got, grads))
        got = vocab_cross_entropy_grads(_views(x)[k], _views(e)[k], t, _views(gl)[k], _views(gs)[k])
        assert all(torch.equal(p, q) for p, q in zip(got, loss))


def test_statistics_negated(gpu_lib):
    """layer_norm_backward's mean and rstd too."""
    from model_amd.layer_norm import layer_norm_backward, layer_norm_forward

    x, gy = torch.randn(6, 32, device="cuda"), torch.randn(6, 32, device="cuda")
    w = torch.randn(32, device="cuda")
    y, s, mean, rstd = layer_norm_forward(x, w, w)
    want = layer_norm_backward(gy, s, w, mean, rstd)
    got = layer_norm_backward(gy, s, w, torch._neg_view(-mean), torch._neg_view(-rstd))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_zeros_without_memory(gpu_lib):
    from model_amd.cross_entropy import vocab_cross_entropy_grads
    from model_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward

    x, w, b = torch.randn(6, 32, device="cuda"), torch.randn(32, device="cuda"), torch.randn(32, device="cuda")
    none = torch._efficientzerotensor((6, 32), device="cuda")
    assert torch.equal(layer_norm(none, w, b), layer_norm(torch.zeros_like(x), w, b))
    _, s, mean, rstd = layer_norm_forward(x, w, b)
    assert all(torch.equal(p, torch.zeros_like(p)) for p in layer_norm_backward(none, s, w, mean, rstd))
    e, t = torch.randn(9, 32, device="cuda"), torch.arange(6, device="cuda")
    gl = torch._efficientzerotensor((6,), device="cuda")
    _, _, dh, de = vocab_cross_entropy_grads(x, e, t, gl)
    assert (dh == 0).all() and (de == 0).all()
