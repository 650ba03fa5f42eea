"""vocab_cross_entropy where rows, words and token weights are of unlike size."""

import math

import pytest
import torch

from tests.test_gpu_cross_entropy import DTYPES, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [40.0, 100.0, 300.0])
@pytest.mark.parametrize("R,V,d", [(12, 300, 128), (100, 300, 128), (300, 3000, 256), (70, 500, 100)])
def test_learned_tokens(gpu_lib, R, V, d, size, dtype):
    """Tokens whose target has all the probability.  With m the largest logit
    and the target's, the loss is log(1 + rest), rest = sum exp(z - m) below
    2^-25 of the target's 1: at least 0, and at most rest with its logits' errors
    (a factor of 2) and two steps of the sum and the log, 2^-22.  The target's dz
    is g (p - 1), p = 1 to two such steps more: d hidden is at most 2^-21 g of
    the target's row, and rest g of the others'."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    gen = torch.Generator(device="cuda").manual_seed(3)
    e = torch.randn((V, d), generator=gen, device="cuda")
    e = (e / e.norm(dim=1, keepdim=True)).to(dtype)
    t = torch.randint(0, V, (R,), generator=gen, device="cuda")
    h = (size * (1 + torch.rand((R, 1), generator=gen, device="cuda")) * e[t].float()).to(dtype)
    gl = torch.rand(R, generator=gen, device="cuda") + 0.5
    z = h.double() @ e.double().t()
    zt = z.gather(1, t[:, None])
    rest = (torch.exp(z - zt).sum(1) - 1).clamp_min(0)
    counted = rest < 2.0 ** -25
    assert counted.sum() > 0.7 * R
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
    assert (loss >= 0).all()
    assert (loss.double() <= 2 * rest + 2.0 ** -22)[counted].all()
    off = (lse.double() - zt[:, 0]).abs()
    assert (off <= d * 2.0 ** -24 * (h.double().abs() @ e.double().abs().t()).amax(1) + 2.0 ** -22 * zt[:, 0]).all()
    most = gl.double() * (2.0 ** -21 * e.double().abs().amax(1)[t] + 2 * rest * e.double().abs().max())
    assert (dh.double().abs().amax(1) <= most)[counted].all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e4, 1e9, 1e13])
@pytest.mark.parametrize("R", [6, 300])
def test_logits_of_any_size(gpu_lib, R, size, dtype):
    """Rows so large that one word has all the probability, to the last bit:
    with e . e of two words at most half of a word's own, the gap to the next
    logit is far above 104 (fp32's smallest exp).  Of target t and top word k the
    loss is z_k - z_t and d hidden is g (e_k - e_t), each within two roundings of
    z (2^-22 with its d products) and of the result."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    d = 64
    e = torch.eye(d, device="cuda").to(dtype)
    h = torch.zeros((R, d), dtype=dtype, device="cuda")
    rows = torch.arange(R, device="cuda")
    top, t = rows % d, (rows * 7 + rows % 2 * 3) % d
    h[rows, top] = size
    gl = torch.linspace(-1, 2, R, device="cuda")
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
    z = h.float()[rows, top].double()
    want = torch.where(t == top, 0.0, z)
    assert ((lse.double() - z).abs() <= 2.0 ** -22 * z).all() and ((loss.double() - want).abs() <= 2.0 ** -22 * want).all()
    dz = torch.zeros((R, d), dtype=torch.float64, device="cuda")
    dz[rows, top] += gl.double()
    dz[rows, t] -= gl.double()
    u = torch.finfo(dtype).eps / 2
    near = dz.abs() * (2.0 ** -11 + u) if dtype != torch.float32 else dz.abs() * 2.0 ** -20
    assert ((dh.double() - dz).abs() <= near + 2.0 ** -37).all()
    assert torch.isfinite(de).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [1, 9, 16, 17, 20, 32])
@pytest.mark.parametrize("V,d", [(300, 128), (1000, 100), (700, 320)])
def test_few_tokens_form_z_twice_alike(gpu_lib, R, V, d, dtype):
    """Learned tokens with logits of some 10^4, where another order of z's sum is
    off by 2^-24 of that: p is exactly 1 where the backward's z has the forward's
    bits, and every gradient exactly 0 (the other words are 104 and more below)."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    gen = torch.Generator(device="cuda").manual_seed(4)
    e = torch.randn((V, d), generator=gen, device="cuda")
    e = (e / e.norm(dim=1, keepdim=True)).to(dtype)
    t = torch.randint(0, V, (R,), generator=gen, device="cuda")
    h = (3e4 * e[t].float()).to(dtype)
    z = h.double() @ e.double().t()
    z.scatter_(1, t[:, None], -math.inf)
    assert (z.amax(1) < 3e4 - 200).all()
    loss, _, dh, de = vocab_cross_entropy_grads(h, e, t, torch.ones(R, device="cuda"))
    assert (loss == 0).all() and (dh == 0).all() and (de == 0).all()
