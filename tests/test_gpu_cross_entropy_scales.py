"""vocab_cross_entropy where rows, words and token weights are of unlike size.

Tolerances as in test_gpu_cross_entropy.py, but with the ends of fp16's range
where the operands' own powers of two put them:

  z        2^-39 of a row's largest and 2^-33 of a word's (32 words may share the
           power of the largest where theirs are within 2^-6 of it); fp32 calls,
           16-bit ones multiply their operands as they are
  lse      twice sum_v p z's error (the weights shift by less than half), and
           2^-20 (1 + |lse|)
  dz       2^-38 of the token's own largest coefficient
  d h      the table to 2^-39 of its largest entry (fp32 and bf16 calls)
  d e      hidden rows times their tokens' coefficients, in dz's powers of two
           (each within a factor of 2 of the largest coefficient, so 4 for a
           quotient of two), to 2^-39 of the largest such product
"""

import math

import pytest
import torch

from tests.test_gpu_cross_entropy import IGNORE, DTYPES, _inputs, _near

pytestmark = pytest.mark.gpu

SIZES = [(torch.float16, 1e4)] + [(t, s) for t in (torch.float32, torch.bfloat16) for s in (1e4, 1e8, 1e13)]


def _formula(h, e, t, gl):
    dtype, (R, d), V = h.dtype, h.shape, e.shape[0]
    u = torch.finfo(dtype).eps / 2
    fp32 = dtype == torch.float32
    H, E = h.double(), e.double()
    hm, em = H.abs().amax(1), E.abs().amax(1)
    z = H @ E.t()
    z_tol = (d * 2.0 ** -24 + (2.0 ** -21 if fp32 else 0)) * (H.abs() @ E.abs().t())
    if fp32:
        z_tol = z_tol + (2.0 ** -33 * em[None] * H.abs().sum(1)[:, None]
                         + 2.0 ** -39 * hm[:, None] * E.abs().sum(1)[None])
    lse = torch.logsumexp(z, 1)
    soft = torch.exp(z - lse[:, None])
    lse_tol = 2 * (soft * z_tol).sum(1) + 2.0 ** -20 * (1 + lse.abs())
    keep = t != IGNORE
    at = torch.where(keep, t, 0)[:, None]
    zt, zt_tol = z.gather(1, at)[:, 0], z_tol.gather(1, at)[:, 0]
    loss = torch.where(keep, lse - zt, 0.0)
    g = torch.where(keep, gl.double(), 0.0)
    p = soft * g[:, None]
    dz = p.clone().scatter_add_(1, at, -g[:, None])
    own = g.abs()
    dz_tol = (p.abs() * (z_tol + lse_tol[:, None] + 2.0 ** -20) + dz.abs() * 2.0 ** (-22 if fp32 else -11)
              + (2.0 ** -38 * own + 2.0 ** -126 * own.clamp_max(1.0))[:, None])

    def product(x, x_tol, y, K):
        out = x @ y
        acc = K * 2.0 ** -24 + (2.0 ** -21 if fp32 else 0)
        floor = 2.0 ** -126 * (K + 1) + (2.0 ** -25 if dtype == torch.float16 else 0)
        return out, (x_tol + acc * x.abs()) @ y.abs() + u * out.abs() + floor

    dh, dh_tol = product(dz, dz_tol, E, V)
    if dtype != torch.float16:
        dh_tol = dh_tol + 2.0 ** -39 * em.max() * dz.abs().sum(1)[:, None]
    Hg = torch.where(own[:, None] > 0, H, 0.0)
    de, de_tol = product(dz.t().contiguous(), dz_tol.t().contiguous(), Hg, R)
    share = torch.where(own[:, None] > 0, dz.abs() / own[:, None].clamp_min(1e-300), 0.0)
    de_tol = de_tol + 4 * 2.0 ** -39 * (own * Hg.abs().amax(1)).max() * share.sum(0)[:, None]
    return {"loss": (loss, lse_tol + zt_tol + 2.0 ** -23 * zt.abs()), "lse": (lse, lse_tol), "dh": (dh, dh_tol),
            "de": (de, de_tol)}


def _check(got, want, rows=slice(None)):
    for name, x in zip(("loss", "lse", "dh", "de"), got):
        ref, tol = want[name]
        if name == "de":
            _near(name, x, (ref, tol))
        else:
            _near(name, x[rows], (ref[rows], tol[rows]))


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("ignored", [False, True])
@pytest.mark.parametrize("R,V,d", [(20, 300, 64), (100, 700, 96), (300, 2000, 128)])
def test_one_large_row(gpu_lib, R, V, d, ignored, size, dtype):
    """A token whose hidden row is far from the others' size (a diverged one, or
    what stands in padding) changes no other token's loss and gradient."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    print(f"one large row R={R} V={V} d={d} {dtype} {size} ignored={ignored}", flush=True)
    h, e, t, gl, _ = _inputs(R, V, d, dtype, ignored=0.1)
    t[:3] = torch.tensor([5, 6, 7], device="cuda")
    t[R - 2] = IGNORE if ignored else 8
    plain = vocab_cross_entropy_grads(h, e, t, gl)
    h2 = h.clone()
    h2[R - 2] *= size
    got = vocab_cross_entropy_grads(h2, e, t, gl)
    others = torch.arange(R, device="cuda") != R - 2
    for a, b in zip(plain[:3], got[:3]):
        assert torch.equal(a[others], b[others])
    if ignored:
        assert torch.equal(plain[3], got[3])
        return
    # what the large row itself adds to the words is as uncertain as its logits
    want = _formula(h2, e, t, gl)
    _check(got, want, others)


@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("R,V,d", [(20, 300, 64), (100, 700, 96), (300, 2000, 128)])
def test_one_large_word(gpu_lib, R, V, d, size, dtype):
    """A word that its row bans (a large negative logit of every token) leaves
    the other words' logits as they are; one with a row of nearly 0 too."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(R, V, d, dtype)
    h[:, 3] = h[:, 3].abs() + 1
    t[t == 11] = 12
    e[11] = 0
    e[11, 3] = -size
    e[12] = e[12] / size
    got = vocab_cross_entropy_grads(h, e, t, gl)
    _check(got, _formula(h, e, t, gl))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.5, 3.0, 9.0])
@pytest.mark.parametrize("R,V,d", [(40, 300, 64), (100, 701, 96), (300, 2000, 128), (4100, 4300, 40)])
def test_words_and_rows_of_every_size(gpu_lib, R, V, d, spread, dtype):
    """Sizes of words and rows by powers of ten: some fragments of 32 words share a
    power of two, some do not."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(R, V, d, dtype)
    gen = torch.Generator(device="cuda").manual_seed(8)
    some = torch.rand((V, 1), generator=gen, device="cuda") < 0.3
    some[V // 2:] = False
    e = torch.where(some, e * 10 ** (spread * (torch.rand((V, 1), generator=gen, device="cuda") * 2 - 1)), e).to(dtype)
    e[5] = 0
    h = (h * 10 ** (spread * (torch.rand((R, 1), generator=gen, device="cuda") * 2 - 1))).to(dtype)
    _check(vocab_cross_entropy_grads(h, e, t, gl), _formula(h, e, t, gl))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("least", [2.0 ** -12, 2.0 ** -24, 2.0 ** -60])
@pytest.mark.parametrize("R,V,d", [(30, 300, 64), (100, 700, 96), (300, 2000, 128), (257, 40000, 320)])
def test_weights_of_unlike_size(gpu_lib, R, V, d, least, dtype):
    """Each token's d hidden is judged by its own size, however small its weight beside the others'."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    print(f"token weights R={R} V={V} d={d} {dtype} {least}", flush=True)
    h, e, t, gl, _ = _inputs(R, V, d, dtype)
    if dtype == torch.float16:  # d hidden within fp16's normal numbers
        least, gl = max(least, 2.0 ** -20), gl * 1024
    gl = gl * torch.logspace(math.log2(least), 0, R, base=2.0, device="cuda")[torch.randperm(R, device="cuda")]
    _check(vocab_cross_entropy_grads(h, e, t, gl), _formula(h, e, t, gl))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,d", [(1, 40, 64), (20, 300, 64), (40, 300, 70), (64, 900, 128), (100, 700, 96),
                                   (300, 2000, 128)])
@pytest.mark.parametrize("junk", [math.nan, math.inf, 3e4])
def test_ignored_rows_hold_anything(gpu_lib, R, V, d, junk, dtype):
    """Padding may hold NaN and infinities: the gradients are those of a call
    with zeros there, the last row (whose memory the tiles read on) among them."""
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(R, V, d, dtype, ignored=0.3)
    t[R - 1] = IGNORE
    pad = t == IGNORE
    zeros, junked = h.clone(), h.clone()
    zeros[pad] = 0
    junked[pad] = junk
    loss, lse, dh, de = vocab_cross_entropy_grads(zeros, e, t, gl)
    got = vocab_cross_entropy_grads(junked, e, t, gl)
    assert torch.equal(got[0], loss) and torch.equal(got[1][~pad], lse[~pad])
    assert torch.equal(got[2], dh) and torch.equal(got[3], de)
    assert (dh[pad] == 0).all()
    a, b = junked.clone().requires_grad_(), e.clone().requires_grad_()
    vocab_cross_entropy(a, b, t).backward(gl)
    assert torch.equal(a.grad, dh) and torch.equal(b.grad, de)


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
@pytest.mark.parametrize("R", [1, 8, 9, 16, 17, 20, 32, 33, 50, 64, 65])
@pytest.mark.parametrize("V,d", [(300, 128), (1000, 100), (700, 320), (70000, 960)])
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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,d", [(70, 300, 20000), (66, 40, 65536), (65, 33, 4100), (200, 90, 2), (130, 513, 264)])
def test_widths(gpu_lib, R, V, d, dtype):
    """Rows far wider than a team of lanes holds, and narrower than a vector."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    print(f"width R={R} V={V} d={d} {dtype}", flush=True)
    h, e, t, gl, _ = _inputs(R, V, d, dtype)
    _check(vocab_cross_entropy_grads(h, e, t, gl), _formula(h, e, t, gl))
