"""vocab_cross_entropy and its gradients against the formula in 64 bits.

Tolerances, elementwise, from the arithmetic (u = half a step of the type,
torch.finfo(t).eps / 2):

  z       sums of d products in fp32: d 2^-24 of sum |h e|; fp32 operands are
          held to 2^-23 each and lo lo (2^-22) is left out: 2^-21 more; where
          operands are held in fp16 (fp32 calls, bf16's gradients), 2^-39 of
          their array's largest, the end of fp16's range under its power of two
  lse     the largest z error, and 2^-20 (1 + |lse|): exp, log and the sums of the
          exps, relative to a sum whose error the log turns into an absolute one
  dz      |z error| + |lse error| + 2^-20 relative (exp of both), one rounding to
          fp16, 2^-11 (fp32 calls: hi and lo, 2^-22), and half of fp16's smallest
          step under dz's power of two, 2^-25 2^-13 of the largest coefficient;
          below 2^-126, fp32's smallest normal number, exp gives 0, so 2^-126 of
          the largest coefficient (or of 1)
  d h, d e   sum |dz error| |operand|, K 2^-24 of sum |dz| |operand| for sums of K
          products (and 2^-21 for fp32 operands, 2^-39 of the array's largest as
          above), one rounding u of the result; products and sums below 2^-126
          are 0 too: (K + 1) 2^-126
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IGNORE = -100


def _inputs(R, V, d, dtype, seed=0, ignored=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    e = (torch.randn((V, d), generator=g, device="cuda") * d ** -0.5).to(dtype)
    t = torch.randint(0, V, (R,), generator=g, device="cuda")
    h = (torch.randn((R, d), generator=g, device="cuda") + 3 * e[t].float()).to(dtype)
    t[torch.rand(R, generator=g, device="cuda") < ignored] = IGNORE
    gl = torch.randn(R, generator=g, device="cuda")
    gs = torch.randn(R, generator=g, device="cuda") * 0.3
    return h, e, t, gl, gs


def _formula(h, e, t, gl, gs):
    """loss, lse, dh, de and their tolerances, all in 64 bits."""
    dtype, (R, d), V = h.dtype, h.shape, e.shape[0]
    u = torch.finfo(dtype).eps / 2
    fp32 = dtype == torch.float32
    H, E = h.double(), e.double()
    z = H @ E.t()
    z_tol = (d * 2.0 ** -24 + (2.0 ** -21 if fp32 else 0)) * (H.abs() @ E.abs().t())
    end = 0 if dtype == torch.float16 else 2.0 ** -39
    z_tol = z_tol + end * (E.abs().max() * H.abs().sum(1)[:, None] + H.abs().max() * E.abs().sum(1)[None])
    lse = torch.logsumexp(z, 1)
    lse_tol = z_tol.amax(1) + 2.0 ** -20 * (1 + lse.abs())
    keep = t != IGNORE
    at = torch.where(keep, t, 0)[:, None]
    loss = torch.where(keep, lse - z.gather(1, at)[:, 0], 0.0)
    g = torch.where(keep, gl.double(), 0.0) if gl is not None else torch.zeros(R, dtype=torch.float64, device=h.device)
    a = g + gs.double() if gs is not None else g
    p = torch.exp(z - lse[:, None]) * a[:, None]
    dz = p.clone().scatter_add_(1, at, -g[:, None])
    most = max(a.abs().max().item(), g.abs().max().item())
    dz_tol = (p.abs() * (z_tol + lse_tol[:, None] + 2.0 ** -20) + dz.abs() * 2.0 ** (-22 if fp32 else -11)
              + 2.0 ** -38 * most + 2.0 ** -126 * max(1.0, most))

    def product(x, x_tol, y, K):
        out = x @ y
        acc = K * 2.0 ** -24 + (2.0 ** -21 if fp32 else 0)
        floor = 2.0 ** -126 * (K + 1) + (2.0 ** -25 if dtype == torch.float16 else 0)
        tol = (x_tol + acc * x.abs()) @ y.abs() + end * y.abs().max() * x.abs().sum(1)[:, None]
        return out, tol + u * out.abs() + floor

    dh, dh_tol = product(dz, dz_tol, E, V)
    de, de_tol = product(dz.t().contiguous(), dz_tol.t().contiguous(), H, R)
    return {"loss": (loss, 2 * lse_tol), "lse": (lse, lse_tol), "dh": (dh, dh_tol), "de": (de, de_tol)}


def _near(name, got, want):
    ref, tol = want
    assert got.shape == ref.shape
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    if bad.any():
        at = torch.where(bad, off / tol.clamp_min(1e-300), 0).argmax()
        pytest.fail(f"{name}: {int(bad.sum())} of {bad.numel()} off; worst: {got.reshape(-1)[at].item():.6g} for "
                    f"{ref.reshape(-1)[at].item():.6g}, tolerance {tol.reshape(-1)[at].item():.3g}")


SHAPES = [
    (1, 1, 1), (1, 7, 3), (2, 64, 32), (3, 300, 65), (31, 129, 64), (33, 1000, 100), (64, 256, 128), (65, 257, 256),
    (130, 2049, 192), (300, 511, 500), (257, 5003, 72), (1000, 700, 320), (5, 20000, 256), (512, 16384, 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,d", SHAPES)
def test_loss_and_gradients(gpu_lib, R, V, d, dtype):
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    print(f"cross entropy R={R} V={V} d={d} {dtype}", flush=True)
    h, e, t, gl, gs = _inputs(R, V, d, dtype)
    want = _formula(h, e, t, gl, gs)
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl, gs)
    for name, got in (("loss", loss), ("lse", lse), ("dh", dh), ("de", de)):
        _near(name, got, want[name])
    assert loss.dtype == lse.dtype == torch.float32 and dh.dtype == de.dtype == dtype
    assert (loss[t == IGNORE] == 0).all()
    with torch.no_grad():
        assert torch.equal(vocab_cross_entropy(h, e, t), loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,d", [(8192, 16384, 256), (4500, 9000, 1024), (16384, 4000, 128)])
def test_many_tiles(gpu_lib, R, V, d, dtype):
    """The 256 x 256 tiles of every product, ragged."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    R, V = R - 3, V - 5
    print(f"cross entropy, large R={R} V={V} d={d} {dtype}", flush=True)
    h, e, t, gl, gs = _inputs(R, V, d, dtype)
    want = _formula(h, e, t, gl, None)
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
    for name, got in (("loss", loss), ("lse", lse), ("dh", dh), ("de", de)):
        _near(name, got, want[name])


@pytest.mark.parametrize("R,V,d,dtype", [(8192, 32768 + 100, 256, torch.bfloat16), (8192, 16384 + 37, 192, torch.float32),
                                         (16384, 16384 + 300, 256, torch.float16)])
def test_short_last_piece(gpu_lib, R, V, d, dtype):
    """Two pieces of the vocabulary, the second with fewer stages than the
    first's d hidden has parts."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    print(f"cross entropy, two pieces R={R} V={V} d={d} {dtype}", flush=True)
    h, e, t, gl, _ = _inputs(R, V, d, dtype)
    t[:50] = V - 1
    want = _formula(h, e, t, gl, None)
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
    for name, got in (("loss", loss), ("lse", lse), ("dh", dh), ("de", de)):
        _near(name, got, want[name])


@pytest.mark.parametrize("h_size,e_size", [(1e-25, 1e-25), (0.0, 1e-25), (1e-30, 1e30), (0.0, 0.0)])
@pytest.mark.parametrize("R", [5, 70, 300])
def test_ends_of_fp32(gpu_lib, R, h_size, e_size):
    """Arrays whose powers of two multiply to less than fp32 holds: logits of 0."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(R, 300, 64, torch.float32)
    h, e = h / h.abs().max() * h_size, e / e.abs().max() * e_size
    if h_size * e_size < 1e-20:  # else ordinary logits
        loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
        assert (lse - math.log(300)).abs().max() <= 2 ** -20 * 7
        assert torch.isfinite(dh).all() and torch.isfinite(de).all()
    want = _formula(h, e, t, gl, None)
    for name, got in zip(("loss", "lse", "dh", "de"), vocab_cross_entropy_grads(h, e, t, gl)):
        _near(name, got, want[name])


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd_equals_direct(gpu_lib, dtype):
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    h, e, t, gl, gs = _inputs(96, 500, 96, dtype)
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl, gs)
    H, E = h.reshape(8, 12, 96).clone().requires_grad_(True), e.clone().requires_grad_(True)
    T = t.reshape(8, 12).int()
    l2, s2 = vocab_cross_entropy(H, E, T, return_lse=True)
    assert l2.shape == s2.shape == (8, 12)
    ((l2 * gl.reshape(8, 12)).sum() + (s2 * gs.reshape(8, 12)).sum()).backward()
    assert torch.equal(l2.reshape(-1), loss) and torch.equal(s2.reshape(-1), lse)
    assert torch.equal(H.grad.reshape(96, 96), dh) and torch.equal(E.grad, de)
    # one of the two gradients alone, and the logsumexp's alone
    H2 = h.clone().requires_grad_(True)
    (vocab_cross_entropy(H2, e, t) * gl).sum().backward()
    _, _, dh1, de1 = vocab_cross_entropy_grads(h, e, t, gl)
    assert torch.equal(H2.grad, dh1)
    E2 = e.clone().requires_grad_(True)
    (vocab_cross_entropy(h, E2, t, return_lse=True)[1] * gs).sum().backward()
    assert torch.equal(E2.grad, vocab_cross_entropy_grads(h, e, t, None, gs)[3])


def test_gradients_against_differences(gpu_lib):
    """d loss along a direction, by central differences of the fp32 loss: a
    step s along unit directions leaves s^2/6 |f'''| <= s^2 |x|^3 (third
    derivatives of a logsumexp are below the cube of the direction's logits,
    here at most |dir . e| <= 3) and the loss's own error / s."""
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(12, 40, 24, torch.float32, ignored=0.3)
    _, _, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
    g = torch.Generator(device="cuda").manual_seed(9)
    for x, grad, which in ((h, dh, 0), (e, de, 1)):
        way = torch.randn(x.shape, generator=g, device="cuda")
        way = way / way.norm()
        s = 2.0 ** -6
        up, down = [(x + k * s * way) for k in (1, -1)]
        args = [((a, e) if which == 0 else (h, a)) for a in (up, down)]
        f = [(vocab_cross_entropy(*a, t).double() * gl.double()).sum().item() for a in args]
        want = (grad.double() * way.double()).sum().item()
        weight = gl.abs().sum().item()
        loss_error = 2 ** -20 * 16  # of a token: z and lse of a few units
        assert abs((f[0] - f[1]) / (2 * s) - want) <= weight * (s * s * 27 / 6 + loss_error / s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_targets(gpu_lib, dtype):
    """All ignored: losses and gradients 0.  First and last word.  An id
    outside the table: NaN for its token alone, and NaN gradients."""
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    h, e, t, gl, gs = _inputs(40, 300, 64, dtype)
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, torch.full_like(t, IGNORE), gl)
    assert (loss == 0).all() and (dh == 0).all() and (de == 0).all() and torch.isfinite(lse).all()
    t = torch.where(torch.arange(40, device="cuda") % 2 == 0, 0, 299)
    want = _formula(h, e, t, gl, None)
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl, ignore_index=7)
    for name, got in (("loss", loss), ("lse", lse), ("dh", dh), ("de", de)):
        _near(name, got, want[name])
    # an ignored index inside the table
    keep = loss.clone()
    assert torch.equal(vocab_cross_entropy(h, e, t, ignore_index=299), torch.where(t == 299, 0.0, keep))
    for wrong in (300, -1, 2 ** 40):
        t2 = t.clone()
        t2[11] = wrong
        loss, _, dh, de = vocab_cross_entropy_grads(h, e, t2, gl)
        assert torch.isnan(loss[11]) and torch.equal(loss[:11], keep[:11]) and torch.equal(loss[12:], keep[12:])
        assert torch.isnan(dh[11]).all() and torch.isfinite(dh[:11]).all() and torch.isnan(de).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-6, 1.0, 300.0])
def test_sizes_of_logits(gpu_lib, dtype, size):
    """Logits near 0 and in the hundreds (a softmax of one word)."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(70, 900, 128, torch.float32)
    h = h * size if size < 100 else h * 40
    h, e = h.to(dtype), e.to(dtype)
    want = _formula(h, e, t, gl, None)
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
    for name, got in (("loss", loss), ("lse", lse), ("dh", dh), ("de", de)):
        _near(name, got, want[name])


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** 40])
def test_fp32_range(gpu_lib, scale):
    """Hidden rows and tables far from 1 whose products are ordinary: the
    powers of two are exact, so the losses have the bits of the plain call."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(50, 300, 100, torch.float32)
    a = vocab_cross_entropy_grads(h, e, t, gl)
    b = vocab_cross_entropy_grads(h * scale, e / scale, t, gl)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(a[2], b[2] * scale) and torch.equal(a[3], b[3] / scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_finite(gpu_lib, dtype):
    """A NaN or infinite hidden row is that token's loss alone; a NaN table
    entry is every token's."""
    from model_amd.cross_entropy import vocab_cross_entropy

    h, e, t, _, _ = _inputs(70, 300, 64, dtype, ignored=0.0)
    good = vocab_cross_entropy(h, e, t)
    for x in (math.nan, math.inf, -math.inf):
        h2 = h.clone()
        h2[33, 5] = x
        loss = vocab_cross_entropy(h2, e, t)
        assert torch.isnan(loss[33]) and torch.equal(loss[:33], good[:33]) and torch.equal(loss[34:], good[34:])
    e2 = e.clone()
    e2[200, 3] = math.nan
    assert torch.isnan(vocab_cross_entropy(h, e2, t)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 70])
def test_strides(gpu_lib, dtype, d):
    """Slices of wider arrays, unaligned, transposed and expanded rows equal
    the contiguous call."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, gs = _inputs(48, 200, d, dtype)
    want = vocab_cross_entropy_grads(h, e, t, gl, gs)

    def same(h2, e2, t2=t):
        got = vocab_cross_entropy_grads(h2, e2, t2, gl, gs)
        for x, y in zip(got, want):
            assert torch.equal(x, y)

    wide = torch.zeros((48, d + 24), dtype=dtype, device="cuda")
    for at in (8, 3):
        wide[:, at:at + d] = h
        same(wide[:, at:at + d], e)
        table = torch.zeros((200, d + 24), dtype=dtype, device="cuda")
        table[:, at:at + d] = e
        same(h, table[:, at:at + d])
    same(h.t().contiguous().t(), e.t().contiguous().t())
    shifted = torch.zeros(48 * d + 1, dtype=dtype, device="cuda")
    shifted[1:] = h.reshape(-1)
    same(shifted[1:].reshape(48, d), e)
    every = torch.stack([t, t], 1)
    same(h, e, every[:, 0])
    one = h[:1].expand(48, d)
    a = vocab_cross_entropy_grads(one, e, t, gl, gs)
    b = vocab_cross_entropy_grads(one.contiguous(), e, t, gl, gs)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_no_rows(gpu_lib):
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    h = torch.zeros((0, 64), device="cuda", requires_grad=True)
    e = torch.randn((10, 64), device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.int64, device="cuda")
    loss = vocab_cross_entropy(h, e, t)
    assert loss.shape == (0,)
    loss.sum().backward()
    assert h.grad.shape == (0, 64) and (e.grad == 0).all()
    _, _, dh, de = vocab_cross_entropy_grads(h, e, t, torch.zeros(0, device="cuda"))
    assert dh.shape == (0, 64) and (de == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeats_bit_for_bit(gpu_lib, dtype):
    """Same bits in every call, whatever lay in the workspaces before."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, gs = _inputs(777, 3001, 136, dtype)
    first = vocab_cross_entropy_grads(h, e, t, gl, gs)
    for _ in range(4):
        junk = torch.full((64 << 20,), math.nan, device="cuda")
        del junk
        again = vocab_cross_entropy_grads(h, e, t, gl, gs)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured(gpu_lib, dtype):
    """Loss and gradients in a HIP graph, replayed with new inputs between
    eager calls, equal the eager ones."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, gs = _inputs(200, 1000, 96, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        vocab_cross_entropy_grads(h, e, t, gl, gs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = vocab_cross_entropy_grads(h, e, t, gl, gs)
    for seed in range(4):
        new = _inputs(200, 1000, 96, dtype, seed=seed + 20)
        for x, y in zip((h, e, t, gl, gs), new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = vocab_cross_entropy_grads(*new)
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_autograd_refused_under_capture(gpu_lib):
    """As the lookup refuses it: a captured autograd step of leaves that an
    eager graph holds ends the process."""
    from model_amd import cross_entropy as ce

    h, e, t, _, _ = _inputs(8, 20, 64, torch.float32)
    h.requires_grad_(True)
    from model_amd import _lib

    saved = ce._capturing
    try:
        loss = ce.vocab_cross_entropy(h, e, t)
        ce._capturing = lambda: True
        with pytest.raises(RuntimeError, match="vocab_cross_entropy_grads"):
            ce.vocab_cross_entropy(h, e, t)
        _lib.ops().pretend_capturing(True)
        with pytest.raises(RuntimeError, match="vocab_cross_entropy_grads"):
            loss.sum().backward()
    finally:
        ce._capturing = saved
        _lib.ops().pretend_capturing(False)


def test_two_streams(gpu_lib):
    """Calls on two streams at once: each has its own workspace."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    a, b = (_inputs(600, 4000, 128, torch.bfloat16, seed=s) for s in (1, 2))
    want = [vocab_cross_entropy_grads(*x) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append(vocab_cross_entropy_grads(*x))
    torch.cuda.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_changed_in_place_is_refused(gpu_lib):
    from model_amd.cross_entropy import vocab_cross_entropy

    h, e, t, _, _ = _inputs(8, 20, 64, torch.float32)
    x = h.clone().requires_grad_(True) * 1
    loss = vocab_cross_entropy(x, e, t)
    x.data_ptr()
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


def test_second_derivative_is_refused(gpu_lib):
    """Under create_graph the gradients are there, and raise when they are
    differentiated again."""
    from model_amd.cross_entropy import vocab_cross_entropy

    h, e, t, gl, _ = _inputs(8, 20, 64, torch.float32)
    h.requires_grad_(True)
    loss = (vocab_cross_entropy(h, e, t) * gl).sum()
    g, = torch.autograd.grad(loss, h, create_graph=True)
    plain, = torch.autograd.grad((vocab_cross_entropy(h, e, t) * gl).sum(), h)
    assert torch.equal(g.detach(), plain)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def _far(x, pitch):
    """x with its rows `pitch` elements apart, in a buffer of more than 2^32 bytes."""
    out = torch.empty(x.shape[0] * pitch, dtype=x.dtype, device="cuda").reshape(x.shape[0], pitch)[:, :x.shape[1]]
    out.copy_(x)
    return out


@pytest.mark.parametrize("dtype,R,d", [(torch.float32, 5, 40), (torch.float32, 300, 40), (torch.float16, 300, 128),
                                       (torch.bfloat16, 9, 128), (torch.bfloat16, 300, 70)])
def test_offsets_past_32_bits(gpu_lib, dtype, R, d):
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    print(f"cross entropy, far rows R={R} d={d} {dtype}", flush=True)
    h, e, t, gl, gs = _inputs(R, 300, d, dtype)
    want = vocab_cross_entropy_grads(h, e, t, gl, gs)
    pitch = 1 << 22 if dtype == torch.float32 else (1 << 23) - 8
    far_e = _far(e, pitch)
    assert 299 * pitch * e.element_size() > 1 << 32
    for x, y in zip(vocab_cross_entropy_grads(h, far_e, t, gl, gs), want):
        assert torch.equal(x, y)
    if R == 300:
        far_h = _far(h, pitch)
        for x, y in zip(vocab_cross_entropy_grads(far_h, far_e, t, gl, gs), want):
            assert torch.equal(x, y)


def test_table_past_2_32_elements(gpu_lib):
    """The last words of a table of more than 2^32 elements: the others are zeros, logits of 0."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    V, d, R = (1 << 24) + 300, 256, 20
    print(f"cross entropy, V={V} d={d}", flush=True)
    h, small, t, gl, gs = _inputs(R, 300, d, torch.bfloat16, ignored=0.0)
    e = torch.zeros((V, d), dtype=torch.bfloat16, device="cuda")
    e[-300:] = small
    loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t + (1 << 24), gl, gs)
    H, E = h.double(), small.double()
    z = H @ E.t()
    ref = torch.logsumexp(torch.cat([z, torch.full((R, 1), math.log(V - 300), device="cuda", dtype=torch.float64)], 1), 1)
    at = t[:, None]
    z_tol = d * 2.0 ** -24 * (H.abs() @ E.abs().t()) + 2.0 ** -39 * (
        E.abs().max() * H.abs().sum(1)[:, None] + H.abs().max() * E.abs().sum(1)[None])
    lse_tol = z_tol.amax(1) + 2.0 ** -20 * (1 + ref)
    _near("lse", lse, (ref, lse_tol))
    _near("loss", loss, (ref - z.gather(1, at)[:, 0], 2 * lse_tol))
    # the gradients of the last words; the zeros add nothing to dh, and get the sum of their own dz
    g, a = gl.double(), (gl + gs).double()
    most = max(g.abs().max().item(), a.abs().max().item())
    p = torch.exp(z - ref[:, None]) * a[:, None]
    dz = p.scatter_add(1, at, -g[:, None])
    dz_tol = p.abs() * (z_tol + lse_tol[:, None] + 2.0 ** -20) + dz.abs() * 2.0 ** -11 + 2.0 ** -38 * most
    zero = torch.exp(-ref) * a
    zero_tol = zero.abs() * (lse_tol + 2.0 ** -20 + 2.0 ** -11) + 2.0 ** -38 * most

    def product(x, x_tol, y, K):
        out = x @ y
        return out, ((x_tol + K * 2.0 ** -24 * x.abs()) @ y.abs() + 2.0 ** -39 * y.abs().max() * x.abs().sum(-1, keepdim=True)
                     + 2.0 ** -8 * out.abs())

    _near("dh", dh, product(dz, dz_tol, E, 300))
    _near("de", de[-300:], product(dz.t().contiguous(), dz_tol.t().contiguous(), H, R))
    for row in (0, 1 << 20, (1 << 24) - 1):
        _near("de of zeros", de[row], product(zero, zero_tol, H, R))


def test_one_tensor_as_both(gpu_lib):
    """The table's own rows as hidden: both gradients reach the one leaf."""
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    _, e, _, _, _ = _inputs(1, 200, 96, torch.float32)
    t = torch.arange(200, device="cuda")
    gl = torch.linspace(-1, 1, 200, device="cuda")
    leaf = e.clone().requires_grad_()
    vocab_cross_entropy(leaf, leaf, t).backward(gl)
    _, _, dh, de = vocab_cross_entropy_grads(e, e, t, gl)
    assert torch.equal(leaf.grad, dh + de)


def test_two_threads(gpu_lib):
    """Autograd steps in two threads, each on a stream of its own."""
    import threading

    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    args = [_inputs(500, 3000, 128, torch.float16, seed=s) for s in (3, 4)]
    want = [vocab_cross_entropy_grads(h, e, t, gl) for h, e, t, gl, _ in args]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        h, e, t, gl, _ = args[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                a, b = h.clone().requires_grad_(), e.clone().requires_grad_()
                loss = vocab_cross_entropy(a, b, t)
                loss.backward(gl)
            torch.cuda.current_stream().synchronize()
            got[i] = (loss.detach(), a.grad, b.grad)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    for (loss, _, dh, de), g in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip((loss, dh, de), g))


def test_memory_is_freed(gpu_lib):
    from model_amd.cross_entropy import vocab_cross_entropy

    h, e, t, gl, _ = _inputs(300, 3000, 128, torch.bfloat16)
    h.requires_grad_(), e.requires_grad_()

    def step(backward):
        loss, lse = vocab_cross_entropy(h, e, t, return_lse=True)
        if backward:
            (loss + lse).sum().backward()
            h.grad = e.grad = None

    used = []
    for i in range(6):
        step(i % 2)
        torch.cuda.synchronize()
        used.append(torch.cuda.memory_allocated())
    assert used[4] == used[2] and used[5] == used[3]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,d", [(1, 1, 4), (1, 33, 5), (7, 31, 127), (8, 64, 128), (16, 1000, 129), (17, 300, 64),
                                   (32, 5003, 257), (33, 70, 130), (40, 2000, 6), (64, 3001, 384), (64, 40000, 40)])
def test_few_tokens(gpu_lib, R, V, d, dtype):
    """Blocks of tokens, groups of words and columns that end anywhere; the
    gradients of both outputs and of either."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    print(f"cross entropy, few tokens R={R} V={V} d={d} {dtype}", flush=True)
    h, e, t, gl, gs = _inputs(R, V, d, dtype)
    t[0] = V - 1
    for a, b in ((gl, gs), (gl, None), (None, gs)):
        want = _formula(h, e, t, a, b)
        for name, got in zip(("loss", "lse", "dh", "de"), vocab_cross_entropy_grads(h, e, t, a, b)):
            _near(name, got, want[name])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [3, 40, 100])
def test_one_of_the_gradients(gpu_lib, R, dtype):
    """A frozen table, or frozen rows: the other's gradient is the same, and nothing else is written."""
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(R, 700, 72, dtype)
    _, _, dh, de = vocab_cross_entropy_grads(h, e, t, gl)
    a, b = h.clone().requires_grad_(), e.clone().requires_grad_()
    vocab_cross_entropy(a, e, t).backward(gl)
    vocab_cross_entropy(h, b, t).backward(gl)
    assert torch.equal(a.grad, dh) and torch.equal(b.grad, de)


@pytest.mark.parametrize("R", [20, 60])
def test_few_tokens_leave_the_rest(gpu_lib, R):
    """The C entry writes d hidden and d embedding and nothing behind them."""
    from model_amd import _lib
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    h, e, t, gl, _ = _inputs(R, 333, 70, torch.float32)
    _, lse, want_h, want_e = vocab_cross_entropy_grads(h, e, t, gl)
    L = _lib.lib()
    n = L.mpl_vocab_cross_entropy_workspace_bytes(R, 333, 70, _lib.MPL_F32, 1)
    ws = torch.full((n + 1024,), 77, dtype=torch.uint8, device="cuda")
    dh, de = (torch.full(((rows + 1) * 70,), 7.0, device="cuda") for rows in (R, 333))
    _lib.check(L.mpl_vocab_cross_entropy_bwd(h.data_ptr(), 70, e.data_ptr(), 70, _lib.MPL_F32, t.data_ptr(), R, 333, 70,
                                             IGNORE, lse.data_ptr(), gl.data_ptr(), None, ws.data_ptr(), n,
                                             dh.data_ptr(), de.data_ptr(), _lib.stream_ptr(h.device)))
    assert torch.equal(dh[:R * 70].view(R, 70), want_h) and torch.equal(de[:333 * 70].view(333, 70), want_e)
    assert (dh[R * 70:] == 7).all() and (de[333 * 70:] == 7).all() and (ws[n:] == 77).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R", [8, 50, 200])
def test_two_graphs(gpu_lib, R, dtype):
    """Two captured graphs replayed in turn and on two streams at once, between
    eager calls, equal the eager ones."""
    from model_amd.cross_entropy import vocab_cross_entropy_grads

    args = [_inputs(R, 1500, 128, dtype, seed=s) for s in (5, 6)]
    want = [vocab_cross_entropy_grads(*x) for x in args]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(vocab_cross_entropy_grads(*x))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for out in outs:
            for x in out:
                x.fill_(math.nan)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            if turn % 2:
                with torch.cuda.stream(stream):
                    graph.replay()
            else:
                graph.replay()
                vocab_cross_entropy_grads(*args[0])
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(out, ref))
