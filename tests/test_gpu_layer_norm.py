"""layer_norm and its backward pass against the formula in 64 bits.

Tolerances, elementwise, from the arithmetic (u = half a step of the type; a
sum over a row is at most 64 additions in a row of terms, so 2^-18 of the sum
of magnitudes):

  mean     2^-18 mean|s|
  rstd     relative: half of 2^-18 (the variance's sum), of the square of the
           mean's error over sigma, and of twice 2^-23 max|s| / sigma (the
           deviations' roundings); 2^-22 for the root and the quotient
  x_hat    |x_hat| of rstd's and 2^-22, and (mean's error + 2^-23 max|s|) rstd
  y        |scale| x_hat's, 2^-22 (|y| + |bias|), one rounding u
  d x      the two row means: 2^-18 of the mean magnitudes and x_hat's error;
           their products, 2^-21 of every term, rstd's error, one rounding u
  d scale, d bias   (64 + rows / 64) 2^-24 of the sum of magnitudes, x_hat's error,
           one rounding u
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-6


def _inputs(R, d, dtype, param=torch.float32, add=False, seed=0, offset=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = (rnd(R, d) * (0.5 + rnd(R, 1).abs()) + offset * rnd(R, 1)).to(dtype)
    r = rnd(R, d).to(dtype) if add else None
    return (x, (1 + 0.3 * rnd(d)).to(param), (0.2 * rnd(d)).to(param), r, rnd(R, d).to(dtype),
            rnd(R, d).to(dtype) if add else None)


def _formula(x, scale, bias, r, gy, gs, eps=EPS):
    u = torch.finfo(x.dtype).eps / 2
    up = torch.finfo(scale.dtype).eps / 2
    floor = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -126
    s = x if r is None else (x.double() + r.double()).to(x.dtype)  # exact in 64 bits, then rounded once
    R, d = s.shape
    S, w, b, g = s.double(), scale.double(), bias.double(), gy.double()
    mean = S.mean(1, keepdim=True)
    dev = S - mean
    sigma = (dev.square().mean(1, keepdim=True) + eps).sqrt()
    rstd = 1 / sigma
    hat = dev * rstd
    big = S.abs().amax(1, keepdim=True)
    mean_e = 2.0 ** -18 * S.abs().mean(1, keepdim=True)
    rstd_e = 0.5 * (2.0 ** -18 + (mean_e * rstd) ** 2 + 2 * 2.0 ** -23 * big * rstd) + 2.0 ** -22
    hat_e = hat.abs() * (rstd_e + 2.0 ** -22) + (mean_e + 2.0 ** -23 * big) * rstd
    y = hat * w + b
    out = {"y": (y, w.abs() * hat_e + 2.0 ** -22 * (y.abs() + b.abs()) + u * y.abs() + floor),
           "mean": (mean[:, 0], mean_e[:, 0] + 2.0 ** -23 * mean[:, 0].abs()), "rstd": (rstd[:, 0], (rstd * rstd_e)[:, 0])}
    gh = g * w
    a, c = gh.mean(1, keepdim=True), (gh * hat).mean(1, keepdim=True)
    a_e = 2.0 ** -18 * gh.abs().mean(1, keepdim=True)
    c_e = 2.0 ** -18 * (gh * hat).abs().mean(1, keepdim=True) + (gh.abs() * hat_e).mean(1, keepdim=True)
    dx = rstd * (gh - a - hat * c)
    dx_e = (rstd * (a_e + hat.abs() * c_e + hat_e * c.abs() + 2.0 ** -21 * (gh.abs() + a.abs() + (hat * c).abs()))
            + dx.abs() * rstd_e)
    if gs is not None:
        dx = dx + gs.double()
        dx_e = dx_e + 2.0 ** -23 * (dx.abs() + gs.double().abs())
    out["dx"] = (dx, dx_e + u * dx.abs() + floor)
    n = (64 + R / 64) * 2.0 ** -24
    pfloor = 2.0 ** -25 if scale.dtype == torch.float16 else 2.0 ** -126
    ds, db = (g * hat).sum(0), g.sum(0)
    out["d_scale"] = (ds, n * (g * hat).abs().sum(0) + (g.abs() * hat_e).sum(0) + up * ds.abs() + pfloor)
    out["d_bias"] = (db, n * g.abs().sum(0) + up * db.abs() + pfloor)
    return s, out


def _near(name, got, want):
    ref, tol = want
    assert got.shape == ref.shape, name
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    if bad.any():
        at = torch.where(bad, off / tol.clamp_min(1e-300), 0).argmax()
        pytest.fail(f"{name}: {int(bad.sum())} of {bad.numel()} off; worst: {got.reshape(-1)[at].item():.6g} for "
                    f"{ref.reshape(-1)[at].item():.6g}, tolerance {tol.reshape(-1)[at].item():.3g}")


def _run(x, scale, bias, r, gy, gs, eps=EPS):
    from model_amd.layer_norm import layer_norm_backward, layer_norm_forward

    y, s, mean, rstd = layer_norm_forward(x, scale, bias, eps, residual=r)
    dx, ds, db = layer_norm_backward(gy, s, scale, mean, rstd, g_residual=gs)
    return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "d_scale": ds, "d_bias": db}, s


SHAPES = [(1, 1), (1, 3), (5, 4), (3, 7), (2, 8), (9, 9), (7, 16), (64, 256), (33, 100), (130, 192), (257, 250), (100, 1000),
          (65, 1283), (40, 1024), (20, 2048), (33, 3001), (9, 4096), (5, 5000), (6, 8192), (3, 10001), (2, 16384), (1, 16383),
          (9000, 64), (4097, 256), (2001, 1024), (700, 4096), (20011, 12)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,d", SHAPES)
def test_forward_and_backward(gpu_lib, R, d, dtype):
    for param, add in ((torch.float32, False), (dtype, True)):
        print(f"layer norm R={R} d={d} {dtype} parameters {param} add {add}", flush=True)
        args = _inputs(R, d, dtype, param, add)
        s, want = _formula(*args)
        got, s2 = _run(*args)
        assert torch.equal(s, s2)
        for name, w in want.items():
            _near(f"{name} ({param}, add {add})", got[name], w)
        assert got["y"].dtype == got["dx"].dtype == dtype and got["d_scale"].dtype == got["d_bias"].dtype == param


@pytest.mark.parametrize("dtype", DTYPES)
def test_autograd_equals_direct(gpu_lib, dtype):
    from model_amd.layer_norm import layer_norm

    x, w, b, r, gy, gs = _inputs(60, 320, dtype, add=True)
    want, s = _run(x, w, b, r, gy, gs)
    leaves = [t.clone().requires_grad_(True) for t in (x.reshape(5, 12, 320), w, b, r.reshape(5, 12, 320))]
    y, total = layer_norm(leaves[0], leaves[1], leaves[2], EPS, residual=leaves[3])
    assert y.shape == total.shape == (5, 12, 320) and torch.equal(y.reshape(60, 320), want["y"])
    assert torch.equal(total.reshape(60, 320), s)
    got = torch.autograd.grad([y, total], leaves, [gy.reshape(5, 12, 320), gs.reshape(5, 12, 320)], retain_graph=True)
    assert torch.equal(got[0].reshape(60, 320), want["dx"]) and torch.equal(got[3], got[0])
    assert torch.equal(got[1], want["d_scale"]) and torch.equal(got[2], want["d_bias"])
    # y alone, the sum alone, and without the residual
    alone = torch.autograd.grad(y, leaves[:1], gy.reshape(5, 12, 320), retain_graph=True)[0]
    assert torch.equal(alone.reshape(60, 320), _run(x, w, b, r, gy, None)[0]["dx"])
    only = torch.autograd.grad(total, [leaves[0], leaves[3]], gs.reshape(5, 12, 320))
    assert torch.equal(only[0].reshape(60, 320), gs) and torch.equal(only[1].reshape(60, 320), gs)
    plain = layer_norm(leaves[0], leaves[1], leaves[2], EPS)
    got = torch.autograd.grad(plain, leaves[:3], gy.reshape(5, 12, 320))
    want, _ = _run(x, w, b, None, gy, None)
    assert torch.equal(got[0].reshape(60, 320), want["dx"]) and torch.equal(got[1], want["d_scale"])
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, EPS), want["y"])
        y2, s2 = layer_norm(x, w, b, EPS, residual=r)
        assert torch.equal(y2, y.reshape(60, 320)) and torch.equal(s2, s)
        assert torch.equal(layer_norm(s, w, b, EPS), y2)  # the bits of the add, then the norm


def test_gradients_against_differences(gpu_lib):
    """Along unit directions: a step t leaves at most t^2 of the third
    derivative, below 32 |gy| max|scale| rstd^3 here (every derivative of a
    normalised row gains one rstd, and the polynomial in x_hat has few terms
    of size 1 to sqrt(d)), and y's error / t."""
    from model_amd.layer_norm import layer_norm

    x, w, b, _, gy, _ = _inputs(6, 24, torch.float32, offset=0.2)
    got, _ = _run(x, w, b, None, gy, None)
    g = torch.Generator(device="cuda").manual_seed(5)
    rstd3 = got["rstd"].max().item() ** 3
    for at, name in ((0, "dx"), (1, "d_scale"), (2, "d_bias")):
        base = (x, w, b)[at]
        way = torch.randn(base.shape, generator=g, device="cuda")
        way = way / way.norm()
        t = 2.0 ** -6
        f = []
        for k in (1, -1):
            args = [x, w, b]
            args[at] = base + k * t * way
            f.append((layer_norm(*args, EPS).double() * gy.double()).sum().item())
        want = (got[name].double() * way.double()).sum().item()
        size = gy.norm().item() * w.abs().max().item()
        assert abs((f[0] - f[1]) / (2 * t) - want) <= 32 * size * max(rstd3, 1) * t * t + size * 12 * 2.0 ** -20 / t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [256, 1023, 4100])
def test_large_mean(gpu_lib, dtype, d):
    """Rows far from zero: the variance is of the centred values."""
    args = _inputs(37, d, dtype, offset=30.0)
    _, want = _formula(*args)
    got, _ = _run(*args)
    for name, w in want.items():
        _near(name, got[name], w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_and_outlying_rows(gpu_lib, dtype):
    """A row of one value has x_hat = 0 (y = bias); one enormous element; zeros."""
    x, w, b, _, gy, _ = _inputs(4, 300, dtype)
    x[0] = 1.5
    x[1] = 0
    x[2, 7] = 3e4
    _, want = _formula(x, w, b, None, gy, None)
    got, _ = _run(x, w, b, None, gy, None)
    for name, v in want.items():
        _near(name, got[name], v)
    assert torch.equal(got["y"][1], b.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_finite(gpu_lib, dtype):
    """A row that is not finite is NaN alone."""
    from model_amd.layer_norm import layer_norm

    for d in (60, 1000, 4096):
        x, w, b, _, _, _ = _inputs(9, d, dtype)
        good = layer_norm(x, w, b, EPS)
        for v in (math.nan, math.inf, -math.inf):
            x2 = x.clone()
            x2[4, d - 1] = v
            y = layer_norm(x2, w, b, EPS)
            assert torch.isnan(y[4]).all() and torch.equal(y[:4], good[:4]) and torch.equal(y[5:], good[5:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [40, 257, 2050])
def test_strides(gpu_lib, dtype, d):
    x, w, b, r, gy, gs = _inputs(21, d, dtype, add=True)
    want, s = _run(x, w, b, r, gy, gs)

    def same(*args):
        got, s2 = _run(*args)
        assert torch.equal(s2, s)
        for name in want:
            assert torch.equal(got[name], want[name]), name

    def wide(t, at):
        out = torch.full((21, d + 11), math.nan, dtype=dtype, device="cuda")
        out[:, at:at + d] = t
        return out[:, at:at + d]

    same(wide(x, 0), w, b, wide(r, 3), wide(gy, 1), wide(gs, 8))
    same(x.t().contiguous().t(), w, b, r.t().contiguous().t(), gy.t().contiguous().t(), gs)
    every = torch.stack([w, b], 1)
    same(x, every[:, 0], every[:, 1], r, gy, gs)
    one = x[:1].expand(21, d)
    a, c = _run(one, w, b, r, gy, gs)[0], _run(one.contiguous(), w, b, r, gy, gs)[0]
    assert all(torch.equal(a[k], c[k]) for k in a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_stand_alone(gpu_lib, dtype):
    """A row's y and dx have the same bits in any batch."""
    for d in (24, 256, 1283, 4096):
        x, w, b, r, gy, gs = _inputs(513, d, dtype, add=True)
        got, _ = _run(x, w, b, r, gy, gs)
        for rows in ((0, 1), (100, 103), (510, 513)):
            part, _ = _run(*(t[rows[0]:rows[1]] if t.dim() == 2 else t for t in (x, w, b, r, gy, gs)))
            for name in ("y", "mean", "rstd", "dx"):
                assert torch.equal(part[name], got[name][rows[0]:rows[1]]), (d, name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeats_and_leaves_no_trace(gpu_lib, dtype):
    """Same bits in every call, whatever the workspace held."""
    args = _inputs(3001, 200, dtype, add=True)
    first, _ = _run(*args)
    for _ in range(3):
        junk = torch.full((16 << 20,), math.nan, device="cuda")
        del junk
        again, _ = _run(*args)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_no_rows(gpu_lib):
    from model_amd.layer_norm import layer_norm

    x = torch.zeros((3, 0, 8), device="cuda", requires_grad=True)
    w, b = (torch.ones(8, device="cuda", requires_grad=True) for _ in range(2))
    y = layer_norm(x, w, b)
    assert y.shape == (3, 0, 8)
    y.sum().backward()
    assert x.grad.shape == (3, 0, 8) and (w.grad == 0).all() and (b.grad == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [256, 1000])
def test_captured(gpu_lib, dtype, d):
    args = _inputs(300, d, dtype, add=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, s = _run(*args)
    for seed in range(4):
        new = _inputs(300, d, dtype, add=True, seed=seed + 30)
        for a, n in zip(args, new):
            a.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want, s2 = _run(*new)
        assert torch.equal(s, s2) and all(torch.equal(out[k], want[k]) for k in want)


def test_autograd_refused_under_capture(gpu_lib):
    from model_amd import layer_norm as ln

    x, w, b, _, _, _ = _inputs(4, 32, torch.float32)
    x.requires_grad_(True)
    from model_amd import _lib

    saved = ln._capturing
    try:
        y = ln.layer_norm(x, w, b)
        ln._capturing = lambda: True
        with pytest.raises(RuntimeError, match="layer_norm_forward"):
            ln.layer_norm(x, w, b)
        _lib.ops().pretend_capturing(True)
        with pytest.raises(RuntimeError, match="layer_norm_forward"):
            y.sum().backward()
    finally:
        ln._capturing = saved
        _lib.ops().pretend_capturing(False)


def test_second_derivative_is_refused(gpu_lib):
    """Under create_graph the gradients are there, and raise when they are
    differentiated again."""
    from model_amd.layer_norm import layer_norm

    x, w, b, _, gy, _ = _inputs(4, 32, torch.float32)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(layer_norm(x, w, b), [x, w, b], gy, create_graph=True)
    plain = torch.autograd.grad(layer_norm(x, w, b), [x, w, b], gy)
    assert all(torch.equal(p.detach(), q) for p, q in zip(grads, plain))
    with pytest.raises(RuntimeError, match="differentiable once"):
        grads[0].sum().backward()


def test_changed_in_place_is_refused(gpu_lib):
    from model_amd.layer_norm import layer_norm

    x, w, b, r, _, _ = _inputs(4, 32, torch.float32, add=True)
    x.requires_grad_(True)
    y, s = layer_norm(x, w, b, residual=r)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 40), (torch.bfloat16, 1000), (torch.float16, 3001)])
def test_offsets_past_32_bits(gpu_lib, dtype, d):
    """Rows 16 MiB apart, in buffers of more than 2^32 bytes."""
    print(f"layer norm, far rows d={d} {dtype}", flush=True)
    R, pitch = 300, 1 << (22 if dtype == torch.float32 else 23)
    x, w, b, r, gy, gs = _inputs(R, d, dtype, add=True)
    want, s = _run(x, w, b, r, gy, gs)

    def far(t):
        out = torch.empty(R * pitch, dtype=dtype, device="cuda").reshape(R, pitch)[:, :d]
        return out.copy_(t)

    got, s2 = _run(far(x), w, b, far(r), far(gy), far(gs))
    assert torch.equal(s2, s)
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_more_than_2_31_elements(gpu_lib):
    """Rows stand alone, so the last of many are those of a small call."""
    from model_amd.layer_norm import layer_norm_backward, layer_norm_forward

    R, d, n = (1 << 17) + 5, 16384, 7
    print(f"layer norm, R={R} d={d}", flush=True)
    x, w, b, _, gy, _ = _inputs(n, d, torch.bfloat16)
    many = torch.zeros((R, d), dtype=torch.bfloat16, device="cuda")
    grad = torch.zeros_like(many)
    many[-n:], grad[-n:] = x, gy
    y, s, mean, rstd = layer_norm_forward(many, w, b)
    dx, ds, db = layer_norm_backward(grad, s, w, mean, rstd)
    y1, s1, mean1, rstd1 = layer_norm_forward(x, w, b)
    dx1, ds1, db1 = layer_norm_backward(gy, s1, w, mean1, rstd1)
    for a, c in ((y, y1), (mean, mean1), (rstd, rstd1), (dx, dx1)):
        assert torch.equal(a[-n:], c)
    # the other rows pass no gradient to the parameters: sums of n terms in another order
    hat = (x.double() - mean1.double()[:, None]) * rstd1.double()[:, None]
    for got, ref, size in ((ds, gy.double() * hat, 1), (ds1, gy.double() * hat, 1), (db, gy.double(), 0), (db1, gy.double(), 0)):
        assert ((got.double() - ref.sum(0)).abs() <= (n + 4) * 2.0 ** -24 * ref.abs().sum(0) + size * 2.0 ** -126).all()


def test_one_tensor_as_rows_and_residual(gpu_lib):
    """x as its own residual: the sum's gradient reaches it twice."""
    from model_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward

    x, w, b, _, gy, gs = _inputs(50, 200, torch.float32, add=True)
    leaf = x.clone().requires_grad_()
    y, s = layer_norm(leaf, w, b, residual=leaf)
    torch.autograd.backward([y, s], [gy, gs])
    _, total, mean, rstd = layer_norm_forward(x, w, b, residual=x)
    dx, _, _ = layer_norm_backward(gy, total, w, mean, rstd, g_residual=gs)
    assert torch.equal(leaf.grad, dx + dx)


def test_residual_gradients_are_apart(gpu_lib):
    """x and the residual get gradients that one may change without the other."""
    from model_amd.layer_norm import layer_norm

    for only_sum in (False, True):
        x, w, b, r, gy, gs = _inputs(20, 64, torch.float32, add=True)
        x.requires_grad_(), r.requires_grad_()
        y, s = layer_norm(x, w, b, residual=r)
        if only_sum:
            s.backward(gs)
        else:
            torch.autograd.backward([y, s], [gy, gs])
        want = r.grad.clone()
        assert torch.equal(x.grad, want)
        x.grad.zero_()
        assert torch.equal(r.grad, want)


def test_memory_is_freed(gpu_lib):
    from model_amd.layer_norm import layer_norm

    x, w, b, r, _, _ = _inputs(300, 512, torch.float32, add=True)
    for t in (x, w, b, r):
        t.requires_grad_()

    def step(backward):
        y, s = layer_norm(x, w, b, residual=r)
        if backward:
            (y + s).sum().backward()
            x.grad = w.grad = b.grad = r.grad = None

    used = []
    for i in range(6):
        step(i % 2)
        torch.cuda.synchronize()
        used.append(torch.cuda.memory_allocated())
    assert used[4] == used[2] and used[5] == used[3]
