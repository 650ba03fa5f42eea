"""packed_attention against its definition in 64 bits, element by element.

Tolerances count roundings.  With u = eps / 2 of the inputs' type where it has 16
bits (0 for fp32, whose products keep it), e = 2^-24 and, for a row, zerr the error
of its scores (products of hd terms, their scaling, the maximum or lse taken off,
the exponential):

  out   (u + 2 zerr + n e) sum p |v| + w |out|          w = eps / 2 of out's type
  dv    (u + 2 zerr + n e) sum p |g| + w |dv|
  dz    p ((u + 2 zerr) |dp - delta| + hd e sum |g| |v| + sum |g| tol(out))
  dq    scale (sum |dz error| |k| + n e sum |dz| |k|) + w |dq|,  dk likewise

fp16's weights and their gradients below 2^-14 are held to 2^-25 absolute."""

import math
import random

import pytest
import torch

from model_amd.attention import packed_attention, packed_attention_backward, packed_attention_forward

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24
F64 = torch.float64


def definition(q, k, v, lq, lk, begin, scale, g_out=None, g_lse=None):
    """{name: (value, tolerance)} of every output, in 64 bits."""
    T, H, hd = q.shape
    G = k.shape[1]
    R = H // G
    t = q.dtype
    w = torch.finfo(t).eps / 2
    u = w if t != torch.float32 else 0.0
    small = 2.0 ** -25 if t == torch.float16 else 0.0
    z64 = lambda x: torch.zeros(x.shape, dtype=F64, device=DEV)  # noqa: E731
    res = {nm: (z64(x), z64(x)) for nm, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    res["lse"] = (torch.full((T, H), -math.inf, dtype=F64, device=DEV), torch.zeros((T, H), dtype=F64, device=DEV))
    a = 0
    for i, (nq, nk) in enumerate(zip(lq, lk)):
        b = begin[i]
        for h in range(H if nq else 0):
            Q, K, V = q[a:a + nq, h].to(F64), k[b:b + nk, h // R].to(F64), v[b:b + nk, h // R].to(F64)
            seen = torch.arange(nk, device=DEV)[None] <= torch.arange(nq, device=DEV)[:, None] + (nk - nq)
            some = seen.any(1)
            z = scale * (Q @ K.t())
            zerr = torch.where(seen, (hd + 4) * E * scale * (Q.abs() @ K.abs().t()) + 8 * E * z.abs(), 0).amax(1) if nk else some * 0.0
            z = z.masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(z, 1) if nk else torch.full((nq,), -math.inf, dtype=F64, device=DEV)
            zerr = zerr + 8 * E + 4 * E * torch.where(some, lse.abs(), 0.0)
            p = torch.where(seen & some[:, None], torch.exp(z - torch.where(some, lse, 0.0)[:, None]), 0.0)
            rel = (u + 2 * zerr + nk * E)[:, None]
            out = p @ V
            tol_out = rel * (p @ V.abs()) + w * out.abs() + small * seen.to(F64) @ V.abs() + small
            res["out"][0][a:a + nq, h], res["out"][1][a:a + nq, h] = out, tol_out
            res["lse"][0][a:a + nq, h], res["lse"][1][a:a + nq, h] = lse, zerr + nk * E
            if g_out is not None:
                g = g_out[a:a + nq, h].to(F64)
                dv = p.t() @ g
                nr = nq * R
                res["dv"][0][b:b + nk, h // R] += dv
                res["dv"][1][b:b + nk, h // R] += (p * (rel + nr * E)).t() @ g.abs() + small * seen.to(F64).t() @ g.abs()
                delta = (g * out).sum(1)
                if g_lse is not None:
                    delta = delta - g_lse[a:a + nq, h].to(F64)
                dp = g @ V.t()
                dz = p * (dp - delta[:, None])
                derr = p * ((u + 2 * zerr)[:, None] * (dp - delta[:, None]).abs() + (hd + 4) * E * (g.abs() @ V.abs().t())
                            + ((g.abs() * tol_out).sum(1) + 4 * E * delta.abs())[:, None])
                derr = derr + seen * small * max(float(g.abs().max()), 0.0) * 4
                res["dq"][0][a:a + nq, h] = scale * (dz @ K)
                res["dq"][1][a:a + nq, h] = scale * (derr @ K.abs() + nk * E * (dz.abs() @ K.abs())) + small
                res["dk"][0][b:b + nk, h // R] += scale * (dz.t() @ Q)
                res["dk"][1][b:b + nk, h // R] += scale * (derr.t() @ Q.abs() + nr * E * (dz.abs().t() @ Q.abs())) + small
        a += nq
    for nm in ("dq", "dk", "dv"):
        res[nm][1].add_(w * res[nm][0].abs())
    # the output's own rounding below fp16's normal numbers: their spacing is 2^-24, half a step 2^-25
    res["dv"][1].add_(small)
    return res


def check(got, want, name):
    value, tol = want
    assert got.shape == value.shape, name
    got = got.to(F64)
    gone = torch.isinf(value)
    assert torch.equal(got[gone], value[gone]), name
    err = torch.where(gone, 0.0, (got - torch.where(gone, 0.0, value)).abs())
    err = torch.where(gone, 0.0, err)
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} beyond, by a factor of {float((err / tol.clamp(min=1e-300))[bad].max()):.3g}"


def sums(x):
    return [0, *torch.tensor(x, dtype=torch.int64).cumsum(0).tolist()] if len(x) else [0]


def make(lq, lk, H, G, hd, dtype, seed=0, std=1.0, tail=0, key_tail=0, fused=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T, S = sum(lq) + tail, sum(lk) + key_tail
    mk = lambda n, h: (torch.randn((n, h, hd), generator=g, device=DEV) * std).to(dtype)  # noqa: E731
    if fused:
        x = torch.stack([mk(T, H), mk(T, H), mk(T, H)], 1)
        return x[:, 0], x[:, 1], x[:, 2], mk(T, H), torch.randn((T, H), generator=g, device=DEV)
    return mk(T, H), mk(S, G), mk(S, G), mk(T, H), torch.randn((T, H), generator=g, device=DEV)


def run_all(q, k, v, lq, lk, g_out, g_lse=None, scale=None, own_keys=False, wide=False, key_lengths=None, begin=None):
    it = torch.int64 if wide else torch.int32
    starts = torch.tensor(sums(lq), dtype=it, device=DEV)
    kw = {"scale": scale}
    if own_keys:
        kw["key_starts"] = torch.tensor(begin if begin is not None else sums(lk), dtype=it, device=DEV)
        if key_lengths is not None:
            kw["key_lengths"] = torch.tensor(key_lengths, dtype=it, device=DEV)
    out, lse = packed_attention_forward(q, k, v, starts, **kw)
    dq, dk, dv = packed_attention_backward(g_out, q, k, v, out, lse, starts, g_lse=g_lse, **kw)
    res = {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    want = definition(q, k, v, lq, lk, begin if begin is not None else sums(lk), scale or q.shape[2] ** -0.5, g_out, g_lse)
    for nm, x in res.items():
        check(x, want[nm], nm)
    return res, starts, kw


DT = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("H,G", [(4, 4), (6, 2), (5, 1), (8, 1)])
def test_whole_sequences(dtype, hd, H, G):
    lq = [1, 0, 31, 32, 33, 2, 64, 65, 0, 127, 129, 5]
    q, k, v, g, gl = make(lq, lq, H, G, hd, dtype, seed=hd + H)
    run_all(q, k, v, lq, lq, g, gl if H == 6 else None, wide=H == 5)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257, 300, 1025])
def test_one_sequence(dtype, n):
    q, k, v, g, gl = make([n], [n], 4, 2, 64, dtype, seed=n)
    run_all(q, k, v, [n], [n], g, gl)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_that_continue_a_cache(dtype, hd):
    lq = [3, 40, 1, 70, 7, 0, 130, 5]
    lk = [3, 100, 200, 71, 600, 9, 131, 0]  # the last: queries without a key
    q, k, v, g, gl = make(lq, lk, 6, 3, hd, dtype, seed=1)
    run_all(q, k, v, lq, lk, g, gl, own_keys=True)


@pytest.mark.parametrize("dtype", DT)
def test_more_queries_than_keys(dtype):
    lq, lk = [40, 100, 33], [10, 37, 32]  # the first queries of each see nothing
    q, k, v, g, gl = make(lq, lk, 4, 2, 64, dtype, seed=2)
    res, _, _ = run_all(q, k, v, lq, lk, g, gl, own_keys=True)
    assert (res["out"][:30] == 0).all() and torch.isinf(res["lse"][:30]).all() and (res["dq"][:30] == 0).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd", [(32, 8, 128), (4, 4, 64), (8, 1, 32), (12, 4, 64)])
def test_single_tokens_over_a_cache(dtype, H, G, hd):
    cap, n = 1500, 5
    used = [1, 1500, 0, 777, 33]
    q, k, v, g, gl = make([1] * n, [cap] * n, H, G, hd, dtype, seed=3)
    begin = [cap * i for i in range(n + 1)]
    for i, x in enumerate(used):  # places not in use hold anything
        k[begin[i] + x:begin[i + 1]] = math.nan
        v[begin[i] + x:begin[i + 1]] = math.inf
    run_all(q, k, v, [1] * n, used, g, gl, own_keys=True, key_lengths=used, begin=begin)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("keys", [513, 5000, 40000])
def test_one_token_many_keys(dtype, keys):
    q, k, v, g, gl = make([1], [keys], 4, 2, 64, dtype, seed=4)
    run_all(q, k, v, [1], [keys], g, gl, own_keys=True)


@pytest.mark.parametrize("dtype", DT)
def test_rows_of_no_sequence(dtype):
    lq = [0, 20, 50]
    q, k, v, g, gl = make(lq, lq, 4, 2, 32, dtype, seed=5, tail=45, key_tail=45)
    q, k, v = q.clone(), k.clone(), v.clone()
    q[70:], k[70:], v[70:], g[70:] = math.nan, math.inf, math.nan, math.nan
    res, _, _ = run_all(q, k, v, lq, lq, g)
    for nm in ("out", "dq", "dk", "dv"):
        assert (res[nm][70:] == 0).all(), nm
    # sequences that begin behind the first token
    starts = torch.tensor([20, 70], dtype=torch.int32, device=DEV)
    out, lse = packed_attention_forward(q, k, v, starts)
    assert (out[:20] == 0).all() and torch.isinf(lse[:20]).all()
    want = definition(q[20:70], k[20:70], v[20:70], [50], [50], [0], 32 ** -0.5)
    check(out[20:70], want["out"], "out")


@pytest.mark.parametrize("dtype", DT)
def test_not_finite_stays_in_its_sequence(dtype):
    lq = [40, 70, 10, 33]
    q, k, v, g, _ = make(lq, lq, 4, 2, 64, dtype, seed=6)
    starts = torch.tensor(sums(lq), dtype=torch.int32, device=DEV)

    def all_of():
        out, lse = packed_attention_forward(q, k, v, starts)
        return [out, lse, *packed_attention_backward(g, q, k, v, out, lse, starts)]

    want = all_of()
    q[45], k[60], v[80], g[109] = math.nan, math.inf, math.nan, -math.inf
    for a, b in zip(want, all_of()):
        assert torch.equal(a[:40], b[:40]) and torch.equal(a[110:], b[110:])


@pytest.mark.parametrize("dtype", DT)
def test_large_scores(dtype):
    """Scores of hundreds: maxima must be taken off, and grow from tile to tile."""
    n = 300
    q, k, v, g, _ = make([n], [n], 2, 1, 64, dtype, seed=7, std=2.0)
    ramp = torch.linspace(0.1, 4.0, n, device=DEV)[:, None, None]
    k, q = (k.float() * ramp).to(dtype), (q.float().abs() * 3).to(dtype)
    k = torch.cat([k[:150], k[150:].abs()])
    run_all(q, k, v, [n], [n], g)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("which", ["fused", "heads first", "gaps", "odd offset", "expanded"])
def test_strides(dtype, which):
    lq, H, G, hd = [70, 1, 50], 4, 4, 64
    n = sum(lq)
    q, k, v, g, gl = make(lq, lq, H, G, hd, dtype, seed=8, fused=which == "fused")
    if which == "heads first":
        q, k, v, g = (x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v, g))
    elif which == "gaps":
        q, k, v, g = (torch.nn.functional.pad(x, (0, hd, 0, 1))[:, :H, :hd] for x in (q, k, v, g))
    elif which == "odd offset":  # not at 16 bytes
        q, k, v, g = (torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(n, H, hd) for x in (q, k, v, g))
    elif which == "expanded":
        k, v, g = k[:, :1].expand(n, G, hd), v[:1].expand(n, G, hd), g[:1, :1].expand(n, H, hd)
    run_all(q, k, v, lq, lq, g, gl)
    gl2 = gl.t().contiguous().t()
    run_all(q, k, v, lq, lq, g, gl2)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [200, 70, 4200])
def test_many_short_sequences(dtype, n):
    rng = random.Random(n)
    lq = [rng.choice([0, 1, 2, 3, 9]) for _ in range(n)]
    q, k, v, g, _ = make(lq, lq, 2, 1, 32, dtype, seed=9)
    T = sum(lq)
    starts = torch.tensor(sums(lq), dtype=torch.int32, device=DEV)
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(lq, device=DEV))
    out, lse = packed_attention_forward(q, k, v, starts)
    dq, dk, dv = packed_attention_backward(g, q, k, v, out, lse, starts)
    if T < 1500:
        want = definition(q, k, v, lq, lq, sums(lq), 32 ** -0.5, g)
        for nm, x in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
            check(x, want[nm], nm)
    else:  # as one batch under a block mask
        Q, K, V, gg = q.to(F64), k.to(F64)[:, 0], v.to(F64)[:, 0], g.to(F64)
        idx = torch.arange(T, device=DEV)
        seen = (seq[:, None] == seq[None]) & (idx[:, None] >= idx[None])
        w = torch.finfo(dtype).eps
        for h in range(2):
            p = torch.softmax((Q[:, h] @ K.t() * 32 ** -0.5).masked_fill(~seen, -math.inf), 1)
            assert ((out[:, h] - p @ V).abs() <= 2 * w * (p @ V.abs()) + 2e-5).all()
        assert torch.isfinite(dq).all() and torch.isfinite(dk).all() and torch.isfinite(dv).all()


@pytest.mark.parametrize("dtype", DT)
def test_autograd(dtype):
    lq = [33, 80, 1]
    q, k, v, g, gl = make(lq, lq, 4, 2, 64, dtype, seed=10)
    res, starts, _ = run_all(q, k, v, lq, lq, g, gl)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out, lse = packed_attention(*leaves, starts, return_lse=True)
    grads = torch.autograd.grad([out, lse], leaves, [g, gl], retain_graph=True)
    for nm, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        assert torch.equal(x, res[nm]), nm
    only, = torch.autograd.grad(packed_attention(leaves[0], k, v, starts), leaves[0], g)
    out0, lse0 = packed_attention_forward(q, k, v, starts)
    assert torch.equal(only, packed_attention_backward(g, q, k, v, out0, lse0, starts)[0])
    # the logsumexp alone
    d_lse = torch.autograd.grad(lse, leaves, gl, retain_graph=True)
    want = packed_attention_backward(torch.zeros_like(g), q, k, v, out0, lse0, starts, g_lse=gl)
    assert all(torch.equal(a, b) for a, b in zip(d_lse, want))
    assert (want[2] == 0).all()
    with torch.no_grad():
        assert torch.equal(packed_attention(*leaves, starts), out0)
    dd = torch.autograd.grad(out, leaves, g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dd[0].float().sum().backward()


def test_gradient_against_differences():
    lq = [5, 40]
    q, k, v, g, gl = make(lq, lq, 4, 2, 32, torch.float32, seed=11)
    res, starts, _ = run_all(q, k, v, lq, lq, g, gl)

    def loss(q, k, v):  # the definition in 64 bits
        r = definition(q, k, v, lq, lq, sums(lq), 32 ** -0.5)
        return float((r["out"][0] * g.to(F64)).sum() + (r["lse"][0] * gl.to(F64)).sum())

    xs = [x.to(F64) for x in (q, k, v)]
    for i, nm in enumerate(("dq", "dk", "dv")):
        way = torch.randn(xs[i].shape, dtype=F64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))
        h = 1e-5
        up, down = ([x + s * h * way if j == i else x for j, x in enumerate(xs)] for s in (1, -1))
        # differences: error h^2 times a third derivative of order 1, and 2^-52 of the loss over h
        assert abs((loss(*up) - loss(*down)) / (2 * h) - float((res[nm].to(F64) * way).sum())) < 1e-3


@pytest.mark.parametrize("dtype", DT)
def test_empty(dtype):
    q, k, v, g, _ = make([0], [0], 4, 2, 32, dtype)
    starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert packed_attention(q, k, v, starts).shape == (0, 4, 32)
    k, v = (torch.ones((7, 2, 32), dtype=dtype, device=DEV) for _ in range(2))
    out, lse = packed_attention_forward(q, k, v, starts, key_starts=starts)
    dq, dk, dv = packed_attention_backward(g, q, k, v, out, lse, starts, key_starts=starts)
    assert dq.shape == q.shape and (dk == 0).all() and (dv == 0).all()
    q = torch.ones((9, 4, 32), dtype=dtype, device=DEV)
    k = v = torch.zeros((0, 2, 32), dtype=dtype, device=DEV)
    out, lse = packed_attention_forward(q, k, v, starts, key_starts=starts)
    assert (out == 0).all() and torch.isinf(lse).all()
    dq, dk, dv = packed_attention_backward(q, q, k, v, out, lse, starts, key_starts=starts)
    assert (dq == 0).all() and dk.shape == k.shape


@pytest.mark.parametrize("dtype", DT)
def test_starts_that_make_no_sense(dtype):
    """Unspecified rows, but no access outside and no endless search."""
    q, k, v, g, _ = make([100], [100], 4, 2, 64, dtype, seed=12)
    for bad in ([50, 20, 90, 10], [-5, 200, 300], [2 ** 31 - 1, -2 ** 31, 0], [0, 2 ** 31 - 1]):
        starts = torch.tensor(bad, dtype=torch.int32, device=DEV)
        lengths = torch.tensor([2 ** 31 - 1, -7, 50][:len(bad) - 1], dtype=torch.int32, device=DEV)
        for kw in ({}, {"key_starts": starts.flip(0), "key_lengths": lengths}):
            out, lse = packed_attention_forward(q, k, v, starts, **kw)
            packed_attention_backward(g, q, k, v, out, lse, starts, **kw)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DT)
def test_runs_alike_on_a_stream_and_in_a_graph(dtype):
    lq, lk = [40, 1, 130, 3], [500, 900, 130, 40]
    q, k, v, g, gl = make(lq, lk, 4, 2, 64, dtype, seed=13)
    res, starts, kw = run_all(q, k, v, lq, lk, g, gl, own_keys=True)

    def call():
        out, lse = packed_attention_forward(q, k, v, starts, **kw)
        return (out, lse, *packed_attention_backward(g, q, k, v, out, lse, starts, g_lse=gl, **kw))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    for a, b in zip(got, res.values()):
        assert torch.equal(a, b)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]  # an eager graph of the same leaves lives
    eager = packed_attention(*leaves, starts, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
        with pytest.raises(RuntimeError, match="HIP graph capture"):
            packed_attention(*leaves, starts, **kw)
    for i in range(3):
        if i:
            q.mul_(0.5)
            eager_now = call()
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, eager_now if i else res.values()):
            assert torch.equal(a, b)
    del eager


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_past_32_bits(dtype):
    """Keys whose rows lie more than 2^31 elements apart."""
    free, _ = torch.cuda.mem_get_info()
    cap, G, hd = 1 << 20, 33, 64
    if free < 40 << 30:
        pytest.fail("needs 40 GiB")
    kv = torch.empty((cap, G, hd), dtype=dtype, device=DEV)
    kv[:50].normal_()
    kv[cap - 50:].normal_()
    q = torch.randn((2, G, hd), device=DEV).to(dtype)
    starts = torch.tensor([0, 1, 2], dtype=torch.int64, device=DEV)
    begin = torch.tensor([0, cap - 50, cap], dtype=torch.int64, device=DEV)
    out = packed_attention(q, kv, kv, starts, key_starts=begin, key_lengths=torch.tensor([50, 50], device=DEV))
    small = torch.cat([kv[:50], kv[cap - 50:]])
    want = packed_attention(q, small, small, starts, key_starts=torch.tensor([0, 50, 100], device=DEV))
    assert torch.allclose(out.float(), want.float(), rtol=2 * torch.finfo(dtype).eps, atol=2 * torch.finfo(dtype).eps)


@pytest.mark.parametrize("g_size,v_size", [(2.0 ** -14, 1.0), (1.0, 500.0), (2.0 ** 9, 100.0), (0.0, 1.0)])
def test_fp16_gradients_of_any_size(g_size, v_size):
    """dz is held under a power of two of the call's own: small gradients keep their bits, large ones do not overflow."""
    lq = [300, 41]
    q, k, v, g, _ = make(lq, lq, 4, 2, 64, torch.float16, seed=14)
    q, k = q * 0.2, k * 0.2  # many alike weights, of 1 / 300 each
    run_all(q, k, (v.float() * v_size).half(), lq, lq, (g.float() * g_size).half(), scale=0.01)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("H,G", [(16, 16), (6, 2), (8, 2), (33, 1)])
def test_many_rows(dtype, hd, H, G):
    """Enough rows and keys for the tiles of large calls: 128 rows, 64 or 128 keys."""
    rng = random.Random(H + hd)
    total = {16: 8_300, 6: 66_000, 8: 66_000, 33: 9_000}[H] // (4 if hd == 128 else 1)
    lq = [0, 1, 127, 128, 129, 257]
    while sum(lq) < total:
        lq.append(rng.choice([1, 2, 63, 65, 200, 300, 511, 640, 900]))
    q, k, v, g, gl = make(lq, lq, H, G, hd, dtype, seed=15, fused=H == G)
    run_all(q, k, v, lq, lq, g, gl, wide=H == 6)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 128])
def test_many_rows_that_continue_a_cache(dtype, hd):
    rng = random.Random(hd)
    lq = [rng.choice([1, 40, 130, 260]) for _ in range(90)] + [0, 50]
    cap = 700
    used = [max(0, min(cap, x + rng.choice([0, 1, 100, 333, -20]))) for x in lq]
    q, k, v, g, gl = make(lq, [cap] * len(lq), 8, 4, hd, dtype, seed=16)
    begin = [cap * i for i in range(len(lq) + 1)]
    for i, x in enumerate(used):  # places not in use hold anything
        k[begin[i] + x:begin[i + 1]] = math.nan
        v[begin[i] + x:begin[i + 1]] = math.inf
    run_all(q, k, v, lq, used, g, gl, own_keys=True, key_lengths=used, begin=begin)


@pytest.mark.parametrize("dtype", DT)
def test_many_rows_not_finite_stays_in_its_sequence(dtype):
    lq = [1500, 700, 2000]
    q, k, v, g, _ = make(lq, lq, 16, 16, 64, dtype, seed=17)
    starts = torch.tensor(sums(lq), dtype=torch.int32, device=DEV)

    def all_of():
        out, lse = packed_attention_forward(q, k, v, starts)
        return [out, lse, *packed_attention_backward(g, q, k, v, out, lse, starts)]

    want = all_of()
    q[1505], k[1700], v[2100], g[2199] = math.nan, math.inf, math.nan, -math.inf
    for a, b in zip(want, all_of()):
        assert torch.equal(a[:1500], b[:1500]) and torch.equal(a[2200:], b[2200:])


@pytest.mark.parametrize("dtype", DT)
def test_many_rows_with_starts_that_make_no_sense(dtype):
    """As test_starts_that_make_no_sense, at sizes that take the large calls' tiles."""
    T = 9000
    q, k, v, g, _ = make([T], [T], 16, 16, 64, dtype, seed=18)
    rng = random.Random(5)
    for n in (3, 100):
        starts = torch.tensor([rng.randint(-T, 2 * T) for _ in range(n)], dtype=torch.int64, device=DEV)
        for kw in ({}, {"key_starts": starts.flip(0), "key_lengths": starts[1:] * 3}):
            out, lse = packed_attention_forward(q, k, v, starts, **kw)
            packed_attention_backward(g, q, k, v, out, lse, starts, **kw)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DT)
def test_heads_that_lie_far_apart(dtype):
    """A cache with its heads outermost is read where it lies; q's heads as far apart are copied."""
    used, cap, G, hd = [70, 3], 1 << 18, 3, 64
    cache = torch.zeros((2, G, cap, hd), dtype=dtype, device=DEV)  # heads 2^24 elements apart
    g = torch.Generator(device=DEV).manual_seed(19)
    cache[:, :, :200] = torch.randn((2, G, 200, hd), generator=g, device=DEV).to(dtype)
    k, v = (c.permute(1, 0, 2)[:200] for c in cache)
    q = torch.zeros((6, 1 << 19, hd), dtype=dtype, device=DEV)[:, :2].permute(1, 0, 2)
    q.copy_(torch.randn((2, 6, hd), generator=g, device=DEV))
    begin = [0, 100, 200]
    run_all(q, k, v, [1, 1], used, torch.ones_like(q), own_keys=True, key_lengths=used, begin=begin)


def test_two_graphs_at_once():
    sets, graphs = [], []
    for i in range(2):
        lq = [40 + i, 1, 300]
        q, k, v, g, gl = make(lq, lq, 4, 2, 64, torch.float16, seed=20 + i)
        starts = torch.tensor(sums(lq), dtype=torch.int32, device=DEV)

        def call(q=q, k=k, v=v, g=g, gl=gl, starts=starts):
            out, lse = packed_attention_forward(q, k, v, starts)
            return (out, lse, *packed_attention_backward(g, q, k, v, out, lse, starts, g_lse=gl))

        want = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        sets.append((want, got))
        graphs.append((graph, call))  # the graph reads the inputs where they were: the call keeps them
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for want, got in sets:
            for a, b in zip(want, got):
                assert torch.equal(a, b)
                b.zero_()
