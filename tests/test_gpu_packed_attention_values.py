"""packed_attention: what values elsewhere do to a sequence's results.  Nothing, in whatever size they come: the same
sequences of one call are compared bit by bit, and values of unlike sizes with the definition in 64 bits."""

import pytest
import torch

from model_amd.attention import packed_attention_backward, packed_attention_forward
from tests.test_gpu_packed_attention import DEV, DT, check, definition, make, run_all, sums

pytestmark = pytest.mark.gpu


def all_of(q, k, v, g, gl, starts, **kw):
    out, lse = packed_attention_forward(q, k, v, starts, **kw)
    return out, lse, *packed_attention_backward(g, q, k, v, out, lse, starts, g_lse=gl, **kw)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("what", ["v", "g_out", "g_lse", "all"])
@pytest.mark.parametrize("lq,H,G,hd", [([40, 300, 33, 70], 4, 2, 64), ([40, 300, 33, 70], 5, 1, 128),
                                       ([1500, 700, 2000], 16, 16, 64), ([900, 5, 1700], 32, 16, 128),
                                       ([2500, 6000, 500], 16, 16, 32)])
def test_another_sequence_of_large_values(dtype, what, lq, H, G, hd):
    """Sequence 1's values times 2^12 (finite in every type): the others' bits stay."""
    q, k, v, g, gl = make(lq, lq, H, G, hd, dtype, seed=31, std=0.5)
    starts = torch.tensor(sums(lq), dtype=torch.int32, device=DEV)
    want = all_of(q, k, v, g, gl, starts)
    one = slice(lq[0], lq[0] + lq[1])
    for nm, x in (("v", v), ("g_out", g), ("g_lse", gl)):
        if what in (nm, "all"):
            x[one] *= 4096
    got = all_of(q, k, v, g, gl, starts)
    for nm, a, b in zip(("out", "lse", "dq", "dk", "dv"), want, got):
        assert torch.equal(a[:one.start], b[:one.start]) and torch.equal(a[one.stop:], b[one.stop:]), nm
        assert torch.isfinite(b[one].float()).all() or dtype == torch.float16, nm


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd,n", [(4, 2, 64, 1), (8, 1, 128, 3), (6, 3, 32, 40)])
def test_places_not_in_use_of_large_values(dtype, H, G, hd, n):
    """A cache's free places hold finite values of 60,000: every bit as if they held 0."""
    cap, used = 700, [1, 700, 0, 333, 64]
    q, k, v, g, gl = make([n] * 5, [cap] * 5, H, G, hd, dtype, seed=32)
    starts = torch.arange(0, 5 * n + 1, n, dtype=torch.int32, device=DEV)
    kw = {"key_starts": torch.arange(0, 5 * cap + 1, cap, dtype=torch.int32, device=DEV),
          "key_lengths": torch.tensor(used, dtype=torch.int32, device=DEV)}
    runs = []
    for fill in (0.0, 60_000.0):
        for i, x in enumerate(used):
            k[cap * i + x:cap * (i + 1)] = fill
            v[cap * i + x:cap * (i + 1)] = fill
        runs.append(all_of(q, k, v, g, gl, starts, **kw))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,hd", [(4, 64), (6, 128), (8, 32)])
def test_sequences_of_unlike_sizes(dtype, H, hd):
    """Each sequence's gradients and values have a size of their own, as small and as large as fp16 takes."""
    lq = [60, 300, 33, 129]
    q, k, v, g, gl = make(lq, lq, H, H // 2, hd, dtype, seed=33)
    q, k = q * 0.2, k * 0.2
    a = 0
    for n, sv, sg in zip(lq, (500.0, 1.0, 2.0 ** -9, 30.0), (2.0 ** -14, 2.0 ** 9, 1.0, 2.0 ** -6)):
        v[a:a + n] *= sv
        g[a:a + n] *= sg
        gl[a:a + n] *= sv * sg
        a += n
    run_all(q, k, v, lq, lq, g, gl, scale=0.05)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [90, 1300])
def test_rows_and_keys_of_unlike_sizes(dtype, n):
    """Within one sequence sizes grow and fall by 2^20 from row to row, so that the largest is met late, early and again."""
    q, k, v, g, gl = make([n], [n], 4, 2, 64, dtype, seed=34)
    gen = torch.Generator(device=DEV).manual_seed(35)
    size = torch.exp2(torch.randint(-14, 6, (n, 1, 1), generator=gen, device=DEV).float())
    g = (g.float() * size).to(dtype)
    v = (v.float() * torch.exp2(torch.randint(-6, 6, (n, 1, 1), generator=gen, device=DEV).float())).to(dtype)
    run_all(q * 0.3, k * 0.3, v, [n], [n], g, gl * size[:, :, 0])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lq,lk,H,G,hd", [([40, 100, 33], [10, 37, 32], 4, 2, 64), ([40, 100, 33], [10, 37, 32], 8, 1, 128),
                                          ([900, 1500, 40], [700, 1400, 0], 16, 16, 64),
                                          ([4500, 1500], [4400, 1], 16, 16, 32)])
def test_queries_without_keys_and_a_senseless_gradient_of_lse(dtype, lq, lk, H, G, hd):
    """The lse of such a query is -inf, and what comes back for it NaN or inf as often as not: it passes no gradient."""
    q, k, v, g, gl = make(lq, lk, H, G, hd, dtype, seed=36)
    starts, begin = (torch.tensor(sums(x), dtype=torch.int32, device=DEV) for x in (lq, lk))
    lost = torch.cat([torch.arange(n, device=DEV) < n - m for n, m in zip(lq, lk)])
    gl[lost] = 0
    want = all_of(q, k, v, g, gl, starts, key_starts=begin)
    assert (want[2][lost] == 0).all() and torch.isinf(want[1][lost]).all()
    for bad in (float("nan"), float("inf"), float("-inf")):
        gl[lost] = bad
        for nm, a, b in zip(("out", "lse", "dq", "dk", "dv"), want, all_of(q, k, v, g, gl, starts, key_starts=begin)):
            assert torch.equal(a, b), (bad, nm)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd,n", [(4, 2, 64, 3), (8, 1, 128, 1), (16, 16, 32, 2100)])
def test_places_not_in_use_have_gradients_0(dtype, H, G, hd, n):
    """Even beside rows whose gradient is not finite."""
    cap, used = 2200, [3, 70, 2101]
    q, k, v, g, gl = make([n] * 3, [cap] * 3, H, G, hd, dtype, seed=37)
    g[0], g[2 * n - 1], gl[-1] = float("nan"), float("inf"), float("nan")
    starts = torch.arange(0, 3 * n + 1, n, dtype=torch.int32, device=DEV)
    got = all_of(q, k, v, g, gl, starts, key_starts=torch.arange(0, 3 * cap + 1, cap, dtype=torch.int32, device=DEV),
                 key_lengths=torch.tensor(used, dtype=torch.int32, device=DEV))
    for x in got[3:]:
        for i, m in enumerate(used):
            assert (x[cap * i + m:cap * (i + 1)] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_grids_of_eleven_million_tiles(dtype):
    """1.4 million empty sequences before one of 2,048 tokens: the grid of the gradients' large tiles would pass 32 bits."""
    n, T, H = 1_400_000, 2048, 8
    q, k, v, g, gl = make([T], [T], H, H, 128, dtype, seed=38)
    starts = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    starts[-1] = T
    want = definition(q, k, v, [T], [T], [0], 128 ** -0.5, g, gl)
    for nm, x in zip(("out", "lse", "dq", "dk", "dv"), all_of(q, k, v, g, gl, starts)):
        check(x, want[nm], nm)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("n", [60, 300, 1100, 2500])
def test_errors_of_16_bits(dtype, hd, n):
    """Weights on few keys (scores of standard deviation 1.7).  Of an output's two roundings, the weights' or dz's and its
    own, each has the error of the exact value rounded once: sqrt(2) of it together.  Up to 1.5 the rest, the most of it
    delta from the rounded out, has half a rounding: sqrt(1.5^2 - 2)."""
    lq = [n, n // 2]
    q, k, v, g, _ = make(lq, lq, 8, 4, hd, dtype, seed=39)
    q, k = q * 1.3, k * 1.3
    starts = torch.tensor(sums(lq), dtype=torch.int32, device=DEV)
    want = definition(q, k, v, lq, lq, sums(lq), hd ** -0.5, g)
    for nm, x in zip(("out", "lse", "dq", "dk", "dv"), all_of(q, k, v, g, None, starts)):
        exact = want[nm][0]
        once = (exact.to(x.dtype).double() - exact).norm()
        if nm != "lse":
            assert (x.double() - exact).norm() <= 1.5 * once, nm
