"""clip_global_norm against its formula in 64 bits.

The norm is a sum in fp64, rounded to fp32 (2^-24); the scale has that, the fp32 sum
norm + 1e-6 and the division (2^-24 each): 2^-22 of slack holds both.  A scaled
gradient is off by the scale's error, one fp32 product and half a step of its type."""

import math

import pytest
import torch

from model_amd.grad_clip import clip_global_norm, global_norm_scale

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = [torch.float32, torch.float16, torch.bfloat16]


def formula(grads, clip, row_sq=None):
    sq = sum((float(g.double().square().sum()) for g in grads), 0.0)
    if row_sq is not None:
        sq += float(row_sq.double().sum())
    norm = math.sqrt(sq)
    return min(1.0, clip / (norm + 1e-6)), norm


def check(grads, clip, row_sq=None):
    before = [g.detach().clone() for g in grads]
    scale, norm = formula(before, clip, row_sq)
    alone = global_norm_scale(grads, clip, row_sq=row_sq)
    for a, b in zip(grads, before):
        assert torch.equal(a, b)
    versions = [g._version for g in grads]
    got = clip_global_norm(grads, clip, row_sq=row_sq)
    assert torch.equal(got, alone) and got.shape == (2,) and got.dtype == torch.float32
    assert abs(float(got[0]) - scale) <= 2 ** -22 * scale and abs(float(got[1]) - norm) <= 2 ** -23 * norm
    for g, b, ver in zip(grads, before, versions):
        assert g._version > ver
        want = b.double() * scale
        tol = want.abs() * (2 ** -22 + 2 ** -24 + torch.finfo(g.dtype).eps / 2)
        if g.dtype == torch.float16:
            tol = tol + 2.0 ** -25  # below its normal numbers
        assert ((g.double() - want).abs() <= tol).all()
        if scale == 1.0:
            assert torch.equal(g, b)
    return got


def rand(shape, dtype, seed=0, std=1.0):
    return (torch.randn(shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)) * std).to(dtype)


@pytest.mark.parametrize("clip", [0.0, 0.3, 1e9])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [1, 2, 7, 4095, 4096, 4097, 100_003, 5_000_000])
def test_one_tensor(dtype, n, clip):
    check([rand(n, dtype, seed=n)], clip)


@pytest.mark.parametrize("count", [2, 191, 192, 193, 400])
def test_many_tensors_of_mixed_types(count):
    grads = [rand((1 + 37 * i % 97, 1 + i % 61), DT[i % 3], seed=i, std=0.1 + i % 5) for i in range(count)]
    grads.insert(1, torch.zeros((0, 5), device=DEV))
    check(grads, 2.0, torch.rand(1000, device=DEV))
    check(grads, 1e6, torch.rand(3, device=DEV))


@pytest.mark.parametrize("rows", [1, 4096, 100_001])
def test_rows_join_the_norm(rows):
    r = torch.rand(rows, device=DEV)
    check([rand(1000, torch.float32)], 1.5, r)
    check([], 1.5, r)
    check([rand(50, torch.bfloat16)], 1.5, torch.rand((rows, 2), device=DEV)[:, 0])


@pytest.mark.parametrize("dtype", DT)
def test_layouts(dtype):
    a, b = rand((60, 70), dtype).t(), rand((4, 3, 20, 30), dtype).contiguous(memory_format=torch.channels_last)
    c = torch.full((100, 50), 7.0, device=DEV, dtype=dtype)
    view = c[:, 3:40]  # not in one piece
    odd = rand(20_001, dtype)[1:]  # off 16 bytes
    every = rand((9000,), dtype)[::3]
    edge = c.clone()
    check([a, b, view, odd, every], 1.0)
    assert torch.equal(c[:, :3], edge[:, :3]) and torch.equal(c[:, 40:], edge[:, 40:])


def test_slices_of_one_bucket():
    bucket = rand(50_000, torch.bfloat16)
    rest = bucket.clone()
    check([bucket[:10_001], bucket[10_001:30_000], bucket[40_000:]], 1.0)
    assert torch.equal(bucket[30_000:40_000], rest[30_000:40_000])


def test_shared_memory_is_refused():
    x = rand(100, torch.float32)
    for grads in ([x, x], [x[:60], x[50:]], [x.view(10, 10), rand(5, torch.float16), x[99:]]):
        with pytest.raises(ValueError, match="share memory"):
            clip_global_norm(grads, 1.0)
        global_norm_scale(grads, 1.0)  # nothing is written


@pytest.mark.parametrize("dtype", DT)
def test_not_finite(dtype):
    big = rand(5000, dtype)
    big[77] = math.inf
    other = rand(5000, torch.float32)
    got = clip_global_norm([big, other], 1.0)
    assert float(got[0]) == 0.0 and math.isinf(float(got[1]))
    assert (other == 0).all() and math.isnan(float(big[77]))
    bad = rand(5000, dtype)
    bad[5] = math.nan
    got = clip_global_norm([bad, other], 1.0)
    assert torch.isnan(got).all() and torch.isnan(bad).all() and torch.isnan(other).all()


def test_squares_beyond_fp32():
    """Squares that overflow or vanish in fp32, norms that do not."""
    check([torch.full((100,), 1e25, device=DEV)], 1.0)
    check([torch.full((100,), 1e-30, device=DEV)], 1.0)
    check([torch.full((100,), 1e25, device=DEV), torch.full((7,), 1e-25, device=DEV)], 1e20)


def test_graph_and_stream():
    grads = [rand((100, 300), DT[i % 3], seed=i) for i in range(300)]
    saved = [g.clone() for g in grads]
    rows = torch.rand(5000, device=DEV)
    want = clip_global_norm(grads, 3.0, row_sq=rows)
    expect = [g.clone() for g in grads]

    def restore(f=1.0):
        for g, s in zip(grads, saved):
            g.copy_(s * f)

    side = torch.cuda.Stream()
    restore()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = clip_global_norm(grads, 3.0, row_sq=rows)
    side.synchronize()
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(grads, expect))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = clip_global_norm(grads, 3.0, row_sq=rows)
    for i in range(3):
        restore(0.5 if i == 1 else 1.0)
        if i == 1:
            half = [g.clone() for g in grads]
            eager = clip_global_norm(half, 3.0, row_sq=rows)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager if i == 1 else want)
        assert all(torch.equal(a, b) for a, b in zip(grads, half if i == 1 else expect))


def test_sparse_update_with_many_dense_gradients():
    from model_amd import rows

    def update():
        values = rand((64, 16), torch.float16, seed=3)
        return rows.SparseRowUpdate(values, grad_clip=1.0, lr=0.1), values

    g = torch.Generator(device=DEV).manual_seed(4)
    aux = {"slots": [torch.randint(0, 64, (20, 2, 4), generator=g, device=DEV, dtype=torch.int32)],
           "weights": [torch.rand((20, 2, 4), generator=g, device=DEV)]}
    probe = {0: rand((20, 16), torch.float32, seed=5)}
    dense = [rand(1000, torch.float32, seed=i) for i in range(6)]
    upd, v0 = update()
    want = upd(aux, probe, [0], dense_grads=dense)
    upd, v1 = update()
    many = [half for d in dense for half in d.clone().chunk(2)]
    got = upd(aux, probe, [0], dense_grads=many)
    assert abs(float(got["grad_scale"]) - float(want["grad_scale"])) <= 2 ** -22 * float(want["grad_scale"])
    # a scale one fp32 step away moves a row by less than a step of fp16 and its neighbour
    assert (v1.float() - v0.float()).abs().max() <= 2 ** -10 * v0.float().abs().max()
    upd, v2 = update()
    clipped = [d.clone() for d in many]
    got2 = upd(aux, probe, [0], dense_grads=clipped, clip_dense=True)
    assert torch.equal(got2["grad_scale"], got["grad_scale"]) and torch.equal(v1, v2)
    for a, b in zip(clipped, many):
        assert torch.equal(a, b * got["grad_scale"])
    upd, _ = update()
    with pytest.raises(ValueError, match="clip_dense"):
        upd(aux, probe, [0], rest_sq=torch.ones(1, device=DEV), clip_dense=True)
