"""clip_global_norm of gradients that do not lie in one piece: such as share an element are refused, whatever their
layout, and nothing is written; such as lie between each other are clipped."""

import pytest
import torch

from model_amd.grad_clip import clip_global_norm, global_norm_scale
from tests.test_gpu_grad_clip import DEV, check, rand

pytestmark = pytest.mark.gpu


def w(dtype=torch.float32):
    return rand((40, 30), dtype, seed=1)


def cases():
    """(name, gradients of a matrix, whether they share an element)"""
    return [
        ("the same columns twice", lambda x: [x[:, :5], x[:, :5]], True),
        ("columns that overlap", lambda x: [x[:, :10], x[:, 9:20]], True),
        ("every second and third", lambda x: [x[:, ::2], x[:, ::3]], True),
        ("a matrix and its columns", lambda x: [x, x[:, 3:7]], True),
        ("the matrix transposed", lambda x: [x.t()[3:7], x[:, 6:9]], True),
        ("columns and a row", lambda x: [x[:, 20:], x[7]], True),
        ("one element", lambda x: [x[:, 29:], x.view(-1)[1199:]], True),
        ("rows of other widths", lambda x: [x.view(-1).as_strided((20, 3), (7, 1)), x.view(-1).as_strided((20, 3), (11, 1), 2)], True),
        ("four axes", lambda x: [x.view(5, 8, 6, 5)[:, 1:7, :, 2], x.view(5, 8, 6, 5)[2, :, 3:5]], True),
        ("another type", lambda x: [x[:, 4:8], x.view(torch.uint8).view(torch.float16 if x.element_size() == 4 else x.dtype)[:, 4 * (x.element_size() // 2):][:, :3]], True),
        ("a negated view", lambda x: [torch._neg_view(x), x[:, 1:3]], True),
        ("columns side by side", lambda x: [x[:, :10], x[:, 10:25], x[:, 25:]], False),
        ("every second", lambda x: [x[:, ::2], x[:, 1::2]], False),
        ("every fourth and second", lambda x: [x.view(-1)[::2], x.view(-1)[1::4], x.view(-1)[3::4]], False),
        ("columns and what lies between them", lambda x: [x[:, :10], x[3, 10:], x[4, 10:], x[5:9, 10:20]], False),
        ("four axes apart", lambda x: [x.view(5, 8, 6, 5)[:, :, 1:3, ::2], x.view(5, 8, 6, 5)[:, :, 3:, 1:], x.view(5, 8, 6, 5)[:, 2, 0]], False),
        ("transposed columns", lambda x: [x.t()[:5], x[:, 5:9], x.t()[9:20].t()], False),
    ]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name,make,share", cases(), ids=[c[0] for c in cases()])
def test_views_of_one_matrix(dtype, name, make, share):
    x = w(dtype)
    grads = make(x)
    if not share:
        check(grads, 1.0)
        return
    before = x.clone()
    for order in (grads, grads[::-1], [rand((9,), dtype), *grads, rand((3, 3), dtype)[:, :2]]):
        with pytest.raises(ValueError, match="share memory"):
            clip_global_norm(order, 1.0)
    assert torch.equal(x, before)
    global_norm_scale(grads, 1.0)  # nothing is written


def test_against_places():
    """Random views of one buffer against the places that they take."""
    import random

    rng = random.Random(7)
    base = rand((2000,), torch.float32)
    seen = {True: 0, False: 0}
    for _ in range(300):
        views, places = [], []
        for _ in range(2):
            dims = rng.randint(1, 3)
            size = [rng.randint(1, 6) for _ in range(dims)]
            stride, step = [], rng.randint(1, 4)
            for n in size:  # no element of a view twice
                stride.append(step)
                step = step * n + rng.randint(0, 5)
            order = rng.sample(range(dims), dims)
            at = rng.randint(0, 60)
            views.append(base.as_strided([size[i] for i in order], [stride[i] for i in order], at))
            where = torch.arange(2000).as_strided(views[-1].shape, views[-1].stride(), at)
            places.append(set(where.reshape(-1).tolist()))
        share = bool(places[0] & places[1])
        seen[share] += 1
        if share:
            with pytest.raises(ValueError, match="share memory"):
                clip_global_norm(views, 1e9)
        else:
            clip_global_norm(views, 1e9)
    assert min(seen.values()) > 30


def test_many_columns():
    x = rand((64, 4000), torch.bfloat16)
    check(list(x.split(10, 1)), 1.0)
