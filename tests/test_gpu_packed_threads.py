"""packed_attention and clip_global_norm in several threads and on several streams at once."""

import threading

import pytest
import torch

from model_amd.attention import packed_attention, packed_attention_backward, packed_attention_forward
from model_amd.grad_clip import clip_global_norm
from tests.test_gpu_packed_attention import DEV, make, sums

pytestmark = pytest.mark.gpu

SETS = [([300, 1, 40], 4, 2, 64, torch.float16), ([5, 700, 90], 6, 2, 32, torch.bfloat16), ([129, 200], 2, 2, 128, torch.float32)]


def attention_inputs(i):
    lq, H, G, hd, dtype = SETS[i]
    return *make(lq, lq, H, G, hd, dtype, seed=50 + i), torch.tensor(sums(lq), dtype=torch.int32, device=DEV)


def direct(q, k, v, g, gl, starts):
    out, lse = packed_attention_forward(q, k, v, starts)
    return out, lse, *packed_attention_backward(g, q, k, v, out, lse, starts, g_lse=gl)


def step(q, k, v, g, gl, starts):
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out, lse = packed_attention(*leaves, starts, return_lse=True)
    return out.detach(), lse.detach(), *torch.autograd.grad([out, lse], leaves, [g, gl])


def gradients(i):
    g = torch.Generator(device=DEV).manual_seed(60 + i)
    return [torch.randn(50 + 997 * j % (3000 + i), generator=g, device=DEV).to((torch.float32, torch.float16, torch.bfloat16)[j % 3])
            for j in range(250 + i)]


def clipped(grads):
    grads = [x.clone() for x in grads]
    return [clip_global_norm(grads, 2.0), *grads]


def alike(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("call,inputs", [(direct, attention_inputs), (lambda *x: clipped(x), gradients)])
def test_on_streams(call, inputs):
    """Calls on three streams at once: each has its own workspace."""
    args = [inputs(i) for i in range(3)]
    want = [call(*x) for x in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        got = []
        for s, x in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(call(*x))
        torch.cuda.synchronize()
        assert all(alike(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("call,inputs", [(step, attention_inputs), (lambda *x: clipped(x), gradients)])
def test_in_threads(call, inputs):
    """Three threads, each on a stream of its own."""
    args = [inputs(i) for i in range(3)]
    want = [call(*x) for x in args]
    torch.cuda.synchronize()
    got, failed = [[] for _ in range(3)], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(8):
                    got[i].append(call(*args[i]))
            stream.synchronize()
        except Exception as e:  # shown by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert all(alike(want[i], x) for i in range(3) for x in got[i])
