"""layer_norm and vocab_cross_entropy in several threads and on several streams at once."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _norm_inputs(seed, R=700, d=520, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return rnd(R, d).to(dtype), rnd(d), rnd(d), rnd(R, d).to(dtype), rnd(R, d).to(dtype), rnd(R, d).to(dtype)


def _norm_calls(x, w, b, r, gy, gs):
    from model_amd.layer_norm import layer_norm_backward, layer_norm_forward

    y, s, mean, rstd = layer_norm_forward(x, w, b, residual=r)
    return y, s, *layer_norm_backward(gy, s, w, mean, rstd, g_residual=gs)


def _norm_step(x, w, b, r, gy, gs):
    from model_amd.layer_norm import layer_norm

    leaves = [t.clone().requires_grad_() for t in (x, r, w, b)]
    y, s = layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    dx, dr, dw, db = torch.autograd.grad([y, s], leaves, [gy, gs])
    assert torch.equal(dx, dr)
    return y.detach(), s.detach(), dx, dw, db


def test_layer_norm_on_two_streams(gpu_lib):
    """Calls on two streams at once: each has its own workspace."""
    args = [_norm_inputs(s) for s in (1, 2)]
    want = [_norm_calls(*x) for x in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        got = []
        for s, x in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(_norm_calls(*x))
        torch.cuda.synchronize()
        for x, y in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_layer_norm_in_two_threads(gpu_lib):
    """Autograd steps in two threads, each on a stream of its own."""
    args = [_norm_inputs(s, 300 + s, 1283, torch.float16) for s in (3, 4)]
    want = [_norm_calls(*x) for x in args]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                got[i] = _norm_step(*args[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    for x, y in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_pretended_capture_is_one_threads(gpu_lib):
    """What makes a thread's backward passes behave as under capture leaves
    those of other threads alone, and ends with its thread."""
    from model_amd import _lib
    from model_amd.cross_entropy import vocab_cross_entropy
    from model_amd.layer_norm import layer_norm

    x = torch.randn(20, 64, device="cuda", requires_grad=True)
    w, b, e = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda"), torch.randn(30, 64, device="cuda")
    t = torch.arange(20, device="cuda")
    ways = [lambda: layer_norm(x, w, b).sum(), lambda: vocab_cross_entropy(x, e, t).sum()]
    ran = []

    def steps():
        for f in ways:
            torch.autograd.grad(f(), x)
            ran.append(f)

    def pretends_and_ends():
        _lib.ops().pretend_capturing(True)

    def in_thread(f):
        thread = threading.Thread(target=f)
        thread.start()
        thread.join()

    steps()
    ops = _lib.ops()
    ops.pretend_capturing(True)
    try:
        for f in ways:
            with pytest.raises(RuntimeError, match="under HIP graph capture"):
                torch.autograd.grad(f(), x)
        in_thread(steps)
        assert len(ran) == 4
    finally:
        ops.pretend_capturing(False)
    in_thread(pretends_and_ends)
    steps()
    assert len(ran) == 6
