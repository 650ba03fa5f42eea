"""packed_attention at the ends of its sizes: rows as far apart as they may lie, thousands of sequences."""

import math
import random

import pytest
import torch

from tests.test_gpu_packed_attention import DEV, DT, E, F64, check, make, sums
from tests.test_gpu_packed_attention_values import all_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd", [(4, 2, 64), (128, 128, 128), (512, 512, 32), (256, 256, 64)])
def test_tokens_2_23_elements_apart(dtype, H, G, hd):
    """q, k, v and the output's gradient lie in one buffer of 5 or 10 GB, so that a stage of the large calls' tiles (128
    rows of heads of 32) spans 2^31 bytes, and a sequence more than 2^32: every bit as of the same rows close together."""
    lq = [130, 1, 169]
    n, pitch = sum(lq), 1 << 23
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.fail("needs 24 GiB")
    q, k, v, g, gl = make(lq, lq, H, G, hd, dtype, seed=41)
    starts = torch.tensor(sums(lq), dtype=torch.int32, device=DEV)
    want = all_of(q, k, v, g, gl, starts)
    buffer = torch.empty(n * pitch, dtype=dtype, device=DEV)
    far, at = [], 0
    for x in (q, k, v, g):
        far.append(buffer.as_strided(x.shape, (pitch, hd, 1), at))
        far[-1].copy_(x)
        at += x[0].numel()
    for nm, a, b in zip(("out", "lse", "dq", "dk", "dv"), want, all_of(*far, gl, starts)):
        assert torch.equal(a, b), nm


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,G,hd", [(2, 1, 32), (4, 4, 64)])
def test_gradients_of_thousands_of_sequences(dtype, H, G, hd):
    """More sequences than two steps of the search tell apart (64^2), against the definition under a block mask in 64
    bits; tolerances as in test_gpu_packed_attention.py, of sequences of up to 9 tokens."""
    rng = random.Random(4300)
    lq = [rng.choice([0, 1, 2, 3, 9]) for _ in range(4300)]
    lq[-1] = 5
    T, R, most = sum(lq), H // G, 9
    q, k, v, g, gl = make(lq, lq, H, G, hd, dtype, seed=42)
    out, lse, dq, dk, dv = all_of(q, k, v, g, gl, torch.tensor(sums(lq), dtype=torch.int64, device=DEV))
    seq = torch.repeat_interleave(torch.arange(len(lq), device=DEV), torch.tensor(lq, device=DEV))
    at = torch.arange(T, device=DEV)
    seen = (seq[:, None] == seq[None]) & (at[:, None] >= at[None])
    w = torch.finfo(dtype).eps / 2
    u, small, scale = w if dtype != torch.float32 else 0.0, 2.0 ** -25 if dtype == torch.float16 else 0.0, hd ** -0.5
    dk_want, dv_want, dk_tol, dv_tol = (torch.zeros((T, G, hd), dtype=F64, device=DEV) for _ in range(4))
    mask = seen.to(F64)
    for h in range(H):
        Q, K, V, go = q[:, h].to(F64), k[:, h // R].to(F64), v[:, h // R].to(F64), g[:, h].to(F64)
        z = scale * (Q @ K.t())
        zerr = ((hd + 4) * E * scale * (Q.abs() @ K.abs().t()) + 8 * E * z.abs()).mul_(mask).amax(1)
        z.masked_fill_(~seen, -math.inf)
        lse_want = torch.logsumexp(z, 1)
        zerr = zerr + 8 * E + 4 * E * lse_want.abs()
        check(lse[:, h], (lse_want, zerr + most * E), "lse")
        p = z.sub_(lse_want[:, None]).exp_()
        rel = (u + 2 * zerr + most * E)[:, None]
        out_want = p @ V
        tol_out = rel * (p @ V.abs()) + w * out_want.abs() + small * (mask @ V.abs()) + small
        check(out[:, h], (out_want, tol_out), "out")
        dv_want[:, h // R] += p.t() @ go
        dv_tol[:, h // R] += (p * (rel + most * R * E)).t() @ go.abs() + small * (mask.t() @ go.abs())
        delta = (go * out_want).sum(1) - gl[:, h].to(F64)
        dz = (go @ V.t()).sub_(delta[:, None])
        err = (u + 2 * zerr)[:, None] * dz.abs() + ((go.abs() * tol_out).sum(1) + 4 * E * delta.abs())[:, None]
        err = p * err.add_((go.abs() @ V.abs().t()).mul_((hd + 4) * E)) + mask * (small * float(go.abs().max()) * 4)
        dz = p * dz
        dq_want = scale * (dz @ K)
        check(dq[:, h], (dq_want, scale * (err @ K.abs() + most * E * (dz.abs() @ K.abs())) + small + w * dq_want.abs()), "dq")
        dk_want[:, h // R] += scale * (dz.t() @ Q)
        dk_tol[:, h // R] += scale * (err.t() @ Q.abs() + most * R * E * (dz.abs().t() @ Q.abs())) + small
    check(dk, (dk_want, dk_tol + w * dk_want.abs()), "dk")
    check(dv, (dv_want, dv_tol + w * dv_want.abs() + small), "dv")
