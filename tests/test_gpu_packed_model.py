"""MemoryPoolLM over packed sequences: each sequence as if it stood alone, the
gradients as the sum of theirs, and a training step of token_loss, backward pass and
clip together.

Tolerances: tests/test_gpu_token_loss.py counts 2e-4 of the norm of each gradient and 2e-5 of
the losses for two ways through the same fp32 blocks."""

import pytest
import torch

from model_amd.grad_clip import clip_global_norm
from model_amd.model import MemoryPoolLM, ModelConfig

pytestmark = pytest.mark.gpu

LENGTHS = [7, 1, 0, 40, 33, 2]


def _setup(**kw):
    base = dict(vocab_size=301, max_len=40, d_model=128, n_layers=3, n_heads=4, ffn_mult=2, memory_layers=(1,),
                n_sub_keys=32, pool_heads=4, d_key=64, d_value=128, top_k=8, values_dtype=torch.float32)
    base.update(kw)
    model = MemoryPoolLM(ModelConfig(**base))
    params = model.init(5)["params"]
    g = torch.Generator(device="cuda").manual_seed(11)
    n = sum(LENGTHS)
    tokens = torch.randint(0, 301, (1, n), generator=g, device="cuda")
    targets = torch.randint(0, 301, (1, n), generator=g, device="cuda")
    starts = torch.tensor([0, *torch.tensor(LENGTHS).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    targets[0, starts[1:][torch.tensor(LENGTHS) > 0] - 1] = -100
    return model, params, tokens, targets, starts


def _leaves(t):
    return [x for v in (t[k] for k in sorted(t)) for x in (_leaves(v) if isinstance(v, dict) else [v])]


def _pieces(starts):
    s = starts.tolist()
    return [slice(a, b) for a, b in zip(s, s[1:]) if b > a]


CASES = [dict(), dict(memory_ffn=True, memory_layers=(0, 2)), dict(use_memory=False, n_heads=1)]


@pytest.mark.parametrize("kw", CASES)
def test_each_sequence_as_if_alone(gpu_lib, kw):
    model, params, tokens, targets, starts = _setup(**kw)
    for grad in (False, True):
        for p in _leaves(params):
            p.requires_grad_(grad and p.is_floating_point())
        with torch.set_grad_enabled(grad):
            logits, _ = model.apply(params, tokens, starts=starts)
            loss, lse, _ = model.token_loss(params, tokens, targets, starts=starts.long(), return_lse=True)
            assert logits.shape == (1, sum(LENGTHS), 301) and loss.shape == targets.shape
            for at in _pieces(starts):
                want, _ = model.apply(params, tokens[:, at])
                assert (logits[:, at] - want).abs().max() <= 2e-5 * want.abs().max().clamp(min=1)
                one, z, _ = model.token_loss(params, tokens[:, at], targets[:, at], return_lse=True)
                assert (loss[:, at] - one).abs().max() <= 2e-5 * one.abs().max().clamp(min=1)
                assert (lse[:, at] - z).abs().max() <= 2e-5 * z.abs().max().clamp(min=1)


@pytest.mark.parametrize("kw", CASES)
def test_gradients_are_the_sum_of_the_sequences(gpu_lib, kw):
    model, params, tokens, targets, starts = _setup(**kw)
    leaves = [p.requires_grad_(True) for p in _leaves(params)]

    def grads(loss):
        return [torch.zeros_like(p) if g is None else g
                for g, p in zip(torch.autograd.grad(loss, leaves, allow_unused=True), leaves)]

    got = grads(model.token_loss(params, tokens, targets, starts=starts)[0].sum())
    want = [torch.zeros_like(p) for p in leaves]
    for at in _pieces(starts):
        for w, g in zip(want, grads(model.token_loss(params, tokens[:, at], targets[:, at])[0].sum())):
            w += g
    # the key's bias adds one number to all scores of a query: its gradient is 0, a sum whose terms
    # cancel, and what rounding leaves of it is measured by the query's, of terms alike in size
    sizes = [w.norm() for w in want]
    for i, p in enumerate(leaves):
        for layer in range(model.cfg.n_layers):
            att = params[f"attn_{layer}"]
            if p is att["key"]["bias"]:
                sizes[i] = sizes[next(j for j, x in enumerate(leaves) if x is att["query"]["bias"])]
    for g, w, size in zip(got, want, sizes):
        assert (g - w).norm() <= 2e-4 * size + 1e-7


def test_a_training_step(gpu_lib):
    """token_loss over packed sequences, its backward pass, the clip and a step: the
    clipped gradients have the clip's norm, and the step is the plain one's."""
    model, params, tokens, targets, starts = _setup()
    leaves = [p.requires_grad_(True) for p in _leaves(params)]
    loss, aux = model.token_loss(params, tokens, targets, starts=starts, train=True, noise_scale=0.0)
    (loss.sum() / (targets != -100).sum() + 0.01 * aux["balance_loss"]).backward()
    dense = [p.grad for p in leaves if p.grad is not None]
    before = [g.clone() for g in dense]
    norm = torch.sqrt(sum(g.double().square().sum() for g in before))
    scale, got = clip_global_norm(dense, 0.25 * float(norm)).tolist()
    assert abs(got - float(norm)) <= 1e-6 * got and abs(scale - 0.25) <= 1e-6
    after = torch.sqrt(sum(g.double().square().sum() for g in dense))
    assert abs(float(after) - 0.25 * float(norm)) <= 1e-5 * float(norm)
    for g, b in zip(dense, before):
        assert torch.equal(g, b * scale)


def test_positions_past_the_table_are_nan(gpu_lib):
    model, params, tokens, targets, starts = _setup(max_len=33)
    with torch.no_grad():
        logits, _ = model.apply(params, tokens, starts=starts)
    bad = torch.isnan(logits).any(-1)[0]
    assert bad[41:48].all() and not bad[:8].any() and not bad[48:].any()  # the sequence of 40 alone


def test_refusals(gpu_lib):
    model, params, tokens, targets, starts = _setup(dropout=0.1)
    model.token_loss(params, tokens, targets, starts=starts)
    for call in (lambda: model.token_loss(params, tokens, targets, starts=starts, train=True),
                 lambda: model.apply(params, tokens, starts=starts, train=True)):
        with pytest.raises(ValueError, match="no dropout"):
            call()
    with pytest.raises(ValueError, match="starts on cpu"):
        model.token_loss(params, tokens, targets, starts=starts.cpu())
    model, params, tokens, targets, starts = _setup(n_heads=8)
    with pytest.raises(ValueError, match="heads of 32, 64 or 128"):
        model.apply(params, tokens, starts=starts)
