"""MemoryPoolLM.token_loss: layer norms with their adds, output layer and loss
together, against apply()'s logits and torch's log_softmax.

Both sides are fp32 through the same blocks; they differ by the roundings of
the norms, the logits and their sums.  A product of K terms is off by at most
K 2^-24 of its terms' magnitudes, some 10 to 20 such products (and as many
norms, 2^-18 each as tests/test_gpu_layer_norm.py has it) follow each other,
K <= 256, and errors of random sign add by their roots: 2e-4 of the norm of
each gradient, and 2e-5 of the losses."""

import pytest
import torch

from model_amd.model import MemoryPoolLM, ModelConfig

pytestmark = pytest.mark.gpu


def _setup(seed=0, **kw):
    base = dict(vocab_size=301, max_len=40, d_model=128, n_layers=3, n_heads=4, ffn_mult=2, memory_layers=(1,),
                n_sub_keys=32, pool_heads=4, d_key=64, d_value=128, top_k=8, values_dtype=torch.float32)
    base.update(kw)
    cfg = ModelConfig(**base)
    model = MemoryPoolLM(cfg)
    params = model.init(seed)["params"]
    g = torch.Generator(device="cuda").manual_seed(seed + 7)
    tokens = torch.randint(0, cfg.vocab_size, (3, 37), generator=g, device="cuda")
    targets = torch.randint(0, cfg.vocab_size, (3, 37), generator=g, device="cuda")
    targets[:, -2:] = -100
    return model, params, tokens, targets


def _leaves(t, out=None, path=""):
    out = {} if out is None else out
    for k in sorted(t):
        if isinstance(t[k], dict):
            _leaves(t[k], out, path + k + "/")
        else:
            out[path + k] = t[k]
    return out


def _reference(logits, targets):
    ls = torch.log_softmax(logits, -1)
    return torch.where(targets == -100, 0.0, -ls.gather(-1, targets.clamp(min=0)[..., None])[..., 0])


@pytest.mark.parametrize("kw", [dict(), dict(memory_ffn=True, memory_layers=(0, 2)), dict(use_memory=False),
                                dict(d_model=100, n_heads=2, use_memory=False), dict(n_layers=1, memory_layers=())])
def test_loss_and_gradients_equal_the_logits_path(gpu_lib, kw):
    model, params, tokens, targets = _setup(**kw)
    print(f"token loss {kw}", flush=True)
    leaves = {k: v.requires_grad_(True) for k, v in _leaves(params).items() if not k.startswith("pool/values")}
    w = torch.rand(targets.shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    logits, aux = model.apply(params, tokens)
    want = _reference(logits, targets)
    loss, aux2 = model.token_loss(params, tokens, targets)
    if model.pool is not None and model.cfg.memory_layers:
        assert all(torch.equal(a, b) for a, b in zip(aux["slots"], aux2["slots"]))  # the same rows are read
    assert loss.shape == targets.shape and (loss[targets == -100] == 0).all()
    assert (loss - want).norm() <= 2e-5 * want.norm()
    names = [k for k in leaves if k != "pool/log_temperature"]
    a = torch.autograd.grad((want * w).sum(), [leaves[k] for k in names], allow_unused=True)
    b = torch.autograd.grad((loss * w).sum(), [leaves[k] for k in names], allow_unused=True)
    size = dict(zip(names, a))
    for k, x, y in zip(names, a, b):
        assert (x is None) == (y is None), k
        if x is None:
            continue
        # a softmax ignores a shift of its scores: the key biases' gradients are 0 but for
        # roundings of what the query biases' are made of
        scale = size[k.replace("key/bias", "query/bias")].norm()
        assert (x - y).norm() <= 2e-4 * scale, (k, (x - y).norm().item(), x.norm().item())


def test_training_step_options(gpu_lib):
    """dropout, routing noise, sparse gradients and probes as apply() takes them."""
    model, params, tokens, targets = _setup(dropout=0.2, memory_layers=(1, 2))
    B, T = tokens.shape

    def step(f):
        probes = {i: torch.zeros((B, T, model.cfg.d_value), device="cuda", requires_grad=True) for i in (1, 2)}
        out, aux = f(probes)
        grads = torch.autograd.grad(out.sum(), [probes[1], probes[2]])
        return out, aux, grads

    kw = dict(train=True, sparse_grad=True, rngs={"dropout": 5, "routing": 9})
    for v in _leaves(params).values():
        v.requires_grad_(True)
    want, aux, ga = step(lambda pr: (lambda r: (_reference(r[0], targets), r[1]))(
        model.apply(params, tokens, probes=pr, **kw)))
    loss, aux2, gb = step(lambda pr: model.token_loss(params, tokens, targets, probes=pr, **kw))
    assert all(torch.equal(a, b) for a, b in zip(aux["slots"], aux2["slots"]))
    assert (loss - want).norm() <= 2e-5 * want.norm()
    for x, y in zip(ga, gb):
        assert (x - y).norm() <= 2e-4 * x.norm()


def test_evaluation(gpu_lib):
    """Under no_grad (the fused launches), with the logsumexp, and with the pool off."""
    model, params, tokens, targets = _setup()
    with torch.no_grad():
        for kw in (dict(), dict(pool_off=True)):
            logits, _ = model.apply(params, tokens, **kw)
            want = _reference(logits, targets)
            loss, lse, _ = model.token_loss(params, tokens, targets.int(), return_lse=True, **kw)
            assert (loss - want).norm() <= 2e-5 * want.norm()
            assert (lse - torch.logsumexp(logits, -1)).norm() <= 2e-5 * lse.norm()


def test_one_token(gpu_lib):
    model, params, tokens, targets = _setup()
    with torch.no_grad():
        logits, _ = model.apply(params, tokens[:1, :1])
        loss, _ = model.token_loss(params, tokens[:1, :1], targets[:1, :1])
        assert (loss - _reference(logits, targets[:1, :1])).abs().max() <= 2e-5 * 10


def test_refusals(gpu_lib):
    model, params, tokens, targets = _setup()
    with pytest.raises(ValueError, match="targets"):
        model.token_loss(params, tokens, targets[:, 1:])
    with pytest.raises(ValueError, match="decode"):
        MemoryPoolLM(model.cfg, decode=True).token_loss(params, tokens, targets)
