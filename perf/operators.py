"""The measured operators of the backbone's training step: layer norm and the softmax cross entropy over the vocabulary.

Each case is a dict of plain values whose ``kind`` names what runs:

  norm        y = LayerNorm(x) (with ``add``: s = x + r, y = LayerNorm(s)), inference
  norm_grad   the same with its gradients: d x (which is also d r), d scale, d bias
  loss        the loss of each token, logsumexp_v(hidden . embedding_v) - hidden . embedding_target, inference
  loss_grad   the same with d hidden and d embedding; with ``lse`` the logsumexp is an output with a gradient too

``rows`` is the number of tokens of a call, ``d`` the width, ``vocab`` the rows of the embedding table, ``dtype`` the
type of the activations (and of the table), ``param`` that of the layer norm's scale and bias.  ``form`` is how the
gradients are asked for: "autograd" through torch's, "direct" through the calls that a captured step makes.

Where ``own`` is false, ``run`` computes the same in elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
IGNORE = -100
DTYPE = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def _norm(name, kind, rows, d, dtype="fp32", param="fp32", add=False, form="autograd"):
    return {"name": name, "kind": kind, "rows": rows, "d": d, "dtype": dtype, "param": param, "add": add, "form": form}


def _loss(name, kind, rows, vocab, d, dtype="fp32", lse=False, form="autograd"):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "d": d, "dtype": dtype, "lse": lse, "form": form}


def listed():
    return [
        # one layer norm of a decode step, 64 streams of the generation workload
        _norm("norm_64x256", "norm", 64, 256),
        # the text-study batch (32 x 256 tokens), the backbone's own width and type, one training step's norm
        _norm("norm_grad_8192x256", "norm_grad", 8192, 256),
        # a ragged batch of odd width in half precision with its residual add
        _norm("norm_add_grad_4001x1283_fp16", "norm_grad", 4001, 1283, "fp16", "fp16", add=True),
        # a long batch of a wide backbone in bfloat16 with fp32 parameters and the residual add before it
        _norm("norm_add_grad_16384x4096_bf16", "norm_grad", 16384, 4096, "bf16", add=True),
        # few very wide rows
        _norm("norm_grad_300x16384", "norm_grad", 300, 16384, form="direct"),
        # the log-probability of one token: latency
        _loss("loss_1x16384", "loss", 1, 16384, 256),
        # evaluation: 16 sequences of 256 tokens on the generation workload's vocabulary and width
        _loss("loss_4096x16384", "loss", 4096, 16384, 256),
        # the text-study batch's training step on that vocabulary
        _loss("loss_grad_8192x16384", "loss_grad", 8192, 16384, 256),
        # a small batch in bfloat16, gradients without autograd as a captured step asks for them
        _loss("loss_grad_256x16384_bf16", "loss_grad", 256, 16384, 256, "bf16", form="direct"),
        # rows, vocabulary and width off the powers of two, half precision, with a gradient through the logsumexp
        _loss("loss_grad_1001x50021_fp16", "loss_grad", 1001, 50021, 500, "fp16", lse=True),
        # a wide backbone's batch
        _loss("loss_grad_8192x32000_bf16", "loss_grad", 8192, 32000, 2048, "bf16"),
        # the largest: 64 x 256 tokens over 131,072 words
        _loss("loss_grad_16384x131072_bf16", "loss_grad", 16384, 131072, 1024, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "norm_grad", "loss", "loss_grad", "loss_grad", "loss_grad"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "bf16", "fp16"])
    form = rng.choice(["autograd", "direct"])
    if kind.startswith("norm"):
        d = _log_int(rng, 16, 16384)
        if rng.random() < 0.6:
            d = -(-d // 8) * 8
        rows = _log_int(rng, 1, min(65536, 16384 * 4096 // d))
        c = _norm("", kind, rows, d, dtype, rng.choice(["fp32", dtype]), rng.random() < 0.5, form)
    else:
        d = _log_int(rng, 32, 2048)
        if rng.random() < 0.7:
            d = -(-d // 64) * 64
        vocab = _log_int(rng, 64, 131072)
        most = 16384 * 131072 * 1024 // (vocab * d * (2 if dtype == "fp32" else 1))
        rows = _log_int(rng, 1, max(1, min(16384, most)))
        c = _loss("", kind, rows, vocab, d, dtype, kind == "loss_grad" and rng.random() < 0.3, form)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def prepare(case, seed):
    c, g, t = case, _gen(seed), DTYPE[case["dtype"]]
    R, d = c["rows"], c["d"]
    grads = c["kind"].endswith("_grad")
    if c["kind"].startswith("norm"):
        pt = DTYPE[c["param"]]
        # the residual stream: a mean and a size of each row's own
        x = torch.randn((R, d), generator=g, device=DEV)
        x = x * (0.3 + torch.rand((R, 1), generator=g, device=DEV)) + torch.randn((R, 1), generator=g, device=DEV)
        s = {"x": x.to(t), "scale": (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(pt),
             "bias": (0.1 * torch.randn(d, generator=g, device=DEV)).to(pt)}
        if c["add"]:
            s["r"] = (0.5 * torch.randn((R, d), generator=g, device=DEV)).to(t)
        leaves = [n for n in ("x", "r", "scale", "bias") if n in s]
        if grads:
            s["g_y"] = torch.randn((R, d), generator=g, device=DEV).to(t)
            if c["add"]:
                s["g_s"] = torch.randn((R, d), generator=g, device=DEV).to(t)
    else:
        V = c["vocab"]
        emb = torch.randn((V, d), generator=g, device=DEV) * d ** -0.5
        # words by Zipf's law; the hidden rows of a model some way into training point towards their targets
        u = torch.rand(R, generator=g, device=DEV)
        target = (torch.exp(u * math.log(V)) - 1).long().clamp_(0, V - 1)
        hidden = torch.randn((R, d), generator=g, device=DEV) + 0.6 * math.log(V) * emb[target]
        target[torch.rand(R, generator=g, device=DEV) < 0.06] = IGNORE  # padding
        s = {"hidden": hidden.to(t), "embedding": emb.to(t), "target": target}
        leaves = ["hidden", "embedding"]
        if grads:
            # the mean over the batch of weighted tokens, under a loss scale where the type is fp16
            unit = (1024.0 if c["dtype"] == "fp16" else 1.0) / R
            s["g_loss"] = torch.rand(R, generator=g, device=DEV) * unit
            if c["lse"]:
                s["g_lse"] = torch.randn(R, generator=g, device=DEV) * 1e-2 * unit
    if grads and c["form"] == "autograd":
        for n in leaves:
            s[n].requires_grad_(True)
    s.update(case=c)
    return s


# -------------------------------------------------------------------- runs
def _own_norm(s, c):
    from model_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward

    if c["kind"] == "norm":
        with torch.no_grad():
            out = layer_norm(s["x"], s["scale"], s["bias"], EPS, residual=s.get("r"))
        return {"y": out[0], "s": out[1]} if c["add"] else {"y": out}
    if c["form"] == "direct":
        y, total, mean, rstd = layer_norm_forward(s["x"], s["scale"], s["bias"], EPS, residual=s.get("r"))
        dx, dscale, dbias = layer_norm_backward(s["g_y"], total, s["scale"], mean, rstd, g_residual=s.get("g_s"))
        out = {"y": y, "d_x": dx, "d_scale": dscale, "d_bias": dbias}
        if c["add"]:
            out["s"] = total
        return out
    if c["add"]:
        y, total = layer_norm(s["x"], s["scale"], s["bias"], EPS, residual=s["r"])
        dx, _, dscale, dbias = torch.autograd.grad([y, total], [s["x"], s["r"], s["scale"], s["bias"]],
                                                   [s["g_y"], s["g_s"]])
        return {"y": y, "d_x": dx, "d_scale": dscale, "d_bias": dbias, "s": total}
    y = layer_norm(s["x"], s["scale"], s["bias"], EPS)
    dx, dscale, dbias = torch.autograd.grad(y, [s["x"], s["scale"], s["bias"]], s["g_y"])
    return {"y": y, "d_x": dx, "d_scale": dscale, "d_bias": dbias}


def _own_loss(s, c):
    from model_amd.cross_entropy import vocab_cross_entropy, vocab_cross_entropy_grads

    h, e, t = s["hidden"], s["embedding"], s["target"]
    if c["kind"] == "loss":
        with torch.no_grad():
            return {"loss": vocab_cross_entropy(h, e, t, ignore_index=IGNORE)}
    if c["form"] == "direct":
        loss, lse, dh, de = vocab_cross_entropy_grads(h, e, t, s["g_loss"], g_lse=s.get("g_lse"), ignore_index=IGNORE)
    elif c["lse"]:
        loss, lse = vocab_cross_entropy(h, e, t, ignore_index=IGNORE, return_lse=True)
        dh, de = torch.autograd.grad([loss, lse], [h, e], [s["g_loss"], s["g_lse"]])
    else:
        loss = vocab_cross_entropy(h, e, t, ignore_index=IGNORE)
        dh, de = torch.autograd.grad(loss, [h, e], s["g_loss"])
    out = {"loss": loss, "d_hidden": dh, "d_embedding": de}
    if c["lse"]:
        out["lse"] = lse
    return out


def _plain_norm(s, c):
    x, t = s["x"], s["x"].dtype
    total = (x.float() + s["r"].float()).to(t) if c["add"] else x
    f, scale = total.float(), s["scale"].float()
    f = f - f.mean(-1, keepdim=True)
    rstd = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    hat = f * rstd
    out = {"y": (hat * scale + s["bias"].float()).to(t)}
    if c["kind"] == "norm_grad":
        gy = s["g_y"].float()
        gh = gy * scale
        dx = rstd * (gh - gh.mean(-1, keepdim=True) - hat * (gh * hat).mean(-1, keepdim=True))
        if c["add"]:
            dx = dx + s["g_s"].float()
        pt = s["scale"].dtype
        out.update(d_x=dx.to(t), d_scale=(gy * hat).sum(0).to(pt), d_bias=gy.sum(0).to(pt))
    if c["add"]:
        out["s"] = total
    return out


def _plain_loss(s, c):
    h, e, target = s["hidden"].float(), s["embedding"].float(), s["target"]
    z = torch.matmul(h, e.t())
    top = z.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    there = target != IGNORE
    at = torch.where(there, target, 0)[:, None]
    loss = torch.where(there, (lse - z.gather(1, at))[:, 0], 0.0)
    out = {"loss": loss}
    if c["kind"] == "loss_grad":
        t = s["hidden"].dtype
        g = torch.where(there, s["g_loss"], 0.0)[:, None]
        g_all = g + s["g_lse"][:, None] if c["lse"] else g
        dz = z.sub_(lse).exp_().mul_(g_all)
        dz.scatter_add_(1, at, -g)
        out.update(d_hidden=torch.matmul(dz, e).to(t), d_embedding=torch.matmul(dz.t(), h).to(t))
        if c["lse"]:
            out["lse"] = lse[:, 0]
    return out


def run(state):
    c = state["case"]
    if c["kind"].startswith("norm"):
        if own:
            return _own_norm(state, c)
        with torch.no_grad():
            return _plain_norm(state, c)
    if own:
        return _own_loss(state, c)
    with torch.no_grad():
        return _plain_loss(state, c)


# -------------------------------------------------------------------- work
def work(case):
    c, size, R, d = case, SIZE[case["dtype"]], case["rows"], case["d"]
    grads = c["kind"].endswith("_grad")
    if c["kind"].startswith("norm"):
        ps = SIZE[c["param"]]
        arrays = 2 + 2 * c["add"]  # x, y, and with the add r and s
        if grads:
            arrays += 2 + c["add"]  # g_y, d_x, and with the add g_s
        return {"bytes": float(arrays * R * d * size + (4 if grads else 2) * d * ps),
                "flops": (20.0 if grads else 8.0) * R * d}
    V = c["vocab"]
    bytes_ = (R + V) * d * size * (2 if grads else 1) + R * (8 + 4 + (4 if grads else 0) + (8 if c["lse"] else 0))
    return {"bytes": float(bytes_), "flops": (6.0 if grads else 2.0) * R * V * d}


# ------------------------------------------------------------------- exact
def _exact_norm(s, c):
    x = s["x"].detach().double()
    if c["add"]:
        # the residual stream is held in its own type, and the norm is that of the stream
        x = (x + s["r"].detach().double()).to(s["x"].dtype).double()
    scale, n = s["scale"].detach().double(), x.shape[1]
    dev = x - (x.sum(1) / n)[:, None]
    inv = 1.0 / torch.sqrt(dev.square().sum(1) / n + EPS)
    out = {"y": dev * inv[:, None] * scale[None] + s["bias"].detach().double()[None]}
    if c["kind"] == "norm_grad":
        gy = s["g_y"].double()
        a = (gy * scale[None]).sum(1) / n
        b = (gy * scale[None] * dev).sum(1) / n * inv.pow(3)
        dx = gy * scale[None] * inv[:, None] - (a * inv)[:, None] - dev * b[:, None]
        if c["add"]:
            dx += s["g_s"].double()
        out.update(d_x=dx, d_scale=torch.mv((gy * dev).t().contiguous(), inv), d_bias=gy.sum(0))
    if c["add"]:
        out["s"] = s["x"].detach().double() + s["r"].detach().double()
    return out


def _exact_loss(s, c):
    h, e, target = s["hidden"].detach().double(), s["embedding"].detach().double(), s["target"]
    R, V, grads = c["rows"], c["vocab"], c["kind"] == "loss_grad"
    loss = torch.zeros(R, dtype=torch.float64, device=h.device)
    lse, dh, de = torch.empty_like(loss), torch.empty_like(h), torch.zeros_like(e)
    step = max(1, (1 << 29) // V)  # rows at a time: 4 GiB of logits
    for i in range(0, R, step):
        part, t = h[i:i + step], target[i:i + step]
        logits = part @ e.t()
        lse[i:i + step] = torch.logsumexp(logits, 1)
        rows = torch.nonzero(t != IGNORE)[:, 0]
        loss[i + rows] = lse[i + rows] - logits[rows, t[rows]]
        if grads:
            g = torch.zeros_like(lse[i:i + step])
            g[rows] = s["g_loss"][i + rows].double()
            weight = g + s["g_lse"][i:i + step].double() if c["lse"] else g
            d_logits = torch.softmax(logits, 1) * weight[:, None]
            d_logits[rows, t[rows]] -= g[rows]
            dh[i:i + step] = d_logits @ e
            de += d_logits.t() @ part
    out = {"loss": loss}
    if grads:
        out.update(d_hidden=dh, d_embedding=de)
        if c["lse"]:
            out["lse"] = lse
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(s, case) if case["kind"].startswith("norm") else _exact_loss(s, case)
