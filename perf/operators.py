"""The operators at the two ends of the language model: token ids in, log probabilities out.

- ``embed``, ``embed_train``   token_embedding: scaled token rows plus position rows behind the persistent
                               rows, and the gradients of the three tables
- ``score``                    token_logprobs of stored logits, with entropy and top alternatives
- ``loss_train``               token_cross_entropy, forward and the logits' gradient
- ``policy_train``             token_logprobs with entropy, forward and backward of both
- ``head``                     head_logprobs: the same scores from the hidden states and the head's weight,
                               the logits never stored

Sizes are those of the model's configurations (d_model 640, vocabularies of 50000 and 128000, sequences of
4096, 16 persistent tokens) and odd ones around them.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100


def _tc():
    pkg = os.path.join(os.getcwd(), "titanmac-standalone_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import titans_core
    return titans_core


# ------------------------------------------------------------------ the cases

def _embed(kind, B, T, V, dtype, d=640, prefix=16, scale=1.0, given=False):
    """given: the positions are given per sequence (decoding), not 0 .. T - 1."""
    return {"kind": kind, "B": B, "T": T, "V": V, "d": d, "prefix": prefix, "scale": scale, "given": given,
            "dtype": dtype}


def _score(kind, B, T, V, dtype, entropy=False, top=0, pad=0):
    """pad: vocabulary entries at the end that are masked with -inf."""
    return {"kind": kind, "B": B, "T": T, "V": V, "entropy": entropy, "top": top, "pad": pad, "dtype": dtype}


def _head(B, T, V, dtype, d=640, entropy=False):
    return {"kind": "head", "B": B, "T": T, "V": V, "d": d, "entropy": entropy, "dtype": dtype}


def listed():
    return [
        # 16 sequences decode one token each, every one at its own position: latency
        dict(_embed("embed", 16, 1, 50000, "bf16", prefix=0, given=True), name="embed_decode_16"),
        # a prefill of 4 sequences of 4096 behind the persistent tokens
        dict(_embed("embed", 4, 4096, 128000, "bf16"), name="embed_prefill_4x4096"),
        # a training batch of 8 sequences of 4096: the lookup and the gradients of all three tables
        dict(_embed("embed_train", 8, 4096, 128000, "bf16"), name="embed_train_8x4096"),
        # a small ragged batch without mixed precision, token rows scaled by sqrt(d)
        dict(_embed("embed_train", 3, 683, 50000, "fp32", d=512, prefix=4, scale=math.sqrt(512.0)),
             name="embed_train_f32_3x683"),
        # a server reports each decoded token's score, its entropy and 20 alternatives
        dict(_score("score", 16, 1, 50000, "bf16", entropy=True, top=20), name="score_decode_16"),
        # one sequence, fp32 logits, the most alternatives that are offered
        dict(_score("score", 1, 1, 128000, "fp32", entropy=True, top=64), name="score_one_top64"),
        # the scores of four prompts with five alternatives at each position
        dict(_score("score", 4, 1024, 128000, "bf16", top=5), name="score_prompt_4x1024"),
        # the loss of a training batch and the gradient of its logits
        dict(_score("loss_train", 4, 2048, 128000, "bf16"), name="loss_train_4x2048"),
        # a policy update: log probabilities and entropies both carry gradients; an odd vocabulary whose
        # padding is masked
        dict(_score("policy_train", 3, 333, 50001, "fp32", entropy=True, pad=17), name="policy_train_f32_3x333"),
        # scores of one decoded token for each of 16 sequences, straight from the hidden states
        dict(_head(16, 1, 128000, "bf16"), name="head_decode_16"),
        # scores of 4 sequences of 2048 without their 2 GB of logits
        dict(_head(4, 2048, 128000, "bf16"), name="head_score_4x2048"),
        # an odd number of rows and of entries, wider model, with entropies
        dict(_head(3, 501, 50001, "fp16", d=1024, entropy=True), name="head_entropy_3x501"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_train", "embed_train", "score", "score", "loss_train", "policy_train",
                       "head", "head"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    V = rng.choice([_log_int(rng, 1000, 128000), _log_int(rng, 30000, 128000), 50000, 128000])
    if kind in ("embed", "embed_train"):
        T = _log_int(rng, 1, 4096)
        B = rng.randint(1, 8) if T > 64 else _log_int(rng, 1, 64)
        return _embed(kind, B, T, V if kind == "embed_train" else max(V, 8000), dtype if dtype != "fp32" else
                      rng.choice(["bf16", "fp32"]), d=rng.choice([256, 512, 640]), prefix=rng.choice([0, 4, 16, 33]),
                      scale=rng.choice([1.0, 1.0, 16.0, 0.5]), given=rng.random() < 0.3)
    if kind == "head":
        d = rng.choice([256, 512, 640])
        M = _log_int(rng, 1, 8192)
        return _head(1, M, V, rng.choice(["bf16", "fp16"]), d=d, entropy=rng.random() < 0.4)
    z = SIZES[dtype]
    M = _log_int(rng, 1, max(1, min(8192, int((0.5e9 if kind == "score" else 1e9) * 2 / z / V))))
    B = rng.choice([1, 2, 3, 4])
    T = max(1, M // B)
    if kind == "score":
        return _score(kind, B, T, V, dtype, entropy=rng.random() < 0.5, top=rng.choice([0, 1, 5, 20, 33, 64]),
                      pad=rng.choice([0, 0, 7, 64]))
    return _score(kind, B, T, V, dtype, entropy=kind == "policy_train", pad=rng.choice([0, 0, 7, 64]))


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _zipf(g, V, *shape):
    """Token ids whose frequency falls as 1 / (rank + 1), as a text's does."""
    u = torch.rand(*shape, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(V + 1.0)).floor().long() - 1).clamp_(0, V - 1)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _targets(g, c):
    """The tokens whose log probability is asked; in training one in 16 is padding."""
    t = _zipf(g, c["V"] - c.get("pad", 0), c["B"], c["T"])
    if c["kind"] in ("loss_train", "policy_train"):
        drop = torch.rand(c["B"], c["T"], generator=g, device=DEV) < 1 / 16
        drop[0, 0] = False
        t = t.masked_fill(drop, IGNORE)
    return t


def prepare(case, seed):
    c, dt, g = case, DTYPES[case["dtype"]], _gen(seed)
    s = {"case": c}
    kind = c["kind"]
    if kind in ("embed", "embed_train"):
        B, T, d, n_pos = c["B"], c["T"], c["d"], 4096
        s["ids"] = _zipf(g, c["V"], B, T)
        s["w"] = _randn(g, c["V"], d, scale=0.02, dtype=dt)
        s["p"] = _randn(g, n_pos, d, scale=0.02, dtype=dt)
        s["prefix"] = _randn(g, c["prefix"], d, scale=0.02, dtype=dt) if c["prefix"] else None
        s["pos"] = None
        if c["given"]:
            first = torch.randint(0, n_pos - T + 1, (B, 1), generator=g, device=DEV)
            s["pos"] = first + torch.arange(T, device=DEV)
        if kind == "embed_train":
            s["gy"] = _randn(g, B, c["prefix"] + T, d, scale=1e-3, dtype=dt)
            for n in ("w", "p", "prefix"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
    elif kind == "head":
        s["h"] = _randn(g, c["B"], c["T"], c["d"], dtype=dt)
        s["w"] = _randn(g, c["V"], c["d"], scale=2.0 / math.sqrt(c["d"]), dtype=dt)
        s["targets"] = _targets(g, c)
    else:
        s["z"] = _randn(g, c["B"], c["T"], c["V"], scale=2.0, dtype=dt)
        if c["pad"]:
            s["z"][..., -c["pad"]:] = float("-inf")
        s["targets"] = _targets(g, c)
        if kind in ("loss_train", "policy_train"):
            s["z"].requires_grad_(True)
        if kind == "policy_train":
            s["g_lp"] = _randn(g, c["B"], c["T"], scale=1e-2)
            s["g_ent"] = _randn(g, c["B"], c["T"], scale=1e-3)
    return s


# ------------------------------------------------------------------ one pass, plain form

def _plain_embed(s, c):
    ids, w, p, prefix = s["ids"], s["w"].detach(), s["p"].detach(), s["prefix"]
    B, T = ids.shape
    pos = torch.arange(T, device=DEV).expand(B, T) if s["pos"] is None else s["pos"]
    y = (w[ids].float() * c["scale"] + p[pos].float()).to(w.dtype)
    if prefix is not None:
        y = torch.cat([prefix.detach().expand(B, -1, -1), y], dim=1)
    if c["kind"] == "embed":
        return y
    n, d = c["prefix"], c["d"]
    g = s["gy"][:, n:].float().reshape(B * T, d)
    dw = torch.zeros(w.shape, dtype=torch.float32, device=DEV).index_add_(0, ids.reshape(-1), g) * c["scale"]
    dp = torch.zeros(p.shape, dtype=torch.float32, device=DEV).index_add_(0, pos.reshape(-1), g)
    out = {"y": y, "dw": dw.to(w.dtype), "dp": dp.to(w.dtype)}
    if prefix is not None:
        out["dprefix"] = s["gy"][:, :n].float().sum(0).to(w.dtype)
    return out


def _plain_scores(z, targets, entropy, top):
    """z [B, T, V] in 32 bits -> the scores, and the exponentials and their sum for the gradients."""
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    lse = (m + torch.log(total)).squeeze(-1)
    skip = targets == IGNORE
    zt = z.gather(-1, targets.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    out = {"logprobs": ((zt - m.squeeze(-1)) - torch.log(total.squeeze(-1))).masked_fill(skip, 0.0)}
    if entropy:
        out["entropy"] = (torch.log(total) - (e * (z - m).clamp(min=-1e30)).sum(-1, keepdim=True) / total).squeeze(-1)
    if top:
        # one whole number that orders by value, then by the lower index
        bits = (z + 0.0).view(torch.int32).long()  # -0 counts as 0
        key = torch.where(bits < 0, ~bits & 0xFFFFFFFF, bits | 0x80000000) - 0x80000000
        key = key * (1 << 24) + (z.shape[-1] - 1 - torch.arange(z.shape[-1], device=DEV))
        out["top_ids"] = key.topk(top, dim=-1).indices
        out["top_logprobs"] = z.gather(-1, out["top_ids"]) - lse.unsqueeze(-1)
    return out, e, total


def _plain_logits(s, c):
    zt, targets = s["z"].detach(), s["targets"]
    z = zt.float()
    out, e, total = _plain_scores(z, targets, c["entropy"], c["top"])
    if c["kind"] == "score":
        return out
    p = e / total
    keep = targets != IGNORE
    if c["kind"] == "loss_train":
        n = keep.sum()
        out = {"loss": (-(out["logprobs"].sum() / n)).to(zt.dtype)}
        g_lp = keep / -n.float()
    else:
        g_lp = s["g_lp"] * keep
    dz = -g_lp.unsqueeze(-1) * p
    dz.scatter_add_(-1, targets.clamp(min=0).unsqueeze(-1), g_lp.unsqueeze(-1))
    if c["kind"] == "policy_train":
        logp = (torch.log(e) - torch.log(total)).clamp(min=-1e30)
        dz -= s["g_ent"].unsqueeze(-1) * p * (logp + out["entropy"].unsqueeze(-1))
    return {**out, "dz": dz.to(zt.dtype)}


def _plain_head(s, c):
    z = s["h"].float() @ s["w"].float().t()
    return _plain_scores(z, s["targets"], c["entropy"], 0)[0]


# ------------------------------------------------------------------ one pass, the framework's calls

def _own_embed(s, c):
    tc = _tc()
    y = tc.token_embedding(s["ids"], s["w"], s["p"], positions=s["pos"], prefix=s["prefix"], scale=c["scale"])
    if c["kind"] == "embed":
        return y
    tables = [s["w"], s["p"]] + ([] if s["prefix"] is None else [s["prefix"]])
    g = torch.autograd.grad(y, tables, s["gy"])
    return {"y": y.detach(), **dict(zip(("dw", "dp", "dprefix"), g))}


def _named(r):
    return {n: t.detach() for n, t in r._asdict().items() if t is not None}


def _own_logits(s, c):
    tc = _tc()
    if c["kind"] == "loss_train":
        loss = tc.token_cross_entropy(s["z"], s["targets"], ignore_index=IGNORE)
        return {"loss": loss.detach(), "dz": torch.autograd.grad(loss, s["z"])[0]}
    r = tc.token_logprobs(s["z"], s["targets"], entropy=c["entropy"], top_k=c["top"], ignore_index=IGNORE)
    if c["kind"] == "score":
        return _named(r)
    dz, = torch.autograd.grad([r.logprobs, r.entropy], s["z"], [s["g_lp"], s["g_ent"]])
    return {**_named(r), "dz": dz}


def run(state):
    s, c = state, state["case"]
    if c["kind"] in ("embed", "embed_train"):
        return _own_embed(s, c) if own else _plain_embed(s, c)
    if c["kind"] == "head":
        if own:
            return _named(_tc().head_logprobs(s["h"], s["w"], s["targets"], entropy=c["entropy"]))
        return _plain_head(s, c)
    return _own_logits(s, c) if own else _plain_logits(s, c)


# ------------------------------------------------------------------ the least work of a pass

def _distinct(V, n):
    """How many different ids n draws of _zipf are expected to hold."""
    p = np.diff(np.log(np.arange(1, V + 2))) / math.log(V + 1.0)
    return float((1.0 - np.exp(n * np.log1p(-p))).sum())


def work(case):
    c = case
    kind, z = c["kind"], SIZES[c["dtype"]]
    n = c["B"] * c["T"]
    if kind in ("embed", "embed_train"):
        d, S = c["d"], c["prefix"] + c["T"]
        rows = _distinct(c["V"], n) + (min(n, 4096) if c["given"] else c["T"]) + c["prefix"]
        b, f = 8 * n + (rows + c["B"] * S) * d * z, 2 * n * d
        if kind == "embed_train":
            b += (c["B"] * S + c["V"] + 4096 + c["prefix"]) * d * z
            f += 2 * c["B"] * S * d
        return {"bytes": int(b), "flops": f}
    if kind == "head":
        return {"bytes": (n + c["V"]) * c["d"] * z + 12 * n, "flops": 2 * n * c["V"] * c["d"]}
    train = kind != "score"
    per = 4 + (2 if c["entropy"] else 0) + ((3 + (3 if c["entropy"] else 0)) if train else 0)
    return {"bytes": n * c["V"] * z * (2 if train else 1) + n * (12 + 4 * c["entropy"] + 12 * c["top"]),
            "flops": n * c["V"] * per}


# ------------------------------------------------------------------ the same in 64 bits

def _exact_embed(s, c):
    w, p = s["w"].detach().double(), s["p"].detach().double()
    ids, B, T = s["ids"], c["B"], c["T"]
    pos = torch.arange(T, device=DEV).repeat(B, 1) if s["pos"] is None else s["pos"]
    y = torch.nn.functional.embedding(ids, w).mul_(c["scale"]).add_(torch.nn.functional.embedding(pos, p))
    n = c["prefix"]
    if n:
        y = torch.cat([s["prefix"].detach().double()[None].repeat(B, 1, 1), y], 1)
    if c["kind"] == "embed":
        return y
    g = s["gy"].double()
    body = g[:, n:]
    dw, dp = torch.zeros_like(w), torch.zeros_like(p)
    for b in range(B):
        dw.index_put_((ids[b],), body[b] * c["scale"], accumulate=True)
        dp.index_put_((pos[b],), body[b], accumulate=True)
    out = {"y": y, "dw": dw, "dp": dp}
    if n:
        out["dprefix"] = sum(g[b, :n] for b in range(B))
    return out


def _exact_rows(z, targets, c):
    """The scores of rows z [n, V] in 64 bits; log_p too, for the gradients."""
    log_p = torch.log_softmax(z, dim=-1)
    skip = targets == IGNORE
    lp = log_p[torch.arange(len(targets), device=DEV), targets.masked_fill(skip, 0)].masked_fill(skip, 0.0)
    out = {"logprobs": lp}
    if c["entropy"]:
        out["entropy"] = -torch.where(log_p == -math.inf, 0.0, log_p.exp() * log_p).sum(-1)
    if c.get("top"):
        order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        out["top_ids"], out["top_logprobs"] = order, log_p.gather(-1, order)
    return out, log_p


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    if kind in ("embed", "embed_train"):
        return _exact_embed(s, c)
    V, n = c["V"], c["B"] * c["T"]
    targets = s["targets"].reshape(-1)
    parts, grads = [], []
    count = int((targets != IGNORE).sum())
    w = s["w"].double() if kind == "head" else None
    step = max(1, (1 << 27) // V)
    for a in range(0, n, step):
        at = slice(a, a + step)
        if kind == "head":
            z = s["h"].reshape(n, -1)[at].double() @ w.t()
        else:
            z = s["z"].detach().reshape(n, V)[at].double()
        out, log_p = _exact_rows(z, targets[at], c)
        parts.append(out)
        if kind in ("loss_train", "policy_train"):
            t = targets[at]
            keep = (t != IGNORE).double()
            g = -keep / count if kind == "loss_train" else s["g_lp"].reshape(-1)[at].double() * keep
            p = log_p.exp()
            dz = p * -g[:, None]
            dz[torch.arange(len(t), device=DEV), t.clamp(min=0)] += g
            if kind == "policy_train":
                ge = s["g_ent"].reshape(-1)[at].double()[:, None]
                dz -= torch.where(p == 0, 0.0, p * (log_p + out["entropy"][:, None])) * ge
            grads.append(dz)
    shape = (c["B"], c["T"])
    res = {k: torch.cat([o[k] for o in parts]) for k in parts[0]}
    res = {k: t.reshape(shape + t.shape[1:]) for k, t in res.items()}
    if kind == "loss_train":
        res = {"loss": -res["logprobs"].sum() / count}
    if grads:
        res["dz"] = torch.cat(grads).reshape(shape + (V,))
    return res
