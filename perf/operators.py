"""Performance cases of the language model's two ends: the token table going in, the losses over the vocabulary coming
out.

The kinds of case, each over the range that `draw` spans:

    ce       `linear_cross_entropy`: per-token losses of the tied head over a vocabulary of about 500 to 32768 words,
             from one token to a batch of 16384, logits never kept; scored only, or with the gradients of the hidden
             rows and of the table. Some labels are padding.
    distill  `linear_distill`: the distillation loss from a teacher's top logits, alone or with the cross entropy of the
             labels from the same pass; scored only or with gradients. Some teachers' lists are shorter than others, and
             some tokens have none.
    embed    `embedding`: rows looked up with a scale, alone or with the table's gradient by sorted tokens; fp32 and
             bf16 tables, frequent and rare words, some ids padding.

Training hands over per-token weights (1 / valid tokens) as the losses' gradients.
"""
import math

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # one reply of a few words scored under the benchmark's model: latency
        {"name": "ce_score_reply", "kind": "ce", "n": 7, "V": 8192, "d": 768, "grad": False},
        # a batch of held-out text scored (bits per byte of an evaluation), d704 model
        {"name": "ce_score_batch", "kind": "ce", "n": 8190, "V": 8192, "d": 704, "grad": False},
        # the benchmark's training shape: 16 sequences of 512
        {"name": "ce_step", "kind": "ce", "n": 8192, "V": 8192, "d": 768, "grad": True},
        # a short ragged batch over an odd vocabulary: a fine-tuning step
        {"name": "ce_step_odd", "kind": "ce", "n": 1001, "V": 10007, "d": 512, "grad": True},
        # the largest: a long batch over a large vocabulary
        {"name": "ce_step_large", "kind": "ce", "n": 16384, "V": 32768, "d": 768, "grad": True},
        # distillation on a micro-batch with the labels' loss beside it, softened
        {"name": "distill_step", "kind": "distill", "n": 8192, "V": 8192, "d": 768, "K": 32, "tau": 2.0, "ce": True,
         "grad": True},
        # distillation alone at temperature one, ragged, odd vocabulary, a long list
        {"name": "distill_odd", "kind": "distill", "n": 1500, "V": 12001, "d": 704, "K": 100, "tau": 1.0, "ce": False,
         "grad": True},
        # a student's distance to its teacher measured on a short text
        {"name": "distill_score", "kind": "distill", "n": 200, "V": 8192, "d": 768, "K": 16, "tau": 1.0, "ce": True,
         "grad": False},
        # a short prompt's rows: latency
        {"name": "embed_prompt", "kind": "embed", "n": 100, "V": 8192, "d": 768, "bf16": False, "grad": False},
        # the benchmark's training shape, fp32 table
        {"name": "embed_step", "kind": "embed", "n": 8192, "V": 8192, "d": 768, "bf16": False, "grad": True},
        # a ragged batch over an odd vocabulary, bf16 table
        {"name": "embed_step_odd", "kind": "embed", "n": 3001, "V": 10007, "d": 704, "bf16": True, "grad": True},
        # a long batch over a large vocabulary
        {"name": "embed_step_large", "kind": "embed", "n": 65536, "V": 32768, "d": 768, "bf16": False, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "distill", "distill", "embed"])
    d = rng.choice([256, 328, 512, 704, 768, 1000, 1024])
    V = _log(rng, 500, 32768)
    if rng.random() < 0.5:
        V = max(512, V // 256 * 256)
    if kind == "embed":
        n = min(_log(rng, 1, 65536), (48 << 20) // d)
        return {"kind": kind, "n": n, "V": V, "d": d, "bf16": rng.random() < 0.4, "grad": rng.random() < 0.8}
    n = max(1, min(_log(rng, 1, 16384), (1 << 37) // (V * d)))
    grad = rng.random() < 0.75
    if kind == "ce":
        return {"kind": kind, "n": n, "V": V, "d": d, "grad": grad}
    return {"kind": kind, "n": n, "V": V, "d": d, "K": _log(rng, 1, 128), "tau": rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]),
            "ce": rng.random() < 0.5, "grad": grad}


# ------------------------------------------------------------------------------------------------------------------
# inputs

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _padded(g, ids, share, pad):
    return torch.where(torch.rand(ids.shape, generator=g, device=DEV) < share, torch.full_like(ids, pad), ids)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, V, d = case["n"], case["V"], case["d"]
    if case["kind"] == "embed":
        # word frequencies fall off as a power of the rank, ranks scattered over the ids; two in a hundred are padding
        rank = (float(V) ** torch.rand(n, generator=g, device=DEV)).long().clamp(1, V) - 1
        ids = _padded(g, torch.randperm(V, generator=g, device=DEV)[rank], 0.02, -1)
        dt = torch.bfloat16 if case["bf16"] else torch.float32
        s = {"kind": "embed", "grad": case["grad"], "ids": ids, "W": (0.02 * _randn(g, V, d)).to(dt), "scale": d ** 0.5}
        if case["grad"]:
            s["gy"] = (_randn(g, n, d) / n).to(dt)
        return s
    # normalised hidden rows, a table whose logits spread by about two: a model some way into its training
    h = torch.nn.functional.layer_norm(_randn(g, n, d), (d,)).bfloat16()
    W = (2.0 * d ** -0.5 * _randn(g, V, d)).bfloat16()
    y = _padded(g, torch.randint(0, V, (n,), generator=g, device=DEV), 0.06, -100)
    per_token = torch.where(y >= 0, 1.0, 0.0) / (y >= 0).sum().clamp(min=1)
    s = {"kind": case["kind"], "grad": case["grad"], "h": h, "W": W, "y": y, "gce": per_token}
    if case["kind"] == "distill":
        # the teacher: the student's own view of a somewhat different hidden row; lists cut short at random, one token
        # in sixteen with none
        K = case["K"]
        z, ids = ((0.8 * h.float() + 0.6 * _randn(g, n, d)) @ W.float().t()).topk(K, dim=1)
        kept = torch.randint(max(1, K // 2), K + 1, (n, 1), generator=g, device=DEV)
        kept = torch.where(torch.rand(n, 1, generator=g, device=DEV) < 0.06, torch.zeros_like(kept), kept)
        ids = torch.where(torch.arange(K, device=DEV) < kept, ids, -1)
        s |= {"ids": ids, "z": z.contiguous(), "tau": case["tau"], "gkd": torch.full((n,), 1.0 / n, device=DEV)}
        if not case["ce"]:
            s["y"] = None
    return s


# ------------------------------------------------------------------------------------------------------------------
# the framework's calls

def _own_ce(s):
    from pragnosia_amd.head import linear_cross_entropy
    if not s["grad"]:
        with torch.no_grad():
            return linear_cross_entropy(s["h"], s["W"], s["y"])
    h, W = s["h"].detach().requires_grad_(), s["W"].detach().requires_grad_()
    loss, lse = linear_cross_entropy(h, W, s["y"])
    return (loss.detach(), lse.detach(), *torch.autograd.grad(loss, (h, W), s["gce"]))


def _own_distill(s):
    from pragnosia_amd.head import linear_distill
    if not s["grad"]:
        with torch.no_grad():
            return linear_distill(s["h"], s["W"], s["ids"], s["z"], s["tau"], s["y"])
    h, W = s["h"].detach().requires_grad_(), s["W"].detach().requires_grad_()
    kd, ce = linear_distill(h, W, s["ids"], s["z"], s["tau"], s["y"])
    if ce is None:
        return (kd.detach(), None, *torch.autograd.grad(kd, (h, W), s["gkd"]))
    return (kd.detach(), ce.detach(), *torch.autograd.grad((kd, ce), (h, W), (s["gkd"], s["gce"])))


def _own_embed(s):
    from pragnosia_amd.embed import embedding
    if not s["grad"]:
        with torch.no_grad():
            return embedding(s["ids"], s["W"], s["scale"])
    W = s["W"].detach().requires_grad_()
    out = embedding(s["ids"], W, s["scale"])
    return (out.detach(), *torch.autograd.grad(out, W, s["gy"]))


# ------------------------------------------------------------------------------------------------------------------
# the plain forms

def _lse(x):
    m = x.amax(1, keepdim=True)
    return (x - m).exp().sum(1).log() + m[:, 0]


def _plain_ce(s):
    h, W, y = s["h"].float(), s["W"].float(), s["y"]
    x = h @ W.t()
    lse = _lse(x)
    valid, at = (y >= 0) & (y < W.shape[0]), y.clamp(0, W.shape[0] - 1)[:, None]
    loss = torch.where(valid, lse - x.gather(1, at)[:, 0], 0.0)
    if not s["grad"]:
        return loss, lse
    g = torch.where(valid, s["gce"], 0.0)[:, None]
    dx = (x - lse[:, None]).exp() * g
    dx.scatter_add_(1, at, -g)
    return loss, lse, (dx @ W).to(s["h"].dtype), (dx.t() @ h).to(s["W"].dtype)


def _plain_distill(s):
    h, W, ids, tau, y = s["h"].float(), s["W"].float(), s["ids"], s["tau"], s["y"]
    V = W.shape[0]
    x = h @ W.t()
    there = (ids >= 0) & (ids < V)
    at, some = ids.clamp(0, V - 1), there.any(1)
    z = torch.where(there, s["z"] / tau, -math.inf)
    e = torch.where(there, (z - torch.where(some, z.amax(1), 0.0)[:, None]).exp(), 0.0)
    p = e / e.sum(1, keepdim=True).clamp(min=1e-30)
    lse_t = _lse(x / tau)
    logp = torch.where(p > 0, p.clamp(min=1e-38).log(), 0.0)
    kd = tau * tau * (p * (logp - (x.gather(1, at) / tau - lse_t[:, None]))).sum(1)
    ce = None
    if y is not None:
        lse = _lse(x)
        valid, yt = (y >= 0) & (y < V), y.clamp(0, V - 1)[:, None]
        ce = torch.where(valid, lse - x.gather(1, yt)[:, 0], 0.0)
    if not s["grad"]:
        return kd, ce
    gk = s["gkd"][:, None] * tau
    dx = (x / tau - lse_t[:, None]).exp() * torch.where(some[:, None], gk, 0.0)
    dx.scatter_add_(1, at, -gk * p)
    if y is not None:
        g = torch.where(valid, s["gce"], 0.0)[:, None]
        dx += (x - lse[:, None]).exp() * g
        dx.scatter_add_(1, yt, -g)
    return kd, ce, (dx @ W).to(s["h"].dtype), (dx.t() @ h).to(s["W"].dtype)


def _plain_embed(s):
    ids, W, scale = s["ids"], s["W"], s["scale"]
    valid, at = ((ids >= 0) & (ids < W.shape[0]))[:, None], ids.clamp(0, W.shape[0] - 1)
    out = torch.where(valid, W[at].float() * scale, 0.0).to(W.dtype)
    if not s["grad"]:
        return out
    gy = torch.where(valid, s["gy"].float() * scale, 0.0)
    return out, torch.zeros(W.shape, device=W.device).index_add_(0, at, gy).to(W.dtype)


def run(state):
    if own:
        return {"ce": _own_ce, "distill": _own_distill, "embed": _own_embed}[state["kind"]](state)
    return {"ce": _plain_ce, "distill": _plain_distill, "embed": _plain_embed}[state["kind"]](state)


def work(case):
    n, V, d, grad = case["n"], case["V"], case["d"], case["grad"]
    if case["kind"] == "embed":
        size = 2 if case["bf16"] else 4
        # distinct rows, as the word frequencies give them: a row is read once however often it is looked up
        rows = round(sum(1 - (1 - math.log1p(1 / r) / math.log(V)) ** (0.98 * n) for r in range(1, V)))
        return {"bytes": 8 * n + size * d * (rows + n) + (size * d * (n + V) if grad else 0),
                "flops": n * d * (3 if grad else 1)}
    sums = 2 * n * V * d
    data = 2 * d * (n + V) * (2 if grad else 1)
    if case["kind"] == "ce":
        return {"bytes": data + 16 * n + (4 * n if grad else 0), "flops": sums * (3 if grad else 1)}
    return {"bytes": data + 12 * n * case["K"] + 4 * n + (12 * n if case["ce"] else 0) + (8 * n if grad else 0),
            "flops": sums * (3 if grad else 1)}


# ------------------------------------------------------------------------------------------------------------------
# in 64 bits, from the definitions: a block of rows at a time

def _exact_head(s):
    W = s["W"].double()
    V, rows = W.shape[0], max(1, (1 << 26) // W.shape[0])
    tau, parts, dW = s.get("tau", 1.0), [], torch.zeros_like(W)
    for a in range(0, s["h"].shape[0], rows):
        h = s["h"][a:a + rows].double()
        x = h @ W.mT
        k, out, dx = torch.arange(h.shape[0], device=DEV), {}, torch.zeros_like(x)
        if s["kind"] == "distill":
            ids = s["ids"][a:a + rows]
            on = ids.ge(0) & ids.lt(V)
            t = torch.zeros_like(x)  # the teacher's distribution over the whole vocabulary
            z = s["z"][a:a + rows].double().div(tau).masked_fill(~on, -math.inf)
            t.scatter_add_(1, ids * on, torch.softmax(z, 1).nan_to_num(0.0))
            lq = torch.log_softmax(x / tau, 1)
            out["kd"] = tau ** 2 * (torch.xlogy(t, t) - t * lq).sum(1)
            if s["grad"]:
                dx += tau * s["gkd"][a:a + rows, None].double() * (lq.exp() * t.sum(1, keepdim=True) - t)
        if s["y"] is not None:
            y = s["y"][a:a + rows]
            on = y.ge(0) & y.lt(V)
            lp = torch.log_softmax(x, 1)
            out["ce"] = -lp[k, y * on] * on
            out["lse"] = torch.logsumexp(x, 1)
            if s["grad"]:
                g = s["gce"][a:a + rows].double() * on
                dx += g[:, None] * lp.exp()
                dx[k, y * on] -= g
        if s["grad"]:
            out["dh"] = dx @ W
            dW += dx.mT @ h
        parts.append(out)
    cat = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    first = (cat["ce"], cat["lse"]) if s["kind"] == "ce" else (cat["kd"], cat.get("ce"))
    return (*first, cat["dh"], dW) if s["grad"] else first


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] != "embed":
        return _exact_head(s)
    V, d = s["W"].shape
    on = s["ids"].ge(0) & s["ids"].lt(V)
    table = torch.cat([s["W"].double() * s["scale"], torch.zeros(1, d, device=DEV, dtype=torch.float64)])
    row = s["ids"].where(on, torch.full_like(s["ids"], V))
    if not s["grad"]:
        return table[row]
    dW = torch.zeros_like(table).index_put_((row,), s["gy"].double() * s["scale"], accumulate=True)
    return table[row], dW[:V]
