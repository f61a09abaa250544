"""Performance cases of generation from 4-bit weights under rules: the weights' rounding to 4 bits, the dense layers of a
decode step on them, and the choice of the next token.

The kinds of case, each over the range that `draw` spans:

    pack    `fp4.quantize` and `fp4.dequantize`: a weight (N, K) rounded to 4-bit floating codes with a bf16 scale for each
            group of 32, 64 or 128 columns, as a generation starts, and read back; from 16 rows to 32768, fp32 and bf16.
    linear  `fp4.linear`: rows times such a weight, from one token to a batch of 512, fp32 and bf16; with a LayerNorm in
            front, a bias, GELU and a residual behind, as a block's layers have them, or without.
    rules   `rules.next_token` and `rules.apply_rules`: penalties for repeated tokens, biases of some words and a grammar's
            masks on the logits of 1 to 256 sequences over 500 to 131072 words; the best word, or the logits for a sampler.
"""
import math

import torch

own = False
DEV = "cuda"

# the values of the codes 0 .. 7; 8 .. 15 are their negatives
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    def linear(name, n, N, K, **kw):
        return {"name": name, "kind": "linear", "n": n, "N": N, "K": K, "group": 64, "bf16": False, "norm": False,
                "bias": False, "gelu": False, "resid": False} | kw

    def rules(name, B, V, L, **kw):
        return {"name": name, "kind": "rules", "B": B, "V": V, "L": L, "bf16": False, "M": 0, "states": 0,
                "token": True} | kw

    return [
        # one sequence's carrier projections (queries, keys, values, decay, gate of the d768 model): latency
        linear("linear_step", 1, 2328, 768, norm=True),
        # one sequence's head over the vocabulary
        linear("linear_head", 1, 8192, 768, norm=True),
        # the MLP's second layer of the d704 model for 64 sequences
        linear("linear_batch", 64, 704, 2816, bias=True, resid=True),
        # a few sequences of a bf16 model, odd vocabulary, the last group cut short
        linear("linear_odd", 5, 10007, 1000, group=128, bf16=True, norm=True),
        # one sequence through a wide layer: the weights' bytes
        linear("linear_one_wide", 1, 16384, 4096, group=32, bf16=True, bias=True, gelu=True),
        # the largest: 512 tokens at once (a prompt's piece, or a large batch)
        linear("linear_large", 512, 8192, 4096, bf16=True, bias=True),
        # the head's table, fp32, as a generation starts
        {"name": "pack_head", "kind": "pack", "N": 8192, "K": 768, "group": 64, "bf16": False},
        # an odd table with a short last group
        {"name": "pack_odd", "kind": "pack", "N": 10007, "K": 1000, "group": 128, "bf16": True},
        # a large bf16 weight
        {"name": "pack_large", "kind": "pack", "N": 32768, "K": 4096, "group": 32, "bf16": True},
        # one sequence that must not repeat itself: latency
        rules("rules_one", 1, 8192, 600),
        # a batch under everything: penalties, biases, a grammar
        rules("rules_batch", 64, 32768, 2000, M=100, states=64),
        # many sequences' bf16 logits for a sampler, large vocabulary
        rules("rules_large", 256, 131072, 4000, bf16=True, M=32, states=300, token=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "pack", "rules", "rules"])
    if kind == "rules":
        V = _log(rng, 500, 131072)
        return {"kind": kind, "B": min(_log(rng, 1, 256), (1 << 25) // V), "V": V, "L": _log(rng, 1, 4000),
                "bf16": rng.random() < 0.5, "M": rng.choice([0, 0, _log(rng, 1, 300)]),
                "states": rng.choice([0, _log(rng, 1, 300)]), "token": rng.random() < 0.6}
    K = rng.choice([256, 328, 512, 704, 768, 1000, 1024, 2816, 4096])
    N = _log(rng, 16, 32768)
    if rng.random() < 0.5:
        N = max(16, N // 16 * 16)
    case = {"kind": kind, "N": N, "K": K, "group": rng.choice([32, 64, 64, 128]), "bf16": rng.random() < 0.5}
    if kind == "linear":
        case |= {"n": max(1, min(_log(rng, 1, 512), (1 << 34) // (N * K)))}
        case |= {k: rng.random() < 0.5 for k in ("norm", "bias", "gelu", "resid")}
    return case


# ------------------------------------------------------------------------------------------------------------------
# inputs

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _weight(case, g):
    """Rows of different sizes, some columns larger than others, as trained weights have them."""
    N, K = case["N"], case["K"]
    W = 0.02 * _randn(g, N, K) * (0.5 * _randn(g, N, 1)).exp() * (0.3 * _randn(g, 1, K)).exp()
    return W.to(torch.bfloat16 if case["bf16"] else torch.float32)


def _linear_inputs(case, g):
    n, N, K = case["n"], case["N"], case["K"]
    dt = torch.bfloat16 if case["bf16"] else torch.float32
    W = _weight(case, g)
    codes, scales = _codes(W.float(), case["group"])
    s = {"case": case, "dtype": dt, "group": case["group"],
         # two codes a byte, the even column's in the low half; a scale for each group
         "codes": (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8), "scales": scales,
         "x": (_randn(g, n, K) * (0.3 * _randn(g, 1, K)).exp()).to(dt)}
    s["norm"] = None
    if case["norm"]:
        s["norm"] = torch.nn.LayerNorm(K, device=DEV, dtype=dt).requires_grad_(False)
        s["norm"].weight.copy_(1 + 0.1 * _randn(g, K))
        s["norm"].bias.copy_(0.1 * _randn(g, K))
    s["bias"] = (0.1 * _randn(g, N)).to(dt) if case["bias"] else None
    s["resid"] = _randn(g, n, N).to(dt) if case["resid"] else None
    return s, W


def _rules_inputs(case, g):
    B, V, L, M, S = case["B"], case["V"], case["L"], case["M"], case["states"]
    rand = lambda *shape: torch.rand(*shape, generator=g, device=DEV)  # noqa: E731
    # words by frequency, as a text repeats them; logits that lean towards what was said
    words = torch.randperm(V, generator=g, device=DEV)
    history = words[(float(V) ** rand(B, L)).long().clamp(1, V) - 1]
    lengths = (rand(B) * (L + 1)).long().clamp(max=L)
    lengths[0] = L
    prompt = (rand(B) * (lengths + 1)).long()
    logits = 3.0 * _randn(g, B, V)
    logits.scatter_add_(1, history, torch.full((B, L), 0.5, device=DEV))
    s = {"case": case, "logits": logits.to(torch.bfloat16) if case["bf16"] else logits, "history": history,
         "lengths": lengths, "prompt": prompt, "repetition": 1.0 + 0.3 * rand(B), "presence": 0.5 * rand(B),
         "frequency": 0.2 * rand(B), "ids": None, "values": None, "mask": None, "state": None}
    if M:
        # distinct words, favoured, disfavoured or banned; lists of different lengths, padded with -1
        s["ids"] = rand(B, V).topk(min(M, V), dim=1).indices
        s["ids"][rand(B, s["ids"].shape[1]) < 0.2] = -1
        s["values"] = torch.where(rand(*s["ids"].shape) < 0.2, -math.inf, 2.0 * _randn(g, *s["ids"].shape))
    if S:
        # a grammar's states: most allow a few words, some nearly all, and one none; some sequences are free
        share = torch.where(rand(S, 1) < 0.3, 0.98, 0.02)
        allowed = torch.zeros(S, (V + 31) // 32 * 32, dtype=torch.bool, device=DEV)
        allowed[:, :V] = rand(S, V) < share
        allowed[S // 2] &= S == 1
        bits = allowed.view(S, -1, 32).long() << torch.arange(32, device=DEV)
        s["mask"] = bits.sum(2).to(torch.int32)
        s["state"] = (rand(B) * (S + 1)).long().clamp(max=S) - 1
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "rules":
        return _rules_inputs(case, g)
    if case["kind"] == "pack":
        return {"case": case, "W": _weight(case, g), "group": case["group"]}
    s, W = _linear_inputs(case, g)
    if own:  # the weights as the framework keeps them: rounded once, before the first step
        from pragnosia_amd import fp4
        s["Q"] = fp4.quantize(W, case["group"])
    return s


# ------------------------------------------------------------------------------------------------------------------
# the framework's calls

def _own_linear(s):
    from pragnosia_amd import fp4
    return fp4.linear(s["x"], s["Q"], s["bias"], norm=s["norm"], act="gelu" if s["case"]["gelu"] else None,
                      resid=s["resid"])


def _own_pack(s):
    from pragnosia_amd import fp4
    Q = fp4.quantize(s["W"], s["group"])
    return fp4.dequantize(Q, s["W"].dtype)


def _own_rules(s):
    from pragnosia_amd import rules
    call = rules.next_token if s["case"]["token"] else rules.apply_rules
    return call(s["logits"], history=s["history"], lengths=s["lengths"], prompt=s["prompt"],
                repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                bias=None if s["ids"] is None else (s["ids"], s["values"]), mask=s["mask"], state=s["state"])


# ------------------------------------------------------------------------------------------------------------------
# the plain forms

def _codes(W, group):
    """Codes (N, K) int16 and bf16 scales of an fp32 weight. A scale has 8 bits and a border between two codes at most 4,
    so their product is exact in 32 bits and no weight falls on the wrong side."""
    N, K = W.shape
    padded = torch.nn.functional.pad(W, (0, -K % group)).view(N, -1, group)
    scales = padded.abs().amax(2)
    scales = (scales / torch.full_like(scales, 6.0)).bfloat16()  # (by a number, torch multiplies by its rounded inverse)
    t, a = scales.float()[:, :, None], padded.abs()
    # ties go to the code whose last bit is zero
    c = ((a > 0.25 * t).short() + (a >= 0.75 * t).short() + (a > 1.25 * t).short() + (a >= 1.75 * t).short()
         + (a > 2.5 * t).short() + (a >= 3.5 * t).short() + (a > 5.0 * t).short())
    c = torch.where(t > 0, c, 0) + torch.where(padded < 0, 8, 0).short()
    return c.view(N, -1)[:, :K], scales


def _values(codes, scales, group):
    """(N, K) fp32 from codes below 16."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = table.index_select(0, codes.reshape(-1).int()).view(codes.shape)
    return v * scales.float().repeat_interleave(group, 1)[:, :codes.shape[1]]


def _plain_linear(s):
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], 2).flatten(1)
    W, z = _values(codes, s["scales"], s["group"]), s["x"].float()
    if s["norm"] is not None:
        z = z - z.mean(1, keepdim=True)
        z = z * ((z * z).mean(1, keepdim=True) + s["norm"].eps).rsqrt()
        z = z * s["norm"].weight.float() + s["norm"].bias.float()
    y = z @ W.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if s["resid"] is not None:
        y = y + s["resid"].float()
    return y.to(s["dtype"])


def _plain_pack(s):
    codes, scales = _codes(s["W"].float(), s["group"])
    return _values(codes, scales, s["group"]).to(s["W"].dtype)


def _plain_rules(s):
    x = s["logits"].float()
    (B, V), L = x.shape, s["history"].shape[1]
    at = torch.arange(L, device=DEV)[None, :]
    there, said = at < s["lengths"][:, None], at >= s["prompt"][:, None]
    seen = torch.zeros(B, V, device=DEV).scatter_add_(1, s["history"], there.float()) > 0
    times = torch.zeros(B, V, device=DEV).scatter_add_(1, s["history"], (there & said).float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - torch.where(times > 0, s["presence"][:, None], 0.0)
    x = x - s["frequency"][:, None] * times
    if s["ids"] is not None:
        x = x.scatter_add(1, s["ids"].clamp(min=0), torch.where(s["ids"] >= 0, s["values"], 0.0))
    if s["mask"] is not None:
        word = torch.arange(V, device=DEV)
        allowed = (s["mask"][s["state"].clamp(min=0)][:, word // 32] >> (word % 32)) & 1
        x = torch.where((allowed == 1) | (s["state"] < 0)[:, None], x, -math.inf)
    if not s["case"]["token"]:
        return x.to(s["logits"].dtype)
    best = x.amax(1, keepdim=True)
    token = torch.where(x == best, torch.arange(V, device=DEV), V).amin(1)
    return torch.where(best[:, 0] == -math.inf, -1, token)


def run(state):
    if own:
        return {"linear": _own_linear, "pack": _own_pack, "rules": _own_rules}[state["case"]["kind"]](state)
    return {"linear": _plain_linear, "pack": _plain_pack, "rules": _plain_rules}[state["case"]["kind"]](state)


def work(case):
    size = 2 if case["bf16"] else 4
    if case["kind"] == "rules":
        B, V, L, M, S = case["B"], case["V"], case["L"], case["M"], case["states"]
        words = (V + 31) // 32 * 4
        return {"bytes": B * V * size * (1 if case["token"] else 2) + 4 * B * (L + 1) + (12 * B * min(M, V)) + 36 * B
                + (min(B, S) * words if S else 0) + (8 * B if case["token"] else 0), "flops": B * V * 2}
    N, K = case["N"], case["K"]
    packed = N * K // 2 + 2 * N * -(-K // case["group"])
    if case["kind"] == "pack":
        return {"bytes": 2 * size * N * K + 2 * packed, "flops": 4 * N * K}
    n = case["n"]
    data = size * (n * (K + N) + (n * N if case["resid"] else 0) + (N if case["bias"] else 0)
                   + (2 * K if case["norm"] else 0))
    return {"bytes": packed + data, "flops": 2 * n * N * K}


# ------------------------------------------------------------------------------------------------------------------
# in 64 bits, from the definitions

def _exact_weight(W, group):
    """The nearest of the fifteen multiples of the group's scale, an equally near pair giving the even code."""
    N, K = W.shape
    out = torch.empty(N, K, dtype=torch.float64, device=DEV)
    grid = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
    rows = max(1, (1 << 23) // K)
    for a in range(0, N, rows):
        for b in range(0, K, group):
            w = W[a:a + rows, b:b + group].double()
            s = (w.abs().amax(1, keepdim=True) / 6).float().bfloat16().double()
            q = (w.abs() / s.where(s > 0, torch.ones_like(s))).clamp(max=6)
            up = torch.searchsorted(grid, q.contiguous()).clamp(1, 7)  # the first code not below
            lo, hi = grid[up - 1], grid[up]
            down, above = w.abs() - lo * s, hi * s - w.abs()
            pick = torch.where((down < above) | ((down == above) & (up % 2 == 1)), lo, hi)
            out[a:a + rows, b:b + group] = torch.copysign(pick * s, w) * (s > 0)
    return out


def exact(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "pack":
        return _exact_weight(_weight(case, g), case["group"])
    if case["kind"] == "linear":
        s, W = _linear_inputs(case, g)
        d = lambda t: None if t is None else t.double()  # noqa: E731
        x = d(s["x"])
        if s["norm"] is not None:
            x = torch.nn.functional.layer_norm(x, (case["K"],), d(s["norm"].weight), d(s["norm"].bias), s["norm"].eps)
        y = torch.nn.functional.linear(x, _exact_weight(W, case["group"]), d(s["bias"]))
        if case["gelu"]:
            y = torch.nn.functional.gelu(y)
        return y if s["resid"] is None else y + d(s["resid"])
    s = _rules_inputs(case, g)
    x = s["logits"].double()
    V, out = case["V"], []
    for b in range(case["B"]):
        row, h = x[b], s["history"][b, :s["lengths"][b]]
        count = torch.bincount(h[s["prompt"][b]:], minlength=V)
        here = torch.bincount(h, minlength=V) > 0
        row = torch.where(here, row * s["repetition"][b].double() ** -row.sign(), row)
        row = row - count.clamp(max=1) * s["presence"][b].double() - count * s["frequency"][b].double()
        if s["ids"] is not None:
            real = s["ids"][b] >= 0
            row[s["ids"][b][real]] += s["values"][b][real].double()
        if s["mask"] is not None and s["state"][b] >= 0:
            bits = s["mask"][s["state"][b]][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)
            row = row.masked_fill((bits & 1).flatten()[:V] == 0, -math.inf)
        out.append(row)
    x = torch.stack(out)
    if not case["token"]:
        return x
    top = x.amax(1, keepdim=True)
    word = torch.arange(V, device=DEV).where(x == top, V).amin(1)
    return word.where(top[:, 0] > -math.inf, torch.full_like(word, -1))
