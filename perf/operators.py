"""Sampled codes and codebook lookup, measured: scores, sample, lookup and lookup_gradient of vq_amd.Context.

Each case is one operator at one size.  With `own` false run() computes it with elementary torch operations; with `own`
true it makes the call a user of vq_amd makes.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

_context = None


def _handle():
    """The one context a program keeps for the calls that need no model."""
    global _context
    if _context is None:
        from vq_amd import Context

        _context = Context(0)
    return _context


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # Iris-shaped data against three prototypes: the smallest model there is, latency only
        {"name": "scores_tiny", "op": "scores", "n": 150, "d": 4, "k": 3},
        # a batch of 128-value rows against a codebook of 256
        {"name": "scores_codebook", "op": "scores", "n": 500_000, "d": 128, "k": 256},
        # image rows of 784 values against 1000 prototypes, an odd number of rows
        {"name": "scores_long_rows", "op": "scores", "n": 20_011, "d": 784, "k": 1000},
        # one token for one request, a large vocabulary in 16 bits, the usual filters
        {"name": "sample_one", "op": "sample", "n": 1, "v": 131_072, "dtype": "bf16", "params": "topk_topp"},
        # a batch of requests, each with parameters of its own, masked tokens, an odd vocabulary
        {"name": "sample_mixed", "op": "sample", "n": 61, "v": 49_999, "dtype": "f32", "params": "rows"},
        # a large batch over a large vocabulary, nucleus only
        {"name": "sample_nucleus", "op": "sample", "n": 256, "v": 131_072, "dtype": "bf16", "params": "topp"},
        # codes drawn for many vectors from the scores of a small codebook
        {"name": "sample_codes", "op": "sample", "n": 400_000, "v": 256, "dtype": "f32", "params": "topp"},
        # one step of serving: the embeddings of a few tokens
        {"name": "lookup_step", "op": "lookup", "n": 16, "d": 4096, "k": 131_072, "dtype": "bf16"},
        # decoding a large batch of codes
        {"name": "lookup_decode", "op": "lookup", "n": 2_000_000, "d": 128, "k": 256, "dtype": "f32"},
        # the gradient of a token embedding, most tokens absent, some very frequent
        {"name": "gradient_tokens", "op": "gradient", "n": 16_384, "d": 4096, "k": 65_536, "dtype": "bf16", "out": "f32"},
        # sums and counts of a codebook's vectors: few bins, many rows
        {"name": "gradient_codebook", "op": "gradient", "n": 2_000_000, "d": 128, "k": 256, "dtype": "f32", "out": "f32"},
        # odd sizes, padded positions
        {"name": "gradient_ragged", "op": "gradient", "n": 3001, "d": 515, "k": 997, "dtype": "f16", "out": "f16"},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["scores", "sample", "lookup", "gradient"])
    if op == "scores":
        while True:
            n, d, k = log(1, 500_000), log(2, 1000), log(2, 4096)
            if n * d * k <= 500_000 * 128 * 256 and n * k <= 128_000_000:
                return {"op": op, "n": n, "d": d, "k": k}
    if op == "sample":
        while True:
            n, v = log(1, 400_000), log(2, 131_072)
            if n * v <= 256 * 131_072:
                return {"op": op, "n": n, "v": v, "dtype": rng.choice(list(TYPES)), "params": rng.choice(["plain", "topk", "topp", "minp", "topk_topp", "rows"])}
    if op == "lookup":
        while True:
            n, d, k = log(1, 2_000_000), log(2, 8192), log(2, 131_072)
            if n * d <= 256_000_000 and k * d <= 536_870_912:
                return {"op": op, "n": n, "d": d, "k": k, "dtype": rng.choice(list(TYPES))}
    while True:
        n, d, k = log(1, 2_000_000), log(2, 8192), log(2, 131_072)
        if n * d <= 256_000_000 and k * d <= 268_435_456:
            dtype = rng.choice(list(TYPES))
            return {"op": op, "n": n, "d": d, "k": k, "dtype": dtype, "out": rng.choice(["f32", dtype])}


# ------------------------------------------------------------------------------------------------ inputs
def _tokens(n, k, g):
    """n tokens of k: half of them by a law that favours few (the frequent words, the crowded codes), half even, in a shuffled order of names."""
    a = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    zipf = (torch.exp(a * math.log(k + 1.0)) - 1.0).long().clamp_(0, k - 1)
    even = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * k).long().clamp_(0, k - 1)
    t = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, zipf, even)
    t = torch.randperm(k, generator=g, device="cuda")[t].int()
    return torch.where(torch.rand(n, generator=g, device="cuda") < 0.01, -1, t)      # one in a hundred is padding


def _params(case, g):
    n, kind = case["n"], case["params"]
    if kind == "rows":
        pick = torch.rand(n, generator=g, device="cuda")
        t = torch.rand(n, generator=g, device="cuda") * 1.5 + 0.25
        return {
            "temperature": torch.where(pick < 0.1, torch.zeros_like(t), t),
            "top_k": (torch.rand(n, generator=g, device="cuda") * 200).int() * (pick < 0.7).int(),
            "top_p": torch.where(pick < 0.3, torch.ones_like(t), 0.5 + 0.5 * torch.rand(n, generator=g, device="cuda")),
            "min_p": torch.where(pick > 0.8, 0.1 * torch.rand(n, generator=g, device="cuda"), torch.zeros_like(t)),
        }
    p = {"temperature": 0.8, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if "topk" in kind:
        p["top_k"] = 50
    if "topp" in kind:
        p["top_p"] = 0.9
    if kind == "minp":
        p["min_p"] = 0.05
    return p


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "scores":
        n, d, k = case["n"], case["d"], case["k"]
        w = torch.rand(k, d, generator=g, device="cuda") * 2 - 1
        x = w[torch.randint(k, (n,), generator=g, device="cuda")] + 0.5 * (torch.rand(n, d, generator=g, device="cuda") * 2 - 1)
        state = {"op": op, "x": x, "w": w}
        if own:
            from vq_amd import Context

            state["ctx"] = Context(0)
            state["ctx"].set_prototypes(w.cpu().numpy())
        return state
    if op == "sample":
        n, v = case["n"], case["v"]
        scores = torch.randn(n, v, generator=g, device="cuda") * 2.5
        scores[:, :: max(1, v // 40)] += 6.0 * torch.rand(n, -(-v // max(1, v // 40)), generator=g, device="cuda")
        if v > 100:
            scores[:, 7:: 50] = -math.inf                                            # masked tokens
        return {"op": op, "scores": scores.to(TYPES[case["dtype"]]), "u": torch.rand(n, generator=g, device="cuda"), **_params(case, g)}
    n, d, k = case["n"], case["d"], case["k"]
    dtype = TYPES[case["dtype"]]
    state = {"op": op, "idx": _tokens(n, k, g), "scale": float(np.float32(math.sqrt(d)))}
    if op == "lookup":
        state["table"] = torch.empty(k, d, dtype=dtype, device="cuda").normal_(0.0, 0.02, generator=g)
    else:
        state.update(grad=torch.empty(n, d, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g), k=k, out=TYPES[case["out"]])
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _calls(state)
    op = state["op"]
    if op == "scores":
        return _plain_scores(state["x"], state["w"])
    if op == "sample":
        return _plain_sample(state)
    if op == "lookup":
        return _plain_lookup(state["table"], state["idx"], state["scale"])
    return _plain_gradient(state["grad"], state["idx"], state["k"], state["scale"], state["out"])


def _calls(state):
    op = state["op"]
    if op == "scores":
        return state["ctx"].scores(state["x"])
    ctx = _handle()
    if op == "sample":
        return ctx.sample(state["scores"], state["u"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    if op == "lookup":
        return ctx.lookup(state["idx"], table=state["table"], scale=state["scale"])
    return ctx.lookup_gradient(state["grad"], state["idx"], K=state["k"], scale=state["scale"], out_dtype=state["out"], want_counts=True)


def _plain_scores(x, w):
    s = x @ w.t()
    s.mul_(2.0).sub_((x * x).sum(1, keepdim=True)).sub_((w * w).sum(1))
    return s.clamp_(max=0.0)


def _column(v, n, dtype):
    """A parameter as one 32-bit value per row (what the call takes), widened."""
    if isinstance(v, torch.Tensor):
        return v.to(dtype)[:, None]
    return torch.full((n, 1), v, device="cuda", dtype=torch.float32 if dtype == torch.float64 else torch.int32).to(dtype)


def _plain_sample(state):
    n, v = state["scores"].shape
    t, p, m = (_column(state[name], n, torch.float64) for name in ("temperature", "top_p", "min_p"))
    k = _column(state["top_k"], n, torch.int64)
    k = torch.where(k == 0, v, k)
    logits = torch.nan_to_num(state["scores"].double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    top = logits.amax(1, keepdim=True)
    w = torch.where(logits == top, 0.0, (logits - top) / torch.where(t > 0, t, 1.0)).exp_()
    w.masked_fill_(top == -math.inf, 0.0)
    order = logits.sort(dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    place = torch.arange(v, device="cuda")
    kept = place < torch.where(t > 0, k, 1)                                          # no temperature: the first maximum
    mass = (ranked * kept).cumsum(1)
    before = torch.cat([torch.zeros_like(t), mass[:, :-1]], 1)
    kept &= (before < p * mass[:, -1:]) | (p >= 1.0) | (place == 0)
    kept &= ranked >= m
    w *= torch.zeros_like(kept).scatter_(1, order, kept)                             # back in the order of the tokens
    mass = w.cumsum(1)
    total = mass[:, -1:]
    idx = (mass <= state["u"].double()[:, None] * total).sum(1, keepdim=True)
    last = (torch.where(w > 0, place, 0)).amax(1, keepdim=True)                      # the rounding of u times the total stays inside
    idx = torch.minimum(idx, last)
    prob = torch.where(total > 0, w.gather(1, idx) / total, 0.0)
    return idx[:, 0].int(), prob[:, 0].float()


def _plain_lookup(table, idx, scale):
    ok = (idx >= 0) & (idx < table.shape[0])
    rows = table[torch.where(ok, idx, 0)].float() * scale
    return torch.where(ok[:, None], rows, 0.0).to(table.dtype)


def _plain_gradient(grad, idx, k, scale, out):
    to = torch.where((idx >= 0) & (idx < k), idx, k)
    sums = torch.zeros(k + 1, grad.shape[1], device="cuda").index_add_(0, to, grad.float())
    counts = torch.zeros(k + 1, device="cuda", dtype=torch.int32).index_add_(0, to, torch.ones_like(to))
    return (sums[:k] * scale).to(out), counts[:k]


# ------------------------------------------------------------------------------------------------ the least a pass can do
def work(case):
    op, n = case["op"], case["n"]
    if op == "scores":
        d, k = case["d"], case["k"]
        return {"bytes": 4 * (n * d + k * d + n * k), "flops": 3 * n * k * d}
    size = TYPES[case["dtype"]].itemsize
    if op == "sample":
        v = case["v"]
        return {"bytes": n * v * size + n * (28 if case["params"] == "rows" else 12), "flops": 2 * n * v}
    d, k = case["d"], case["k"]
    if op == "lookup":
        return {"bytes": n * d * size + min(n, k) * d * size + 4 * n, "flops": n * d}
    return {"bytes": n * d * size + 4 * n + k * d * TYPES[case["out"]].itemsize + 4 * k, "flops": n * d}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "scores":
        x, w = state["x"].double(), state["w"].double()
        out = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
        step = max(1, 100_000_000 // (case["d"] * case["k"]))
        for at in range(0, case["n"], step):
            out[at:at + step] = -(x[at:at + step, None, :] - w).square_().sum(2)
        return out
    if op == "sample":
        return None, _exact_prob(state)
    if op == "lookup":
        table, idx = state["table"].double(), state["idx"].long()
        inside = (idx >= 0) & (idx < case["k"])
        out = torch.zeros(case["n"], case["d"], dtype=torch.float64, device="cuda")
        out[inside] = table.index_select(0, idx[inside]) * state["scale"]
        return out
    idx = state["idx"].long()
    rows = torch.nonzero((idx >= 0) & (idx < case["k"]))[:, 0]
    sums = torch.zeros(case["k"], case["d"], dtype=torch.float64, device="cuda")
    for part in rows.split(max(1, 100_000_000 // case["d"])):
        sums.index_put_((idx[part],), state["grad"][part].double(), accumulate=True)
    return sums * state["scale"], None


def _exact_prob(state):
    """The probability of the drawn token, row by row of the definition: ranks by counting up from the least, sums from the tail."""
    scores = state["scores"]
    n, v = scores.shape
    step = max(1, 8_000_000 // v)
    prob = torch.zeros(n, dtype=torch.float64, device="cuda")
    value = lambda name, a, b: (state[name][a:b].double() if isinstance(state[name], torch.Tensor) else torch.full((b - a,), float(np.float32(state[name])), dtype=torch.float64, device="cuda"))
    for a in range(0, n, step):
        b = min(n, a + step)
        x = scores[a:b].double()
        t, k, p, m = (value(name, a, b).unsqueeze(1) for name in ("temperature", "top_k", "top_p", "min_p"))
        best = x.max(1, keepdim=True).values
        greedy = t == 0
        w = torch.exp((x - best) / torch.where(greedy, torch.ones_like(t), t))
        back = torch.flip(x, [1]).sort(dim=1, stable=True).indices                   # ascending, the later of equals first
        back = v - 1 - back
        rank = torch.empty_like(back).scatter_(1, back, (v - 1 - torch.arange(v, device="cuda")).expand_as(back))
        first = torch.where(k == 0, torch.full_like(k, v), k)
        w1 = torch.where(rank < first, w, 0.0)
        z1 = w1.sum(1, keepdim=True)
        down = w1.gather(1, back)                                                    # least first: the mass before a place is the rest
        upto = z1 - down.cumsum(1)
        before = torch.empty_like(upto).scatter_(1, back, upto)
        keep = (rank < first) & ((before < p * z1) | (p >= 1) | (rank == 0)) & (w >= m)
        w2 = torch.where(keep, w, 0.0)
        z = w2.sum(1, keepdim=True)
        at = torch.searchsorted(w2.cumsum(1), state["u"][a:b].double().unsqueeze(1) * z, right=True).clamp_(max=v - 1)
        prob[a:b] = torch.where(greedy, torch.ones_like(z), w2.gather(1, at) / z)[:, 0]
    return prob
