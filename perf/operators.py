"""Decoding over the key / value cache beyond one greedy token: the operators' work as cases that can be
timed and compared, each with its plain form.

  tree     attention of drafted tokens over a cache (attention.decode_tree)
  weights  the attention weight each key has drawn, summed up (attention.add_key_weights)
  evict    a cache cut to a budget of rows by that weight (cache.evict)
  beam     a beam search step's choice over beams and vocabulary (ops.beam_select)
  reorder  the beams' key / value states put in the chosen order (cache.reorder)

Shapes are Gemma 4 E2B's (8 query heads on one KV head, head_dim 256 with a 512-key window or 512 without
one, vocabulary 262144, the 3658-token prompt) and generic grouped-query ones of head_dim 128.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # a sliding layer's attention over a small drafted tree: the smallest call, 28 of 35 layers
        {"name": "tree_sliding_n8", "kind": "tree", "h": 8, "kv": 1, "d": 256, "past": 700, "m": 8, "n": 8, "window": 512},
        # a full-attention layer verifying 16 drafted tokens after the 3658-token prompt
        {"name": "tree_full_n16_t3658", "kind": "tree", "h": 8, "kv": 1, "d": 512, "past": 3658, "m": 16, "n": 16,
         "window": 0},
        # a wide tree over a long conversation: as much product as traffic
        {"name": "tree_full_n64_t32k", "kind": "tree", "h": 8, "kv": 1, "d": 512, "past": 32749, "m": 64, "n": 64,
         "window": 0},
        # one more level of a drafted tree (33 of its 50 tokens), eight KV heads, a very long cache
        {"name": "tree_gqa_n33_t64k", "kind": "tree", "h": 32, "kv": 8, "d": 128, "past": 65521, "m": 50, "n": 33,
         "window": 0},
        # what one decoded token adds to the keys' weights
        {"name": "weights_token_t8191", "kind": "weights", "h": 8, "kv": 1, "d": 512, "start": 8190, "t": 1, "window": 0},
        # what the whole prompt adds
        {"name": "weights_prompt_t3658", "kind": "weights", "h": 8, "kv": 1, "d": 512, "start": 0, "t": 3658, "window": 0},
        # the steady state of a bounded cache: one token in, one row out
        {"name": "evict_step_4096", "kind": "evict", "kv": 1, "d": 512, "rows": 4097, "budget": 4096, "recent": 1024},
        # a long prompt's cache cut to a quarter
        {"name": "evict_prompt_64k", "kind": "evict", "kv": 8, "d": 128, "rows": 65521, "budget": 16384, "recent": 2048},
        # one request with four beams, the LM head's bf16 logits
        {"name": "beam_nb4_bf16", "kind": "beam", "batch": 1, "nb": 4, "vocab": 262144, "k": 8, "dtype": "bf16"},
        # a batch of requests, softcapped fp32 logits
        {"name": "beam_b8_nb8_fp32", "kind": "beam", "batch": 8, "nb": 8, "vocab": 262144, "k": 16, "dtype": "fp32"},
        # a sliding layer's cache of four beams
        {"name": "reorder_nb4_t511", "kind": "reorder", "nb": 4, "kv": 1, "d": 256, "t": 511, "layers": 1},
        # the caches of four full-attention layers, eight beams with long contexts
        {"name": "reorder_nb8_t8191", "kind": "reorder", "nb": 8, "kv": 1, "d": 512, "t": 8191, "layers": 4},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng, kind):
    kv, g = rng.choice([(1, 8), (1, 8), (1, 1), (2, 4), (4, 3), (8, 4), (5, 1), (1, 16)])
    d = rng.choice([128, 256, 512])
    if kind == "tree":
        n = _log(rng, 1, 64)
        return {"kind": kind, "h": kv * g, "kv": kv, "d": d, "past": _log(rng, 1, 65536), "m": n + rng.choice([0, 0, rng.randint(1, 40)]),
                "n": n, "window": rng.choice([0, 0, 512, rng.randint(1, 4096)])}
    if kind == "weights":
        t = rng.choice([1, _log(rng, 1, 3658)])
        return {"kind": kind, "h": kv * g, "kv": kv, "d": d, "start": rng.choice([0, _log(rng, 1, 8191)]), "t": t,
                "window": rng.choice([0, 0, 512, rng.randint(1, 2048)])}
    if kind == "evict":
        rows = _log(rng, 16, 65521)
        budget = rng.choice([rows - 1, _log(rng, 1, rows)])
        return {"kind": kind, "kv": kv, "d": d, "rows": rows, "budget": budget, "recent": rng.randint(0, budget)}
    if kind == "beam":
        return {"kind": kind, "batch": _log(rng, 1, 8), "nb": rng.randint(1, 8), "vocab": _log(rng, 100, 262144),
                "k": rng.randint(1, 32), "dtype": rng.choice(["bf16", "fp32"])}
    return {"kind": kind, "nb": rng.randint(2, 16), "kv": kv, "d": d, "t": _log(rng, 1, 8191), "layers": _log(rng, 1, 8)}


def draw(rng):
    kind = rng.choice(["tree", "tree", "weights", "evict", "beam", "reorder"])
    most = [work(c) for c in listed() if c["kind"] == kind]
    while True:
        case = _draw(rng, kind)
        w = work(case)
        if all(w[x] <= max(m[x] for m in most) for x in ("bytes", "flops")):
            return case


# ---- inputs ------------------------------------------------------------------------------


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _parents(m, seed):
    """A drafted tree: each token hangs on one of the eight before it, or on the context's last token."""
    g = torch.Generator().manual_seed(seed)
    at = torch.arange(m)
    back = (torch.rand(m, generator=g) * torch.clamp(at + 1, max=8)).long()
    return (at - 1 - back).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 7)
    kind = case["kind"]
    if kind == "tree":
        rows = case["past"] + case["m"]
        # scores of standard deviation 2, as normed queries and keys give them
        return {**case, "q": (_randn(g, case["h"], case["n"], case["d"]) * (2 * case["d"] ** -0.5)).bfloat16(),
                "k": _randn(g, case["kv"], rows, case["d"]).bfloat16(),
                "v": _randn(g, case["kv"], rows, case["d"]).bfloat16(),
                "parents": _parents(case["m"], int(seed)).to(DEV)}
    if kind == "weights":
        rows = case["start"] + case["t"]
        s = {**case, "q": (_randn(g, case["h"], case["t"], case["d"]) * (2 * case["d"] ** -0.5)).bfloat16(),
             "k": _randn(g, case["kv"], rows, case["d"]).bfloat16(),
             # what earlier calls summed up
             "weights": torch.rand(case["kv"], rows, generator=g, device=DEV).square()}
        # the attention call before it returns the logsumexp of its scores
        s["lse"] = torch.stack([torch.logsumexp(_scores(s, h, torch.float32), dim=1) for h in range(case["h"])])
        return s
    if kind == "evict":
        w = torch.exp(2.0 * _randn(g, case["kv"], case["rows"]))
        # one row in eight has drawn nothing that fp32 holds
        w = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.125, torch.zeros_like(w), w)
        return {**case, "k": _randn(g, case["kv"], case["rows"], case["d"]).bfloat16(),
                "v": _randn(g, case["kv"], case["rows"], case["d"]).bfloat16(), "weights": w,
                "positions": torch.arange(case["rows"], device=DEV, dtype=torch.int32).repeat(case["kv"], 1)}
    if kind == "beam":
        x = 30.0 * torch.tanh(_randn(g, case["batch"], case["nb"], case["vocab"]) * 0.1)
        scores = -20.0 * torch.rand(case["batch"], case["nb"], generator=g, device=DEV)
        return {**case, "logits": x.bfloat16() if case["dtype"] == "bf16" else x, "scores": scores}
    shape = (case["nb"], case["kv"], case["t"] + 33, case["d"])  # room for the tokens to come
    return {**case, "states": [_randn(g, *shape).bfloat16() for _ in range(2 * case["layers"])],
            "index": torch.randint(0, case["nb"], (case["nb"],), generator=g, device=DEV)}


# ---- plain forms ---------------------------------------------------------------------------


def _scores(s, h, dtype):
    """One head's masked scores [t, rows] of a weights case."""
    k = s["k"][h // (s["h"] // s["kv"])]
    x = s["q"][h].to(dtype) @ k.to(dtype).t().contiguous()
    p = torch.arange(s["start"], s["start"] + s["t"], device=x.device)[:, None]
    j = torch.arange(k.shape[0], device=x.device)[None]
    seen = (j <= p) if s["window"] == 0 else (j <= p) & (p - j < s["window"])
    return x.masked_fill(~seen, -math.inf)


def _tree(s):
    past, m, n, kv = s["past"], s["m"], s["n"], s["kv"]
    at = torch.arange(m, device=DEV)
    parents = s["parents"].long()
    # reach[i, j]: j is i or above it in the tree, by doubling the length of the chains
    reach = (at[:, None] == at[None]) | (parents[:, None] == at[None])
    reach = reach.float()
    for _ in range(max(1, (m - 1).bit_length())):
        reach = (reach @ reach).clamp(max=1.0)
    depth = reach.sum(1).long() - 1
    pos = torch.cat([torch.arange(past, device=DEV), past + depth])
    own_pos = pos[past + m - n:, None]
    seen = torch.cat([torch.ones(n, past, device=DEV, dtype=torch.bool), reach[m - n:] > 0], 1)
    if s["window"]:
        seen = seen & (own_pos - pos[None] < s["window"])
    q = s["q"].float().view(kv, s["h"] // kv, n, s["d"]).reshape(kv, -1, s["d"])
    x = (q @ s["k"].float().transpose(1, 2).contiguous()).view(kv, -1, n, past + m)
    x = x.masked_fill(~seen, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = x.view(kv, -1, past + m) @ s["v"].float()
    return (o / x.sum(-1).view(kv, -1, 1)).view(s["h"], n, s["d"]).bfloat16()


def _weights(s):
    g = s["h"] // s["kv"]
    k = s["k"].float().transpose(1, 2).contiguous()
    x = (s["q"].float().view(s["kv"], g * s["t"], s["d"]) @ k).view(s["kv"], g, s["t"], -1)
    p = torch.arange(s["start"], s["start"] + s["t"], device=DEV)[:, None]
    j = torch.arange(k.shape[2], device=DEV)[None]
    seen = (j <= p) if s["window"] == 0 else (j <= p) & (p - j < s["window"])
    x = torch.exp(x - s["lse"].view(s["kv"], g, s["t"], 1)).masked_fill(~seen, 0.0)
    return s["weights"].add_(x.sum((1, 2)))


def _evict(s):
    n, budget = s["rows"], s["budget"]
    w, pos = s["weights"], s["positions"]
    fresh = pos > pos.amax(1, keepdim=True) - s["recent"]
    order = torch.sort(w, dim=1, descending=True, stable=True).indices
    order = order.gather(1, torch.sort(fresh.gather(1, order).int(), dim=1, descending=True, stable=True).indices)
    keep = torch.zeros_like(fresh).scatter(1, order[:, :budget], True)
    rows = torch.arange(n, device=DEV).expand_as(w)
    movers = torch.sort(torch.where(keep[:, budget:], rows[:, budget:], n), dim=1).values
    movers = torch.nn.functional.pad(movers, (0, budget), value=n)
    hole = ~keep[:, :budget]
    kept = torch.where(hole, movers.gather(1, (torch.cumsum(hole.long(), 1) - 1).clamp(min=0)), rows[:, :budget])
    at = kept[:, :, None].expand(-1, -1, s["d"])
    s["k"][:, :budget] = s["k"].gather(1, at)
    s["v"][:, :budget] = s["v"].gather(1, at)
    return [kept.int(), w.gather(1, kept), pos.gather(1, kept), s["k"][:, :budget], s["v"][:, :budget]]


def _beam(s):
    # in 64 bits: the choice lies between values that may differ in the last bits of 32
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True)) + s["scores"].double()[:, :, None]
    value, at = torch.sort(x.flatten(1), dim=1, descending=True, stable=True)
    value, at = value[:, : s["k"]], at[:, : s["k"]]
    return [value.float(), at // s["vocab"], at % s["vocab"]]


def _reorder(s):
    for t in s["states"]:
        live = t[:, :, : s["t"]]
        live.copy_(live[s["index"]])
    return [t[:, :, : s["t"]] for t in s["states"]]


def run(state):
    s = state
    if own:
        if "w8a8" not in sys.modules:
            sys.path.insert(0, os.path.join(os.getcwd(), "gemma-npu_amd"))
        from w8a8 import attention, cache, ops
        if s["kind"] == "tree":
            return attention.decode_tree(s["q"], s["k"], s["v"], s["parents"], s["past"], s["window"])
        if s["kind"] == "weights":
            return attention.add_key_weights(s["q"], s["k"], s["lse"], s["weights"], s["start"], s["window"])
        if s["kind"] == "evict":
            kept = cache.evict(s["k"], s["v"], s["weights"], s["positions"], s["rows"], s["budget"], s["recent"])
            return [*kept, s["k"][:, : s["budget"]], s["v"][:, : s["budget"]]]
        if s["kind"] == "beam":
            return list(ops.beam_select(s["logits"], s["scores"], s["k"]))
        live = [t[:, :, : s["t"]] for t in s["states"]]
        cache.reorder(live, s["index"])
        return live
    return {"tree": _tree, "weights": _weights, "evict": _evict, "beam": _beam, "reorder": _reorder}[s["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    if kind == "tree":
        seen = c["past"] + c["m"]
        if c["window"]:
            seen = min(seen, c["window"] + c["m"])
        qo = 2 * c["h"] * c["n"] * c["d"]
        return {"bytes": 2 * (2 * c["kv"] * seen * c["d"] + qo) + 4 * c["m"], "flops": 4 * c["h"] * c["n"] * seen * c["d"]}
    if kind == "weights":
        w = c["window"] or c["start"] + c["t"]
        pairs = sum(min(w, p + 1) for p in range(c["start"], c["start"] + c["t"]))
        keys = min(c["start"] + c["t"], w + c["t"])
        return {"bytes": 2 * (c["kv"] * keys * c["d"] + c["h"] * c["t"] * c["d"]) + 4 * c["h"] * c["t"] + 8 * c["kv"] * keys,
                "flops": 2 * c["h"] * pairs * c["d"]}
    if kind == "evict":
        tail = c["rows"] - c["budget"]
        fresh = min(c["recent"], c["rows"])
        rest = c["rows"] - fresh
        moved = min(fresh, tail) + (c["budget"] - fresh) * max(0, tail - fresh) / max(1, rest)
        return {"bytes": c["kv"] * (8 * c["rows"] + 12 * c["budget"] + moved * 8 * c["d"]), "flops": 0}
    if kind == "beam":
        n = c["batch"] * c["nb"] * c["vocab"]
        return {"bytes": n * (2 if c["dtype"] == "bf16" else 4) + 4 * c["batch"] * c["nb"] + 20 * c["batch"] * c["k"],
                "flops": 3 * n}
    nb = c["nb"]
    rows = nb - 1 + nb * (1 - (1 - 1 / nb) ** nb)  # moved ones written, distinct ones read, on average
    return {"bytes": rows * 2 * c["layers"] * c["kv"] * c["t"] * c["d"] * 2 + 8 * nb, "flops": 0}


# ---- the definitions in 64 bits -------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "tree":
        past, m, n = s["past"], s["m"], s["n"]
        up = s["parents"].tolist()
        chains = [[i] for i in range(m)]
        for i in range(m):
            if up[i] >= 0:
                chains[i] = chains[up[i]] + [i]
        out = torch.empty(s["h"], n, s["d"], device=DEV, dtype=torch.float64)
        for i in range(n):
            chain = chains[m - n + i]
            rows = torch.tensor(list(range(past)) + [past + c for c in chain], device=DEV)
            if s["window"]:
                rows = rows[max(0, len(rows) - s["window"]):]
            for g in range(s["kv"]):
                heads = slice(g * s["h"] // s["kv"], (g + 1) * s["h"] // s["kv"])
                p = torch.softmax(s["q"][heads, i].double() @ s["k"][g, rows].double().t(), dim=-1)
                out[heads, i] = p @ s["v"][g, rows].double()
        return out
    if kind == "weights":
        total = s["weights"].double()
        for h in range(s["h"]):
            total[h // (s["h"] // s["kv"])] += torch.exp(_scores(s, h, torch.float64) - s["lse"][h].double()[:, None]).sum(0)
        return total
    if kind == "evict":
        kept_all = []
        for g in range(s["kv"]):
            w, pos = s["weights"][g].tolist(), s["positions"][g].tolist()
            newest = max(pos)
            ranked = sorted(range(s["rows"]), key=lambda r: (pos[r] <= newest - s["recent"], -w[r] if pos[r] <= newest - s["recent"] else 0, r))
            chosen = set(ranked[: s["budget"]])
            spare = iter(sorted(r for r in chosen if r >= s["budget"]))
            kept_all.append([r if r in chosen else next(spare) for r in range(s["budget"])])
        kept = torch.tensor(kept_all, device=DEV)
        take = lambda t: torch.stack([t[g][kept[g]] for g in range(s["kv"])])  # noqa: E731
        return [kept.int(), take(s["weights"]).double(), take(s["positions"]), take(s["k"]).double(), take(s["v"]).double()]
    if kind == "beam":
        x = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[:, :, None]
        found = []
        for row in x.flatten(1):
            least = torch.topk(row, s["k"]).values[-1]
            at = torch.nonzero(row >= least)[:, 0].tolist()
            found.append(sorted(zip((-row[at]).tolist(), at))[: s["k"]])
        value = torch.tensor([[-v for v, _ in f] for f in found], device=DEV, dtype=torch.float64)
        at = torch.tensor([[a for _, a in f] for f in found], device=DEV)
        return [value, at // s["vocab"], at % s["vocab"]]
    return [torch.stack([t[i, :, : s["t"]] for i in s["index"].tolist()]).double() for t in s["states"]]
