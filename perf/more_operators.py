"""Long conversations with drafted tokens: the operators' work as cases that can be timed and compared, each
with its plain form.

  verify  drafted tokens tested against the target's probabilities, the next token drawn (ops.verify_drafts)
  sinks   attention with a sliding window and the first tokens visible (attention.sink_attention)
  store   keys and values put into an 8-bit cache with a scale per block of tokens and head, and read back
          (cache.append, cache.read)
  attend  attention over such a cache (attention.block_attention)

Shapes are Gemma 4 E2B's (8 query heads on one KV head, head_dim 256 with a 512-key window or 512 without
one, vocabulary 262144, the 3658-token prompt) and generic grouped-query ones of head_dim 128.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
BLOCK = 64  # tokens that share a scale


def listed():
    return [
        # one request, four tokens drafted by a small model: bf16 logits of both models
        {"name": "verify_chain4_bf16", "kind": "verify", "batch": 1, "n": 4, "vocab": 262144, "dtype": "bf16", "draft": "model",
         "temperature": 1.0},
        # a batch of requests with ragged drafts, softcapped fp32 logits
        {"name": "verify_b8_n8_fp32", "kind": "verify", "batch": 8, "n": 8, "vocab": 262144, "dtype": "fp32", "draft": "model",
         "temperature": 0.7},
        # a tree of drafted tokens, as attention.decode_tree attends to it
        {"name": "verify_tree48_bf16", "kind": "verify", "batch": 1, "n": 48, "vocab": 262144, "dtype": "bf16", "draft": "tree",
         "temperature": 1.0},
        # one decoded token in a sliding layer of a conversation long past its window
        {"name": "sinks_token_t8191", "kind": "sinks", "h": 8, "kv": 1, "d": 256, "start": 8190, "t": 1, "window": 1020, "sinks": 4},
        # a sliding layer over the whole prompt
        {"name": "sinks_prompt_t3658", "kind": "sinks", "h": 8, "kv": 1, "d": 256, "start": 0, "t": 3658, "window": 512, "sinks": 4},
        # one piece of a long prompt, eight KV heads, a wide window
        {"name": "sinks_chunk_t16k", "kind": "sinks", "h": 32, "kv": 8, "d": 128, "start": 14317, "t": 2048, "window": 4096,
         "sinks": 16},
        # the token that completes a block
        {"name": "store_token_t4096", "kind": "store", "kv": 1, "d": 512, "start": 4095, "t": 1, "codes": "int8"},
        # a long prompt's keys and values of eight KV heads
        {"name": "store_prompt_64k", "kind": "store", "kv": 8, "d": 128, "start": 0, "t": 65521, "codes": "int8"},
        # one decoded token after the 3658-token prompt, a full-attention layer: the smallest call
        {"name": "attend_token_t3659", "kind": "attend", "h": 8, "kv": 1, "d": 512, "rows": 3659, "n": 1, "window": 0, "sinks": 0,
         "codes": "int8"},
        # one decoded token, eight KV heads, a very long conversation
        {"name": "attend_token_t64k", "kind": "attend", "h": 32, "kv": 8, "d": 128, "rows": 65521, "n": 1, "window": 0, "sinks": 0,
         "codes": "int8"},
        # a run of five drafted tokens, e4m3 codes
        {"name": "attend_drafts5_t32k", "kind": "attend", "h": 8, "kv": 1, "d": 512, "rows": 32749, "n": 5, "window": 0, "sinks": 0,
         "codes": "e4m3"},
        # the user's next turn of 509 tokens, a window with sinks
        {"name": "attend_turn509_t8k", "kind": "attend", "h": 8, "kv": 1, "d": 256, "rows": 8191, "n": 509, "window": 4096,
         "sinks": 64, "codes": "int8"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng, kind):
    kv, g = rng.choice([(1, 8), (1, 8), (1, 1), (2, 4), (4, 3), (8, 4), (5, 1), (1, 16)])
    d = rng.choice([128, 256, 512])
    window = rng.choice([0, 512, rng.randint(1, 4096)])
    sinks = rng.choice([0, 4, _log(rng, 1, 256)])
    if kind == "verify":
        draft = rng.choice(["model", "model", "certain", "tree"])
        return {"kind": kind, "batch": 1 if draft == "tree" else _log(rng, 1, 8), "n": rng.randint(1, 48 if draft == "tree" else 8),
                "vocab": _log(rng, 100, 262144), "dtype": rng.choice(["bf16", "fp32"]), "draft": draft,
                "temperature": rng.choice([0.7, 1.0, 1.3])}
    if kind == "sinks":
        return {"kind": kind, "h": kv * g, "kv": kv, "d": d, "start": rng.choice([0, _log(rng, 1, 16384)]),
                "t": rng.choice([1, rng.randint(2, 8), _log(rng, 1, 3658)]), "window": window, "sinks": sinks}
    if kind == "store":
        return {"kind": kind, "kv": kv, "d": d, "start": rng.choice([0, _log(rng, 1, 8191)]), "t": rng.choice([1, _log(rng, 1, 65521)]),
                "codes": rng.choice(["int8", "e4m3"])}
    n = rng.choice([1, rng.randint(2, 8), _log(rng, 1, 512)])
    return {"kind": kind, "h": kv * g, "kv": kv, "d": d, "rows": n + _log(rng, 1, 65521), "n": n, "window": window, "sinks": sinks,
            "codes": rng.choice(["int8", "e4m3"])}


def draw(rng):
    kind = rng.choice(["verify", "sinks", "store", "attend", "attend"])
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


def _sample(g, logits):
    """A token of each row's distribution."""
    u = torch.rand(logits.shape, generator=g, device=DEV).clamp_(min=1e-20)
    return (logits.float() - torch.log(-torch.log(u))).argmax(-1)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma-npu_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import w8a8
    return w8a8


def _code_type(name):
    return torch.int8 if name == "int8" else torch.float8_e4m3fn


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 11)
    kind = case["kind"]
    if kind == "verify":
        b, n, v = case["batch"], case["n"], case["vocab"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        logits = (30.0 * torch.tanh(_randn(g, b, n + 1, v) * 0.1)).to(dt)
        s = {**case, "logits": logits, "uniforms": torch.rand(b, n + 1, generator=g, device=DEV), "draft_logits": None,
             "parents": None, "lengths": None}
        if case["draft"] == "tree":
            s["parents"] = _parents(n, int(seed)).to(DEV)
            s["tokens"] = _sample(g, logits[:, s["parents"].long() + 1])
        else:
            near = (logits[:, :n].float() + 0.6 * _randn(g, b, n, v)).to(dt)  # a smaller model's logits of the same tokens
            s["tokens"] = _sample(g, near.float() / case["temperature"])
            if case["draft"] == "model":
                s["draft_logits"] = near
            if b > 1:
                s["lengths"] = torch.randint(0, n + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
        return s
    d, kv = case["d"], case["kv"]
    if kind == "store":
        rows = case["start"] + case["t"]
        k, v = _randn(g, kv, rows, d).bfloat16(), _randn(g, kv, rows, d).bfloat16()
        s = {**case, "k": k, "v": v}
        if own:
            cache = _package().cache
            s["cache"] = cache.BlockCache(kv, rows, d, _code_type(case["codes"]))
            if case["start"]:
                cache.append(s["cache"], k[:, : case["start"]], v[:, : case["start"]], 0)
        return s
    n, rows = (case["n"], case["rows"]) if kind == "attend" else (case["t"], case["start"] + case["t"])
    # scores of standard deviation 2, as normed queries and keys give them
    q = (_randn(g, case["h"], n, d) * (2 * d ** -0.5)).bfloat16()
    k, v = _randn(g, kv, rows, d).bfloat16(), _randn(g, kv, rows, d).bfloat16()
    if kind == "sinks":
        return {**case, "q": q, "k": k, "v": v}
    s = {**case, "q": q}
    if own:
        cache = _package().cache
        s["cache"] = cache.BlockCache(kv, rows, d, _code_type(case["codes"]))
        cache.append(s["cache"], k, v, 0)
    else:
        s["plain"] = [_stored(x, case["codes"]) for x in (k, v)]
    return s


# ---- plain forms ---------------------------------------------------------------------------


def _codes(x, codes):
    """Whole blocks [KV, blocks, 64, D] in fp32 -> their codes and scales."""
    s = x.abs().amax((2, 3), keepdim=True).clamp(min=1e-8) / (127.0 if codes == "int8" else 448.0)
    if codes == "int8":
        return torch.round(x / s).clamp(-127, 127).to(torch.int8), s
    return (x / s).to(torch.float8_e4m3fn), s


def _stored(x, codes):
    """Rows [KV, n, D] as the cache holds them: codes and scales of the whole blocks, the others in bf16."""
    full = x.shape[1] // BLOCK * BLOCK
    c, s = _codes(x[:, :full].float().view(x.shape[0], -1, BLOCK, x.shape[2]), codes)
    return c, s, x[:, full:]


def _values(stored):
    """What stored rows stand for, fp32 [KV, n, D]."""
    c, s, rest = stored
    return torch.cat([(c.float() * s).flatten(1, 2), rest.float()], 1)


def _seen(p, j, window, sinks):
    return (j <= p) if window == 0 else (j <= p) & ((p - j < window) | (j < sinks))


def _attention(q, k, v, start, window, sinks):
    """Masked attention in fp32, one KV head at a time: q [H, T, D], k / v [KV, n, D]."""
    h, t, d = q.shape
    kv, n = k.shape[:2]
    p = torch.arange(start, start + t, device=DEV)[:, None]
    seen = _seen(p, torch.arange(n, device=DEV)[None], window, sinks)
    out = []
    for i in range(kv):
        x = (q.view(kv, h // kv, t, d)[i].reshape(-1, d).float() @ k[i].float().t().contiguous()).view(h // kv, t, n)
        x = x.masked_fill(~seen, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        out.append((x.view(-1, n) @ v[i].float()) / x.sum(-1).view(-1, 1))
    return torch.stack(out).view(h, t, d).bfloat16()


def _softmax(x, temperature):
    x = x.double() / temperature
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return x / x.sum(-1, keepdim=True)


def _draw_token(r, p, u):
    """The first token of each row [B, V] whose running sum passes u of the whole."""
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, p)
    c = r.cumsum(-1)
    return (c > u[:, None].double() * c[:, -1:]).int().argmax(-1)


def _verify(s):
    b, n, t = s["batch"], s["n"], s["temperature"]
    tokens, u = s["tokens"], s["uniforms"].double()
    p = _softmax(s["logits"], t)
    if s["draft"] == "tree":
        parents = s["parents"].long()
        pt = p[0, parents + 1, tokens[0]]
        at = torch.full((1,), -1, device=DEV)
        gone = torch.zeros(1, device=DEV, dtype=torch.float64)
        refused = torch.zeros(n, device=DEV, dtype=torch.bool)
        path = torch.full((n,), -1, device=DEV)
        count = torch.zeros(1, device=DEV, dtype=torch.int64)
        index = torch.arange(n, device=DEV)
        for m in range(n):
            child = parents[m] == at
            again = (refused & (tokens[0] == tokens[0, m])).any()  # a refused sibling's token has nothing left
            pm = torch.where(again, torch.zeros_like(gone), pt[m])
            ok = child & (u[0, m] * (1.0 - gone) < pm)
            gone = torch.where(ok, torch.zeros_like(gone), torch.where(child, gone + pm, gone))
            refused = torch.where(ok, torch.zeros_like(refused), refused | ((index == m) & child))
            path = torch.where(ok & (index == count), m, path)
            count = count + ok
            at = torch.where(ok, m, at)
        last = p[0].index_select(0, at + 1)
        kill = torch.zeros_like(last).index_put_((torch.zeros_like(index), tokens[0]), refused.double(), accumulate=True)
        nxt = _draw_token(torch.where(kill > 0, torch.zeros_like(last), last), last, u[:, n])
        return [count.int(), path[None], nxt]
    if s["draft_logits"] is None:
        q = torch.zeros(b, n, p.shape[2], device=DEV, dtype=torch.float64).scatter_(2, tokens[:, :, None], 1.0)
    else:
        q = _softmax(s["draft_logits"], t)
    index = torch.arange(n, device=DEV)[None]
    length = torch.full((b,), n, device=DEV) if s["lengths"] is None else s["lengths"].long()
    ok = u[:, :n] * q.gather(2, tokens[:, :, None])[..., 0] < p[:, :n].gather(2, tokens[:, :, None])[..., 0]
    count = (ok & (index < length[:, None])).long().cumprod(1).sum(1)
    rows = torch.arange(b, device=DEV)
    last = p[rows, count]
    drafted = torch.where((count < length)[:, None], q[rows, count.clamp(max=n - 1)], torch.zeros_like(last))
    nxt = _draw_token((last - drafted).clamp(min=0), last, u[:, n])
    path = torch.where(index < count[:, None], index, torch.full_like(index, -1))
    return [count.int(), path, nxt]


def run(s):
    kind = s["kind"]
    if kind == "verify":
        if not own:
            return _verify(s)
        return list(_package().ops.verify_drafts(s["logits"], s["tokens"], s["uniforms"], s["draft_logits"], s["parents"], s["lengths"],
                                                 s["temperature"]))
    if kind == "sinks":
        if own:
            return _package().attention.sink_attention(s["q"], s["k"], s["v"], s["start"], s["window"], s["sinks"])
        return _attention(s["q"], s["k"], s["v"], s["start"], s["window"], s["sinks"])
    if kind == "store":
        # the new rows, read back from the first block that they lie in
        start, first = s["start"], s["start"] // BLOCK * BLOCK
        if own:
            cache = _package().cache
            # a cache that went on further than a block takes rows back to a whole block only, so a pass over the same
            # state puts its first block's old rows in again there
            at = start if (start + s["t"] - 1) // BLOCK - start // BLOCK <= 1 else first
            cache.append(s["cache"], s["k"][:, at:], s["v"][:, at:], at)
            return list(cache.read(s["cache"], first, start + s["t"]))
        return [_values(_stored(x[:, first:], s["codes"])).bfloat16() for x in (s["k"], s["v"])]
    if own:
        return _package().attention.block_attention(s["q"], s["cache"], s["rows"], s["window"], s["sinks"])
    k, v = (_values(x) for x in s["plain"])
    return _attention(s["q"], k, v, s["rows"] - s["n"], s["window"], s["sinks"])


# ---- the least work -----------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "verify":
        rows = case["batch"] * (case["n"] + 1 + (case["n"] if case["draft"] == "model" else 0))
        values = rows * case["vocab"]
        return {"bytes": values * (2 if case["dtype"] == "bf16" else 4) + 16 * case["batch"] * (case["n"] + 1), "flops": 4 * values}
    if kind == "store":
        first = case["start"] // BLOCK * BLOCK
        new, back = 2 * case["kv"] * case["d"] * case["t"], 2 * case["kv"] * case["d"] * (case["start"] + case["t"] - first)
        # the new rows read, their codes written and read again, and what they stand for written
        return {"bytes": 3 * new + 3 * back, "flops": 4 * new + back}
    t, start = (case["n"], case["rows"] - case["n"]) if kind == "attend" else (case["t"], case["start"])
    rows, w, first = start + t, case["window"], case["sinks"]
    pairs = 0
    if w == 0:
        pairs, union = t * start + t * (t + 1) // 2, rows
    else:
        for p in range(start, rows):
            near = min(p + 1, w)
            pairs += near + min(first, p + 1 - near)
        oldest = max(0, start + 1 - w)
        union = rows - oldest + min(first, oldest)
    width = 2 if kind == "sinks" else 1
    return {"bytes": 2 * union * case["kv"] * case["d"] * width + 4 * case["h"] * t * case["d"],
            "flops": 4 * case["h"] * case["d"] * pairs}


# ---- in 64 bits ---------------------------------------------------------------------------


def _exact_attention(q, k, v, start, window, sinks):
    out = torch.empty(q.shape, device=DEV, dtype=torch.float64)
    per = q.shape[0] // k.shape[0]
    for h in range(q.shape[0]):
        keys, values = k[h // per].t().contiguous(), v[h // per]
        for a in range(0, q.shape[1], 512):
            b = min(a + 512, q.shape[1])
            x = q[h, a:b].double() @ keys
            p = torch.arange(start + a, start + b, device=DEV)[:, None]
            j = torch.arange(k.shape[1], device=DEV)[None]
            hidden = j > p
            if window:
                hidden |= (j <= p - window) & (j >= sinks)
            out[h, a:b] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ values
    return out


def _exact_values(x, codes):
    """[KV, n, D] in 64 bits as the cache holds them: the scale in fp32, the quotient rounded to fp32, then to a code."""
    out = x.double()
    for b in range(x.shape[1] // BLOCK):
        rows = out[:, b * BLOCK:(b + 1) * BLOCK]
        top = torch.maximum(rows.abs().flatten(1).max(1).values, torch.tensor(1e-8, device=DEV).double())
        scale = (top.float() / (127.0 if codes == "int8" else 448.0))[:, None, None].double()
        ratio = (rows / scale).float()
        code = torch.round(ratio).double() if codes == "int8" else ratio.to(torch.float8_e4m3fn).double()
        out[:, b * BLOCK:(b + 1) * BLOCK] = code * scale
    return out


def _exact_verify(s):
    b, n = s["batch"], s["n"]
    counts, paths, tokens = [], [], []
    drafted = s["tokens"].tolist()
    u = s["uniforms"].tolist()
    soft = lambda row: torch.softmax(row.double() / s["temperature"], -1)  # noqa: E731
    for i in range(b):
        path, refused = [], []
        if s["draft"] == "tree":
            parents = s["parents"].tolist()
            at, left, p = -1, 1.0, soft(s["logits"][i, 0])
            r = p.clone()
            for m in range(n):
                if parents[m] != at:
                    continue
                x = r[drafted[i][m]].item()
                if u[i][m] * left < x:
                    at = m
                    path.append(m)
                    left, p = 1.0, soft(s["logits"][i, m + 1])
                    r = p.clone()
                else:
                    left -= x
                    r[drafted[i][m]] = 0.0
        else:
            length = n if s["lengths"] is None else int(s["lengths"][i])
            r = p = soft(s["logits"][i, 0])
            for m in range(length):
                t = drafted[i][m]
                if s["draft_logits"] is None:
                    q = torch.zeros_like(p)
                    q[t] = 1.0
                else:
                    q = soft(s["draft_logits"][i, m])
                if u[i][m] * q[t].item() < p[t].item():
                    path.append(m)
                    r = p = soft(s["logits"][i, m + 1])
                else:
                    r = torch.relu(p - q)
                    break
        if r.sum().item() <= 0:
            r = p
        c = torch.cumsum(r, 0)
        tokens.append(int(torch.searchsorted(c, torch.tensor([u[i][n]], device=DEV).double() * c[-1], right=True)))
        counts.append(len(path))
        paths.append(path + [-1] * (n - len(path)))
    return [torch.tensor(counts, device=DEV, dtype=torch.int32), torch.tensor(paths, device=DEV), torch.tensor(tokens, device=DEV)]


def exact(case, seed):
    global own
    kind = case["kind"]
    mine, own = own, False  # the inputs alone
    try:
        if kind == "attend":
            g = torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 11)
            q = (_randn(g, case["h"], case["n"], case["d"]) * (2 * case["d"] ** -0.5)).bfloat16()
            k, v = (_randn(g, case["kv"], case["rows"], case["d"]).bfloat16() for _ in range(2))
            return _exact_attention(q, _exact_values(k, case["codes"]), _exact_values(v, case["codes"]), case["rows"] - case["n"],
                                    case["window"], case["sinks"])
        s = prepare(case, seed)
    finally:
        own = mine
    if kind == "verify":
        return _exact_verify(s)
    if kind == "sinks":
        return _exact_attention(s["q"], s["k"].double(), s["v"].double(), s["start"], s["window"], s["sinks"])
    first = s["start"] // BLOCK * BLOCK
    return [_exact_values(s[x][:, first:], s["codes"]) for x in ("k", "v")]
