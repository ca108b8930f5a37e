"""Cases of the operators that keep long contexts affordable: attention over a window with sinks, attention of a batch behind
one shared prefix, attention that accumulates the cache's attention weights, and eviction by those weights.

``listed()`` / ``draw()`` give cases, ``prepare`` what a serving loop has in hand (rotated q, the new K / V rows, caches,
positions), ``run`` one pass: elementary torch operations in 32 bits, or with ``own`` the framework's ops.
"""

import math

import numpy as np
import torch

own = False

# (query heads, KV heads): the 8B and 70B shapes, a 70B rank's share, groups that are no power of two, one head per group
HEADS = ((32, 8), (64, 8), (8, 1), (14, 2), (12, 4), (16, 16))


def listed():
    return [
        # one user of a streaming chat, a short window: latency
        {"name": "window b1", "op": "window", "B": 1, "H": 32, "KV": 8, "D": 128, "n": 1, "S": 8192, "lo": 7000, "hi": 7000,
         "window": 1024, "sinks": 4, "bf16": False, "write": True},
        # a batch at ragged positions, rows already appended by the fused RoPE + append
        {"name": "window b32", "op": "window", "B": 32, "H": 32, "KV": 8, "D": 128, "n": 1, "S": 16384, "lo": 2000, "hi": 16300,
         "window": 4096, "sinks": 4, "bf16": True, "write": False},
        # a long prompt's second chunk
        {"name": "window prompt 2048", "op": "window", "B": 1, "H": 32, "KV": 8, "D": 128, "n": 2048, "S": 8192, "lo": 6000, "hi": 6000,
         "window": 4096, "sinks": 16, "bf16": False, "write": True},
        # short prompts of a small model, odd everywhere
        {"name": "window prompt 77 odd", "op": "window", "B": 3, "H": 14, "KV": 2, "D": 64, "n": 77, "S": 2501, "lo": 100, "hi": 2300,
         "window": 333, "sinks": 5, "bf16": True, "write": True},
        # a few users behind one system prompt
        {"name": "prefix b16", "op": "prefix", "B": 16, "H": 32, "KV": 8, "D": 128, "n": 1, "P": 4096, "S": 512, "lo": 0, "hi": 500,
         "bf16": False, "write": True},
        # many answers about one long document, 70B heads
        {"name": "prefix b64 32k", "op": "prefix", "B": 64, "H": 64, "KV": 8, "D": 128, "n": 1, "P": 32768, "S": 1024, "lo": 100, "hi": 1000,
         "bf16": False, "write": False},
        # verification of three tokens, odd sizes
        {"name": "prefix b7 odd", "op": "prefix", "B": 7, "H": 12, "KV": 4, "D": 64, "n": 3, "P": 1531, "S": 300, "lo": 0, "hi": 290,
         "bf16": True, "write": True},
        # one user, weights kept
        {"name": "scored b1", "op": "scored", "B": 1, "H": 32, "KV": 8, "D": 128, "n": 1, "S": 4096, "lo": 4000, "hi": 4000,
         "bf16": False, "write": True},
        {"name": "scored b32", "op": "scored", "B": 32, "H": 32, "KV": 8, "D": 128, "n": 1, "S": 8192, "lo": 1000, "hi": 8100,
         "bf16": False, "write": False},
        # the last tokens of a prompt look back over it, to decide what of it stays
        {"name": "scored observe 16", "op": "scored", "B": 4, "H": 32, "KV": 8, "D": 128, "n": 16, "S": 8192, "lo": 5000, "hi": 8100,
         "bf16": False, "write": False},
        # one prompt's cache cut down
        {"name": "evict b1", "op": "evict", "B": 1, "KV": 8, "D": 128, "S": 8192, "lo": 8000, "hi": 8000, "keep": 2048, "room": 2560,
         "sinks": 4, "recent": 256},
        {"name": "evict b16", "op": "evict", "B": 16, "KV": 8, "D": 128, "S": 16384, "lo": 3000, "hi": 16384, "keep": 4096, "room": 4352,
         "sinks": 4, "recent": 512},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("window", "window", "prefix", "scored", "evict"))
    h, kv = rng.choice(HEADS)
    d = rng.choice((64, 128, 128, 256))
    case = {"op": op, "B": _log(rng, 1, 32), "H": h, "KV": kv, "D": d}
    if op == "evict":
        del case["H"]
        s = _log(rng, 300, 16384)
        case["B"] = max(1, min(case["B"], (1 << 27) // (s * kv * d)))
        keep = rng.randint(max(16, s // 16), s // 2)
        sinks, recent = rng.randint(0, min(16, keep // 4)), rng.randint(0, keep // 2)
        hi = rng.randint(s // 2, s)
        return {**case, "S": s, "lo": rng.randint(hi // 4, hi), "hi": hi, "keep": keep, "room": keep + rng.randint(0, keep // 4), "sinks": sinks,
                "recent": recent}
    case["bf16"] = rng.random() < 0.4
    case["write"] = rng.random() < 0.3
    if op == "window":
        prompt = rng.random() < 0.4
        n = _log(rng, 2, 1500) if prompt else 1
        s = _log(rng, max(64, n + 1), 12000)
        case["B"] = max(1, min(case["B"], (1 << 27) // (s * kv * d), (1 << 26) // (n * h * s // 8 + 1)))
        hi = rng.randint((s - n) // 2, s - n)
        case = {**case, "n": n, "S": s, "lo": rng.randint(0, hi), "hi": hi, "window": _log(rng, 16, 8192), "sinks": rng.choice((0, 1, 4, 16, 37, 100))}
        while work(case)["flops"] > 1.3e11:                                    # a prompt as large as the largest listed one, no larger
            case["n"] = case["n"] * 3 // 4
        return case
    case["n"] = rng.choice((1, 1, 1, 2, 3, 5)) if op == "prefix" else rng.choice((1, 1, 1, 4, 13))
    if op == "prefix":
        case["P"] = _log(rng, 200, 30000)
        case["B"] = max(2, min(case["B"], (1 << 32) // (case["P"] * h * d * case["n"])))
        s = _log(rng, 32, 2000)
    else:
        s = _log(rng, 64, 12000)
        case["B"] = max(1, min(case["B"], (1 << 27) // (s * kv * d)))
    hi = rng.randint((s - case["n"]) // 2, s - case["n"])
    return {**case, "S": s, "lo": rng.randint(0, hi), "hi": hi}


def _spread(c):
    """The sequences' positions, i.e. the cache rows that each holds before the call: from hi down to lo, scattered."""
    return [c["hi"] - int((c["hi"] - c["lo"]) * (i * 0.6180339887498949 % 1.0)) for i in range(c["B"])]


def _normal(gen, shape, scale=1.0, dtype=torch.float16):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen).to(dtype)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    if own:
        import alloy_b200  # noqa: F401
    b, kv, d, s = c["B"], c["KV"], c["D"], c["S"]
    st = {"case": dict(c), "k": torch.empty((b, kv, s, d), dtype=torch.float16, device="cuda").normal_(generator=gen),
          "v": torch.empty((b, kv, s, d), dtype=torch.float16, device="cuda").normal_(generator=gen),
          "pos": torch.tensor(_spread(c), dtype=torch.int32, device="cuda")}
    if c["op"] in ("scored", "evict"):
        # sums of probabilities over earlier steps: heavy-tailed, positive; one in eight never attended to
        w = torch.empty((b, kv, s), dtype=torch.float32, device="cuda").normal_(-3.0, 1.5, generator=gen).exp_()
        st["w"] = w * (torch.rand((b, kv, s), device="cuda", generator=gen) > 0.125)
    if c["op"] == "evict":
        st["k_out"] = torch.zeros((b, kv, c["room"], d), dtype=torch.float16, device="cuda")
        st["v_out"] = torch.zeros((b, kv, c["room"], d), dtype=torch.float16, device="cuda")
        st["w_out"] = torch.zeros((b, kv, c["room"]), dtype=torch.float32, device="cuda")
        return st
    h, n = c["H"], c["n"]
    # what the projections leave: (B, n, heads, D), seen as (B, heads, n, D)
    st["q"] = _normal(gen, (b, n, h, d), 1.5, torch.bfloat16 if c["bf16"] else torch.float16).transpose(1, 2)
    st["nk"] = _normal(gen, (b, n, kv, d)).transpose(1, 2)
    st["nv"] = _normal(gen, (b, n, kv, d)).transpose(1, 2)
    if not c["write"]:
        _append(st)
    if c["op"] == "prefix":
        # the prefix's rows at the front of a store with room for more
        st["pk"] = _normal(gen, (kv, c["P"] + 16, d))[:, :c["P"]]
        st["pv"] = _normal(gen, (kv, c["P"] + 16, d))[:, :c["P"]]
    return st


def _rows(st):
    """(B, n): the cache rows of the new tokens."""
    return st["pos"].long()[:, None] + torch.arange(st["case"]["n"], device="cuda")


def _append(st):
    at = torch.arange(st["case"]["B"], device="cuda")[:, None]
    st["k"][at, :, _rows(st)] = st["nk"].transpose(1, 2)
    st["v"][at, :, _rows(st)] = st["nv"].transpose(1, 2)


def _softmax(s, seen):
    s = torch.where(seen, s, torch.full((), -math.inf, device="cuda"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    z = p.sum(-1, keepdim=True)
    return p / torch.where(z == 0, torch.ones_like(z), z)


def _plain(st):
    c = st["case"]
    if c["op"] == "evict":
        return _plain_evict(st)
    b, h, kv, d, n = c["B"], c["H"], c["KV"], c["D"], c["n"]
    g, scale = h // kv, 1.0 / math.sqrt(d)
    if c["write"]:
        _append(st)
    q = st["q"].float().reshape(b, kv, g * n, d) * scale                      # rows (head of the group, token)
    j = torch.arange(c["S"], device="cuda")
    p_row = _rows(st).repeat(1, g)[:, None, :, None]                           # position of each row
    seen = j <= p_row
    if c["op"] == "window":
        seen = seen & ((j > p_row - c["window"]) | (j < c["sinks"]))
    s = q @ st["k"].float().transpose(-1, -2)
    seen = seen.expand(s.shape)
    if c["op"] == "prefix":
        qp = q.transpose(0, 1).reshape(kv, b * g * n, d)
        sp = (qp @ st["pk"].float().transpose(-1, -2)).reshape(kv, b, g * n, c["P"]).transpose(0, 1)
        p = _softmax(torch.cat([sp, s], -1), torch.cat([torch.ones_like(sp, dtype=torch.bool), seen], -1))
        pp = p[..., :c["P"]].transpose(0, 1).reshape(kv, b * g * n, c["P"])
        o = p[..., c["P"]:] @ st["v"].float() + (pp @ st["pv"].float()).reshape(kv, b, g * n, d).transpose(0, 1)
    else:
        p = _softmax(s, seen)
        o = p @ st["v"].float()
    out = {"out": o.reshape(b, h, n, d).to(st["q"].dtype)}
    if c["op"] == "scored":
        add = p.sum(2)
        first = st["pos"].long()[:, None, None]
        w = st["w"]
        st["w"].copy_(torch.where(j < first, w + add, torch.where(j < first + n, add, w)))
        out["weights"] = st["w"]
    if c["write"]:
        out["k"], out["v"] = st["k"], st["v"]
    return out


def _plain_evict(st):
    c = st["case"]
    length = st["pos"].long()[:, None, None]
    j = torch.arange(c["S"], device="cuda")
    kept_for_sure = (j < c["sinks"]) | (j >= length - c["recent"])
    key = torch.where(kept_for_sure, torch.full((), math.inf, device="cuda"), st["w"])
    key = torch.where(j < length, key, torch.full((), -math.inf, device="cuda"))
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    kept = torch.where(best < length, best, torch.full((), c["S"], device="cuda")).sort(-1).values
    live = kept < c["S"]
    at = torch.where(live, kept, torch.zeros_like(kept))
    rows = at[..., None].expand(-1, -1, -1, c["D"])
    keep = c["keep"]
    for name in ("k", "v"):
        dst = st[name + "_out"][:, :, :keep]
        dst.copy_(torch.where(live[..., None], st[name].gather(2, rows), dst))
    dst = st["w_out"][:, :, :keep]
    dst.copy_(torch.where(live, st["w"].gather(2, at), dst))
    return {"k": st["k_out"], "v": st["v_out"], "weights": st["w_out"],
            "kept": torch.where(live, kept, torch.full_like(kept, -1)).to(torch.int32),
            "lengths": torch.clamp(st["pos"], max=keep)}


def _own(st):
    c, ops = st["case"], torch.ops.alloy
    if c["op"] == "evict":
        kept, lengths = ops.kv_evict(st["k"], st["v"], st["w"], st["pos"], st["k_out"], st["v_out"], st["w_out"], c["keep"], c["sinks"],
                                     c["recent"])
        return {"k": st["k_out"], "v": st["v_out"], "weights": st["w_out"], "kept": kept, "lengths": lengths}
    args = (st["q"], st["nk"], st["nv"], st["pos"])
    if c["op"] == "window":
        out = {"out": ops.attention_cache_window(*args, st["k"], st["v"], c["window"], c["sinks"], -1.0, c["write"])}
    elif c["op"] == "prefix":
        out = {"out": ops.attention_shared_prefix(*args, st["pk"], st["pv"], st["k"], st["v"], -1.0, c["write"])}
    else:
        out = {"out": ops.attention_cache_scored(*args, st["k"], st["v"], st["w"], -1.0, c["write"]), "weights": st["w"]}
    if c["write"]:
        out["k"], out["v"] = st["k"], st["v"]
    return out


def run(state):
    return _own(state) if own else _plain(state)


def _seen(c, p):
    """How many cache rows a query at position p sees."""
    if c["op"] != "window":
        return p + 1
    lo = max(0, p - c["window"] + 1)
    return p + 1 - lo + min(c["sinks"], lo)


def work(case):
    c = case
    b, kv, d = c["B"], c["KV"], c["D"]
    pos = _spread(c)
    if c["op"] == "evict":
        kept = [min(p, c["keep"]) for p in pos]
        return {"bytes": kv * sum(4 * p + 2 * 2 * k * 2 * d + (4 + 4) * k for p, k in zip(pos, kept)), "flops": 0}
    h, n = c["H"], c["n"]
    pairs = sum(_seen(c, p + i) for p in pos for i in range(n))                # (query token, row) pairs, per query head
    rows = 0                                                                   # cache rows that some query of a sequence sees
    for p in pos:
        lo = max(0, p - c["window"] + 1) if c["op"] == "window" else 0
        rows += p + n - lo + (min(c["sinks"], lo) if c["op"] == "window" else 0)
    size = 2 * kv * rows * d * 2 + 2 * 2 * b * n * h * d
    if c["write"]:
        size += 2 * 2 * b * n * kv * d                                         # the new rows go into the cache
    if c["op"] == "prefix":
        pairs += b * n * c["P"]
        size += 2 * kv * c["P"] * d * 2
    if c["op"] == "scored":
        size += 2 * 4 * kv * rows
    return {"bytes": size, "flops": 4 * d * h * pairs}


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    b, kv, d, s = c["B"], c["KV"], c["D"], c["S"]
    if c["op"] == "evict":
        k_out, v_out, w_out = (st[x].double() for x in ("k_out", "v_out", "w_out"))
        kept = np.full((b, kv, c["keep"]), -1, dtype=np.int64)
        w = st["w"].double().cpu().numpy()
        for i, p in enumerate(_spread(c)):
            for h in range(kv):
                fixed = set(range(min(c["sinks"], p))) | set(range(max(0, p - c["recent"]), p))
                rest = np.array([x for x in range(p) if x not in fixed], dtype=np.int64)
                order = rest[np.lexsort((rest, -w[i, h, rest]))] if rest.size else rest
                rows = np.sort(np.concatenate([np.array(sorted(fixed), dtype=np.int64), order[:max(0, c["keep"] - len(fixed))]]))
                kept[i, h, :rows.size] = rows
                at = torch.from_numpy(rows).cuda()
                k_out[i, h, :rows.size], v_out[i, h, :rows.size] = st["k"][i, h, at].double(), st["v"][i, h, at].double()
                w_out[i, h, :rows.size] = st["w"][i, h, at].double()
        return {"k": k_out, "v": v_out, "weights": w_out, "kept": kept.astype(np.int32),
                "lengths": torch.tensor([min(p, c["keep"]) for p in _spread(c)], dtype=torch.int32)}
    h, n = c["H"], c["n"]
    g = h // kv
    out = torch.zeros((b, h, n, d), dtype=torch.float64, device="cuda")
    weights = st["w"].double() if c["op"] == "scored" else None
    for i, p in enumerate(_spread(c)):
        if c["write"]:
            st["k"][i, :, p:p + n], st["v"][i, :, p:p + n] = st["nk"][i], st["nv"][i]
        at = torch.arange(p + n, device="cuda")
        row = p + torch.arange(n, device="cuda")[:, None]
        hidden = at > row
        if c["op"] == "window":
            hidden |= (at <= row - c["window"]) & (at >= c["sinks"])
        for kh in range(kv):
            k, v = st["k"][i, kh, :p + n].double(), st["v"][i, kh, :p + n].double()
            z = torch.einsum("gnd,jd->gnj", st["q"][i, kh * g:(kh + 1) * g].double(), k) / math.sqrt(d)
            z.masked_fill_(hidden, -math.inf)
            if c["op"] == "prefix":
                z = torch.cat([torch.einsum("gnd,jd->gnj", st["q"][i, kh * g:(kh + 1) * g].double(), st["pk"][kh].double()) / math.sqrt(d), z], -1)
                v = torch.cat([st["pv"][kh].double(), v], 0)
            z = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
            out[i, kh * g:(kh + 1) * g] = torch.einsum("gnj,jd->gnd", z, v)
            if weights is not None:
                weights[i, kh, p:p + n] = 0.0
                weights[i, kh, :p + n] += z.sum((0, 1))
    got = {"out": out}
    if weights is not None:
        got["weights"] = weights
    if c["write"]:
        got["k"], got["v"] = st["k"], st["v"]
    return got
