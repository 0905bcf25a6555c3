"""The attention cache's operators as they are measured: cases, inputs, plain forms and exact values.

A cache holds the key and value rows of `n_seqs` sequences in 4 bits. Four operators work on it:

append  quantises new key and value rows into the cache; the pass reads the rows back as values.
attend  softmax attention of each sequence's query tokens over its cached rows, with the
        log-sum-exp and, where the case asks for it, the rows' accumulated attention weight.
found   the same over rows named by a list per token, as an index search returns them (ids padded
        with 2^64 - 1, which is -1 in a signed tensor).
evict   keeps each sequence's heaviest rows by accumulated weight and closes the gaps; the pass
        reads the kept rows back as values.

The format. A row of one head is cut into groups of 64 dimensions. A group has
step = bf16(f32(f32(max - min) / 15)), low = bf16(min), and per element the code in 0..15 whose level
low + step * code is nearest (ties to the even code; 0 where the step is 0). A code stands for
f32(low + step * code).
"""
import math
import random

import torch

own = False

GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases ----------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a batch: a token a sequence
        {"name": "append_step", "op": "append", "dtype": "bf16", "n_seqs": 64, "heads": 8, "dim": 128,
         "rows_min": 300, "rows_max": 4000, "new_min": 1, "new_max": 1},
        # prompts of a ragged batch, stored before their first token is answered
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "n_seqs": 8, "heads": 8, "dim": 128,
         "rows_min": 0, "rows_max": 0, "new_min": 1000, "new_max": 8000},
        # odd sizes: three heads of 80, continued prompts, empty sequences among them
        {"name": "append_odd", "op": "append", "dtype": "f16", "n_seqs": 13, "heads": 3, "dim": 80,
         "rows_min": 0, "rows_max": 777, "new_min": 0, "new_max": 333},
        # the smallest call: one sequence, one token, where latency counts
        {"name": "attend_one", "op": "attend", "dtype": "bf16", "n_seqs": 1, "heads": 8, "group": 4, "dim": 128,
         "rows_min": 777, "rows_max": 777, "new_min": 1, "new_max": 1, "weights": False},
        # a decoding step of a serving batch whose cache evicts by weight
        {"name": "attend_batch_weights", "op": "attend", "dtype": "bf16", "n_seqs": 64, "heads": 8, "group": 4,
         "dim": 128, "rows_min": 500, "rows_max": 8000, "new_min": 1, "new_max": 1, "weights": True},
        # one long document: few rows of queries, the work is split over the rows
        {"name": "attend_long", "op": "attend", "dtype": "f16", "n_seqs": 1, "heads": 8, "group": 8, "dim": 128,
         "rows_min": 262144, "rows_max": 262144, "new_min": 1, "new_max": 1, "weights": False},
        # a chunk of a prompt over a long prefix
        {"name": "attend_chunk", "op": "attend", "dtype": "bf16", "n_seqs": 4, "heads": 8, "group": 4, "dim": 128,
         "rows_min": 20000, "rows_max": 32000, "new_min": 32, "new_max": 64, "weights": False},
        # single-precision read-out of stored embeddings of the index's dimension, odd lengths
        {"name": "attend_f32", "op": "attend", "dtype": "f32", "n_seqs": 5, "heads": 1, "group": 3, "dim": 384,
         "rows_min": 0, "rows_max": 5001, "new_min": 1, "new_max": 3, "weights": True},
        # the read-out after a search: the best rows of one query each
        {"name": "found_step", "op": "found", "dtype": "bf16", "n_seqs": 16, "heads": 1, "group": 8, "dim": 128,
         "rows_min": 20000, "rows_max": 100000, "new_min": 1, "new_max": 1, "k": 100},
        # a batch of 1,000 queries over one store, some lists not full
        {"name": "found_batch", "op": "found", "dtype": "f32", "n_seqs": 1, "heads": 2, "group": 2, "dim": 64,
         "rows_min": 500000, "rows_max": 500000, "new_min": 1000, "new_max": 1000, "k": 257},
        # a decoding step at the budget: one row goes out
        {"name": "evict_step", "op": "evict", "dtype": "bf16", "n_seqs": 32, "heads": 4, "dim": 128,
         "rows_min": 1025, "rows_max": 1025, "keep": 1024, "recent": 32},
        # long prompts cut down to the budget
        {"name": "evict_prompts", "op": "evict", "dtype": "bf16", "n_seqs": 16, "heads": 8, "dim": 128,
         "rows_min": 3000, "rows_max": 32768, "keep": 2048, "recent": 128},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "found", "evict"])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "heads": rng.choice([1, 2, 3, 4, 8]),
            "dim": rng.choice([32, 40, 64, 80, 96, 128, 128, 192, 256, 384]), "rows_seed": rng.randrange(1 << 30)}
    row_elems = case["heads"] * case["dim"]
    if op == "append":
        n = _log_int(rng, 1, 96)
        hi = _log_int(rng, 1, max(1, min(8000, 15_000_000 // (row_elems * n))))
        case.update(n_seqs=n, rows_min=0, rows_max=_log_int(rng, 1, 1500), new_min=rng.randint(0, min(hi, 3)),
                    new_max=hi)
    elif op == "attend":
        n = _log_int(rng, 1, 64)
        new = rng.choice([1, 1, 1, 2, 5, _log_int(rng, 2, 64)])
        group = rng.choice([1, 2, 3, 4, 5, 8, 16])
        top = max(64, min(200_000, 200_000_000 // (row_elems * n), 40_000_000 // (n * new * case["heads"] * group)))
        hi = _log_int(rng, 64, top)
        case.update(n_seqs=n, group=group, rows_min=rng.choice([0, hi // 2, hi]), rows_max=hi,
                    new_min=rng.choice([0, 1, new]), new_max=new, weights=rng.random() < 0.5)
    elif op == "found":
        n = _log_int(rng, 1, 16)
        new = _log_int(rng, 1, max(1, 1000 // n))
        group = rng.choice([1, 2, 4, 7, 8])
        hi = _log_int(rng, 100, max(100, min(500_000, 60_000_000 // (row_elems * n))))
        k = _log_int(rng, 1, max(1, min(1000, 60_000_000 // (row_elems * n * new))))
        case.update(n_seqs=n, group=group, rows_min=hi // 2, rows_max=hi, new_min=1, new_max=new, k=k)
    else:
        n = _log_int(rng, 1, 32)
        hi = _log_int(rng, 2, max(2, min(40_000, 120_000_000 // (row_elems * n))))
        case.update(n_seqs=n, rows_min=hi // 3, rows_max=hi, keep=_log_int(rng, 1, hi), recent=rng.choice([0, 1, 32]))
        case["keep"] = max(1, min(case["keep"], 25_000_000 // (row_elems * n)))
    return case


def _plan(case):
    """Rows held before the call and new tokens of every sequence; from the case alone."""
    rng = random.Random(case.get("rows_seed", 12345))
    rows = [rng.randint(case["rows_min"], case["rows_max"]) for _ in range(case["n_seqs"])]
    new = [rng.randint(case["new_min"], case["new_max"]) if "new_max" in case else 0 for _ in range(case["n_seqs"])]
    if sum(rows) == 0:
        rows[0] = max(1, case["rows_max"])
    if "new_max" in case and sum(new) == 0:
        new[-1] = case["new_max"]
    if case["op"] == "append" and case["rows_max"] == 0:
        rows = [0] * case["n_seqs"]
    return rows, new


def _row_bytes(case):
    return 2 * case["heads"] * (case["dim"] / 2 + 4 * -(-case["dim"] // GROUP))


def work(case):
    rows, new = _plan(case)
    es = 4 if case["dtype"] == "f32" else 2
    hd = case["heads"] * case["dim"]
    rb = _row_bytes(case)
    if case["op"] == "append":
        t = sum(new)
        return {"bytes": t * (2 * hd * es + rb + 2 * hd * es + 8), "flops": t * hd * 2 * 8}
    if case["op"] == "evict":
        kept = [min(r, case["keep"]) for r in rows]
        moved = sum(k * (r - k) / r for k, r in zip(kept, rows) if r)
        out = sum(kept)
        return {"bytes": sum(rows) * 12 + out * 12 + (sum(rows) - out) * 8 + moved * 2 * rb + out * (rb + 2 * hd * es),
                "flops": sum(rows) * 4}
    q = sum(new) * hd * case["group"]
    if case["op"] == "found":
        pairs = sum(n * min(case["k"], r) for n, r in zip(new, rows))
        touched = sum(min(r, n * case["k"]) for n, r in zip(new, rows))
        return {"bytes": touched * rb + pairs * (8 + 4) + 2 * q * es, "flops": 4 * pairs * hd * case["group"]}
    total = [r + n for r, n in zip(rows, new)]
    pairs = sum(n * r + n * (n + 1) // 2 for r, n in zip(rows, new))
    seen = sum(t for t, n in zip(total, new) if n)
    return {"bytes": seen * rb + 2 * q * es + (8 * sum(total) if case["weights"] else 0),
            "flops": 4 * pairs * hd * case["group"]}


# ---- inputs ---------------------------------------------------------------------------------------
def _tokens(n, heads, dim, dtype, gen, scale, spread):
    """n rows of every head: a fixed offset per channel, larger in a few of them, plus noise."""
    mean = torch.randn(heads, dim, generator=gen, device="cuda") * spread
    mean[:, :: max(1, dim // 4)] *= 4.0
    out = torch.empty(n, heads, dim, dtype=dtype, device="cuda")
    step = max(1, 100_000_000 // max(1, heads * dim))
    for i in range(0, n, step):
        m = min(step, n - i)
        out[i:i + m] = (torch.randn(m, heads, dim, generator=gen, device="cuda") + mean) * scale
    return out


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, new = _plan(case)
    dt = DTYPES[case["dtype"]]
    n_seqs, heads, dim = case["n_seqs"], case["heads"], case["dim"]
    # what a cache already holds (attend: the step's own rows are in it as well)
    held = [r + n for r, n in zip(rows, new)] if case["op"] == "attend" else rows
    d = {"rows": rows, "new": new, "held": held, "total": [r + n for r, n in zip(rows, new)]}
    d["capacity"] = max(max(d["total"]), 1)
    if case["op"] == "append":
        d["keys"] = _tokens(sum(new), heads, dim, dt, gen, 1.0, 0.5)
        d["values"] = _tokens(sum(new), heads, dim, dt, gen, 0.7, 0.1)
    else:
        d["keys"] = _tokens(sum(held), heads, dim, dt, gen, 1.0, 0.5)
        d["values"] = _tokens(sum(held), heads, dim, dt, gen, 0.7, 0.1)
    if case["op"] in ("attend", "found"):
        t, hq = sum(new), heads * case["group"]
        q = torch.randn(t, hq, dim, generator=gen, device="cuda") * 0.7
        # every query leans towards one stored key, as a trained model's queries do
        first, pick = 0, []
        for h, n in zip(held, new):
            pick.append(first + (torch.rand(n, generator=gen, device="cuda") * max(h, 1)).long().clamp(max=max(h - 1, 0)))
            first += h
        if sum(held):
            near = d["keys"][torch.cat(pick).clamp(max=sum(held) - 1)].float()
            q += 0.3 * near.repeat_interleave(case["group"], dim=1)
        d["q"] = q.to(dt)
        d["scale"] = 1.0 / math.sqrt(dim)
    if case["op"] == "attend" and case["weights"]:
        d["w_in"] = torch.rand(n_seqs, d["capacity"], generator=gen, device="cuda") ** 4
        d["decay"] = 0.97
    if case["op"] == "found":
        k = case["k"]
        lists = []
        for h, n in zip(held, new):
            if k <= h // 4:
                # distinct rows of one stretch each, as the cells of an index give them
                base = (torch.rand(n, 1, generator=gen, device="cuda") * h).long()
                gap = torch.randint(1, max(2, h // k), (n, k), generator=gen, device="cuda").cumsum(1)
                ids = (base + gap) % max(h, 1)
            else:
                ids = torch.rand(n, max(h, 1), generator=gen, device="cuda").argsort(dim=1)[:, :k] if h else \
                    torch.full((n, k), -1, device="cuda")
                if ids.shape[1] < k:
                    ids = torch.cat([ids, torch.full((n, k - ids.shape[1]), -1, device="cuda")], dim=1)
            short = torch.rand(n, 1, generator=gen, device="cuda") < 0.2
            cut = (torch.rand(n, 1, generator=gen, device="cuda") * (k + 1)).long()
            drop = short & (torch.arange(k, device="cuda")[None] >= cut)
            lists.append(ids.masked_fill(drop, -1))
        d["lists"] = torch.cat(lists).contiguous()
    if case["op"] == "evict":
        w = torch.rand(n_seqs, d["capacity"], generator=gen, device="cuda") ** 6
        # rows that were never looked at share the weight 0
        w[torch.rand(n_seqs, d["capacity"], generator=gen, device="cuda") < 0.2] = 0.0
        d["w_in"] = w
        d["ids"] = torch.arange(d["capacity"], device="cuda").repeat(n_seqs, 1) + 1000
        d["protect"] = torch.tensor([1000 + max(r - case["recent"], 0) for r in rows], device="cuda")
    return d


def _offsets(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device="cuda")


# ---- the plain form -------------------------------------------------------------------------------
def _quantise(x):
    """Rows [n, heads, dim] -> codes [n, heads, dim] (uint8), step and low [n, heads, groups] (f32)."""
    n, heads, dim = x.shape
    groups = -(-dim // GROUP)
    codes = torch.empty(n, heads, dim, dtype=torch.uint8, device=x.device)
    step = torch.empty(n, heads, groups, device=x.device)
    low = torch.empty(n, heads, groups, device=x.device)
    for g in range(groups):
        part = x[:, :, g * GROUP:(g + 1) * GROUP].float()
        hi, lo = part.amax(dim=-1), part.amin(dim=-1)
        s = ((hi - lo) / 15.0).to(torch.bfloat16).float()
        lo = lo.to(torch.bfloat16).float()
        # 64 bits: the nearest level of values next to the middle between two
        at = (part.double() - lo[..., None].double()) / torch.where(s == 0, 1.0, s)[..., None].double()
        c = torch.where(s[..., None] == 0, 0.0, at.round().clamp(0, 15))
        codes[:, :, g * GROUP:(g + 1) * GROUP] = c.to(torch.uint8)
        step[:, :, g], low[:, :, g] = s, lo
    return codes, step, low


def _quantise_rows(x):
    rows = max(1, 60_000_000 // max(1, x.shape[1] * x.shape[2]))
    parts = [_quantise(x[i:i + rows]) for i in range(0, max(1, x.shape[0]), rows)]
    return tuple(torch.cat(p) for p in zip(*parts)) if len(parts) > 1 else parts[0]


def _values(codes, step, low):
    """What the codes stand for, f32; step and low are per group of the last dimension."""
    dim = codes.shape[-1]
    s = step.repeat_interleave(GROUP, dim=-1)[..., :dim]
    lo = low.repeat_interleave(GROUP, dim=-1)[..., :dim]
    return lo + s * codes.float()


def _store(codes, step, low, held, capacity):
    """Packed rows laid out per sequence: [n_seqs, capacity, heads, ...]."""
    out = []
    for t in (codes, step, low):
        b = torch.zeros(len(held), capacity, *t.shape[1:], dtype=t.dtype, device=t.device)
        first = 0
        for s, n in enumerate(held):
            b[s, :n] = t[first:first + n]
            first += n
        out.append(b)
    return out


def _prepare_plain(case, d):
    st = dict(case=case, rows=d["rows"], new=d["new"], held=d["held"], capacity=d["capacity"])
    dev = "cuda"
    st["lengths"] = torch.tensor(d["rows"], dtype=torch.int32, device=dev)
    st["offsets"] = _offsets(d["new"])
    for name in ("q", "scale", "w_in", "decay", "lists", "ids", "protect"):
        if name in d:
            st[name] = d[name]
    if case["op"] == "append":
        st["keys"], st["values"] = d["keys"], d["values"]
        st["w_table"] = torch.ones(case["n_seqs"], d["capacity"], device=dev)
        st["where"] = torch.cat([s * d["capacity"] + r + torch.arange(n, device=dev)
                                 for s, (r, n) in enumerate(zip(d["rows"], d["new"]))])
    else:
        st["k"] = _store(*_quantise_rows(d["keys"]), d["held"], d["capacity"])
        st["v"] = _store(*_quantise_rows(d["values"]), d["held"], d["capacity"])
    if case["op"] == "attend" and case["weights"]:
        st["w_out"] = torch.zeros_like(d["w_in"])
    return st


def _plain_append(st):
    dt = st["keys"].dtype
    out = [_values(*_quantise(x)).to(dt) for x in (st["keys"], st["values"])]
    st["w_table"].view(-1)[st["where"]] = 0.0
    return out + [st["w_table"]]


def _softmax_read(q, k, v, seen, scale, group):
    """q [n, t, hq, d]; k, v [n, r, h, d]; seen [n, t, r]. Returns out, lse and p [n, h, g, t, r], f32."""
    n, t, hq, dim = q.shape
    h = hq // group
    qh = q.view(n, t, h, group, dim).permute(0, 2, 3, 1, 4).reshape(n, h, group * t, dim).float()
    z = torch.matmul(qh, k.permute(0, 2, 3, 1)) * scale
    z = z.view(n, h, group, t, -1).masked_fill(~seen[:, None, None], -math.inf)
    top = z.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(z - top)
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p.view(n, h, group * t, -1), v.permute(0, 2, 1, 3)).view(n, h, group, t, dim)
    lse = (torch.log(total) + top)[..., 0]
    return (out.permute(0, 3, 1, 2, 4).reshape(n, t, hq, dim), lse.permute(0, 3, 1, 2).reshape(n, t, hq), p)


def _plain_attend(st):
    case, q = st["case"], st["q"]
    heads, dim, group = case["heads"], case["dim"], case["group"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[0], q.shape[1], device=q.device)
    first = [0]
    for n in st["new"]:
        first.append(first[-1] + n)
    s = 0
    while s < case["n_seqs"]:
        # sequences of one number of tokens go through together while they fit
        e, t = s + 1, st["new"][s]
        longest = st["held"][s]
        while e < case["n_seqs"] and st["new"][e] == t:
            longest_e = max(longest, st["held"][e])
            if (e + 1 - s) * longest_e * heads * (dim * 2 + group * t * 3) > 2_000_000_000:
                break
            longest, e = longest_e, e + 1
        n = e - s
        if t > 0:
            k = _values(*(x[s:e, :longest] for x in st["k"]))
            v = _values(*(x[s:e, :longest] for x in st["v"]))
            at = torch.arange(longest, device=q.device)
            limit = st["lengths"][s:e, None].long() + torch.arange(1, t + 1, device=q.device)
            seen = at[None, None] < limit[..., None]
            o, l, p = _softmax_read(q[first[s]:first[e]].view(n, t, q.shape[1], dim), k, v, seen, st["scale"], group)
            out[first[s]:first[e]] = o.reshape(n * t, -1, dim).to(q.dtype)
            lse[first[s]:first[e]] = l.reshape(n * t, -1)
        if case["weights"]:
            held = torch.tensor(st["held"][s:e], device=q.device)
            live = torch.arange(longest, device=q.device)[None] < held[:, None]
            w = st["decay"] * st["w_in"][s:e, :longest]
            if t > 0:
                w = w + p.sum(dim=(1, 2, 3))
            st["w_out"][s:e, :longest] = torch.where(live, w, st["w_out"][s:e, :longest])
        s = e
    return [out, lse] + ([st["w_out"]] if case["weights"] else [])


def _plain_found(st):
    case, q, lists = st["case"], st["q"], st["lists"]
    heads, dim, group, k = case["heads"], case["dim"], case["group"], case["k"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[0], q.shape[1], device=q.device)
    weights = torch.empty(q.shape[0], k, device=q.device)
    seq = torch.repeat_interleave(torch.arange(case["n_seqs"], device=q.device),
                                  torch.tensor(st["new"], device=q.device), output_size=q.shape[0])
    step = max(1, 500_000_000 // (k * heads * dim))
    for i in range(0, q.shape[0], step):
        rows, s = lists[i:i + step], seq[i:i + step]
        seen = (rows >= 0) & (rows < st["lengths"][s].long()[:, None])
        at = torch.where(seen, rows, 0)
        kk = _values(*(x[s[:, None], at] for x in st["k"]))
        vv = _values(*(x[s[:, None], at] for x in st["v"]))
        o, l, p = _softmax_read(q[i:i + step, None], kk, vv, seen[:, None], st["scale"], group)
        out[i:i + step] = o[:, 0].to(q.dtype)
        lse[i:i + step] = l[:, 0]
        weights[i:i + step] = p.sum(dim=(1, 2, 3))
    return [out, lse, weights]


def _plain_evict(st):
    case = st["case"]
    dt = DTYPES[case["dtype"]]
    n, cap, keep = case["n_seqs"], st["capacity"], min(case["keep"], st["capacity"])
    at = torch.arange(cap, device="cuda")
    live = at[None] < st["lengths"][:, None]
    rank = torch.where((st["ids"] >= st["protect"][:, None]) | torch.isnan(st["w_in"]), math.inf, st["w_in"])
    rank = torch.where(live, rank, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices
    kept = torch.zeros(n, cap, dtype=torch.bool, device="cuda")
    kept.scatter_(1, order[:, :keep], True)
    kept &= live
    length = torch.clamp(st["lengths"], max=keep)
    # rows that stay, then the others in ascending order into the freed places in ascending order
    inside = at[None] < length[:, None]
    hole, src = inside & ~kept, kept & ~inside
    from_row = at.repeat(n, 1)
    from_row[hole] = at.repeat(n, 1)[src]
    w_out, ids_out = torch.zeros(n, cap, device="cuda"), torch.zeros(n, cap, dtype=torch.int64, device="cuda")
    w_out[inside] = st["w_in"].gather(1, from_row)[inside]
    ids_out[inside] = st["ids"].gather(1, from_row)[inside]
    gone = live & ~kept
    evicted = torch.full((n, cap), -1, dtype=torch.int64, device="cuda")
    place = gone.long().cumsum(1) - 1
    evicted[torch.arange(n, device="cuda")[:, None].expand(n, cap)[gone], place[gone]] = st["ids"][gone]
    sel = torch.nonzero(inside)
    sel_from = from_row[inside]
    out = [_values(*(x[sel[:, 0], sel_from] for x in st[name])).to(dt) for name in ("k", "v")]
    return [length, w_out, ids_out, evicted] + out


# ---- the framework's calls ------------------------------------------------------------------------
def _prepare_own(case, d):
    from maivs_b200 import AttentionCache

    st = dict(case=case)
    n, heads, dim, cap = case["n_seqs"], case["heads"], case["dim"], d["capacity"]
    st["cache"] = cache = AttentionCache(n, cap, heads, dim, device=torch.cuda.current_device())
    st["lengths"] = torch.tensor(d["rows"], dtype=torch.int32, device="cuda")
    st["offsets"] = _offsets(d["new"])
    st["tokens"] = sum(d["new"])
    for name in ("q", "scale", "w_in", "decay", "lists", "ids", "protect"):
        if name in d:
            st[name] = d[name]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "append":
        st["keys"], st["values"] = d["keys"], d["values"]
        st["k_out"], st["v_out"] = torch.empty_like(d["keys"]), torch.empty_like(d["values"])
        st["w_table"] = torch.ones(n, cap, device="cuda")
    else:
        zero = torch.zeros(n, dtype=torch.int32, device="cuda")
        held = _offsets(d["held"])
        cache.append(d["keys"].data_ptr(), d["values"].data_ptr(), sum(d["held"]), held.data_ptr(), zero.data_ptr(),
                     dtype=case["dtype"], stream=stream)
        torch.cuda.current_stream().synchronize()
    if case["op"] in ("attend", "found"):
        st["out"] = torch.empty_like(d["q"])
        st["lse"] = torch.empty(d["q"].shape[:2], device="cuda")
    if case["op"] == "attend":
        st["max_rows"], st["max_tokens"] = max(d["total"]), max(d["new"])
        if case["weights"]:
            st["w_out"] = torch.zeros_like(d["w_in"])
        size = cache.attend_workspace(st["tokens"], d["q"].shape[1], max_rows=st["max_rows"],
                                      max_tokens=st["max_tokens"], weights=case["weights"])
    elif case["op"] == "found":
        st["weights"] = torch.empty(st["tokens"], case["k"], device="cuda")
        size = cache.attend_found_workspace(st["tokens"], d["q"].shape[1], case["k"])
    elif case["op"] == "evict":
        kept = [min(r, case["keep"]) for r in d["rows"]]
        st["kept"], st["kept_offsets"] = sum(kept), _offsets(kept)
        st["zero"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        st["new_lengths"] = torch.empty(n, dtype=torch.int32, device="cuda")
        st["w_out"] = torch.zeros_like(d["w_in"])
        st["ids_out"] = torch.zeros_like(d["ids"])
        st["evicted"] = torch.full_like(d["ids"], -1)
        dt = DTYPES[case["dtype"]]
        st["k_out"] = torch.empty(st["kept"], heads, dim, dtype=dt, device="cuda")
        st["v_out"] = torch.empty_like(st["k_out"])
        size = cache.evict_workspace()
    else:
        size = 0
    st["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return st


def _run_own(st):
    case, cache = st["case"], st["cache"]
    stream = torch.cuda.current_stream().cuda_stream
    off, lengths = st["offsets"].data_ptr(), st["lengths"].data_ptr()
    ws = dict(d_workspace=st["workspace"].data_ptr(), workspace_bytes=st["workspace"].numel(), stream=stream)
    if case["op"] == "append":
        cache.append(st["keys"].data_ptr(), st["values"].data_ptr(), st["tokens"], off, lengths, dtype=case["dtype"],
                     d_weights=st["w_table"].data_ptr(), stream=stream)
        cache.read(st["k_out"].data_ptr(), st["v_out"].data_ptr(), st["tokens"], off, lengths, dtype=case["dtype"],
                   stream=stream)
        return [st["k_out"], st["v_out"], st["w_table"]]
    if case["op"] == "attend":
        w = dict(d_weights_in=st["w_in"].data_ptr(), d_weights_out=st["w_out"].data_ptr(),
                 decay=st["decay"]) if case["weights"] else {}
        cache.attend(st["q"].data_ptr(), st["tokens"], st["q"].shape[1], off, lengths, st["out"].data_ptr(),
                     dtype=case["dtype"], causal=True, scale=st["scale"], max_rows=st["max_rows"],
                     max_tokens=st["max_tokens"], d_lse=st["lse"].data_ptr(), **w, **ws)
        return [st["out"], st["lse"]] + ([st["w_out"]] if case["weights"] else [])
    if case["op"] == "found":
        cache.attend_found(st["q"].data_ptr(), st["tokens"], st["q"].shape[1], off, lengths, st["lists"].data_ptr(),
                           case["k"], st["out"].data_ptr(), dtype=case["dtype"], scale=st["scale"],
                           d_lse=st["lse"].data_ptr(), d_weights=st["weights"].data_ptr(), **ws)
        return [st["out"], st["lse"], st["weights"]]
    cache.evict(lengths, case["keep"], st["w_in"].data_ptr(), st["w_out"].data_ptr(), st["new_lengths"].data_ptr(),
                d_ids_in=st["ids"].data_ptr(), d_ids_out=st["ids_out"].data_ptr(),
                d_protect_from=st["protect"].data_ptr(), d_evicted=st["evicted"].data_ptr(), **ws)
    cache.read(st["k_out"].data_ptr(), st["v_out"].data_ptr(), st["kept"], st["kept_offsets"].data_ptr(),
               st["zero"].data_ptr(), dtype=case["dtype"], stream=stream)
    return [st["new_lengths"], st["w_out"], st["ids_out"], st["evicted"], st["k_out"], st["v_out"]]


def prepare(case, seed):
    d = _inputs(case, seed)
    return _prepare_own(case, d) if own else _prepare_plain(case, d)


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "found": _plain_found,
            "evict": _plain_evict}[state["case"]["op"]](state)


# ---- exact values, 64 bits ------------------------------------------------------------------------
def _exact_rows(x):
    """The values that rows [n, heads, dim] stand for once they are in 4 bits, f64."""
    x = x.double()
    n, heads, dim = x.shape
    pad = -dim % GROUP
    full = torch.nn.functional.pad(x, (0, pad)).view(n, heads, -1, GROUP)
    real = (torch.arange(dim + pad, device=x.device) < dim).view(1, 1, -1, GROUP)
    hi = full.masked_fill(~real, -math.inf).max(dim=3, keepdim=True).values
    lo = full.masked_fill(~real, math.inf).min(dim=3, keepdim=True).values
    # the format's own roundings: 32 bits, then bf16
    step = ((hi - lo).float() / 15.0).bfloat16().double()
    lo = lo.float().bfloat16().double()
    code = torch.zeros_like(full)
    ok = (step != 0).expand_as(full)
    code[ok] = ((full - lo) / step)[ok].round().clamp(0.0, 15.0)
    return (lo + step * code).float().double().view(n, heads, dim + pad)[:, :, :dim]


def exact(case, seed):
    d = _inputs(case, seed)
    rows, new, held, cap = d["rows"], d["new"], d["held"], d["capacity"]
    heads, dim = case["heads"], case["dim"]
    if case["op"] == "append":
        w = torch.ones(case["n_seqs"], cap, dtype=torch.float64, device="cuda")
        for s, (r, n) in enumerate(zip(rows, new)):
            w[s, r:r + n] = 0.0
        return [_exact_rows(d["keys"]), _exact_rows(d["values"]), w]
    if case["op"] == "evict":
        length, w_out, ids_out, evicted, ko, vo = [], torch.zeros(case["n_seqs"], cap, dtype=torch.float64), \
            torch.zeros(case["n_seqs"], cap, dtype=torch.int64), \
            torch.full((case["n_seqs"], cap), -1, dtype=torch.int64), [], []
        w_host, id_host, protect = d["w_in"].double().cpu(), d["ids"].cpu(), d["protect"].cpu()
        first = 0
        for s, r in enumerate(rows):
            w, ids = w_host[s, :r].tolist(), id_host[s, :r].tolist()
            rank = [math.inf if i >= int(protect[s]) or x != x else x for x, i in zip(w, ids)]
            order = sorted(range(r), key=lambda j: (-rank[j], j))
            m = min(r, case["keep"])
            kept = set(order[:m])
            movers = iter(sorted(j for j in kept if j >= m))
            at = [j if j in kept else next(movers) for j in range(m)]
            gone = [ids[j] for j in range(r) if j not in kept]
            length.append(m)
            w_out[s, :m] = w_host[s, at]
            ids_out[s, :m] = id_host[s, at]
            evicted[s, :len(gone)] = torch.tensor(gone, dtype=torch.int64)
            idx = torch.tensor(at, dtype=torch.int64, device="cuda") + first
            ko.append(_exact_rows(d["keys"][idx]))
            vo.append(_exact_rows(d["values"][idx]))
            first += r
        return [torch.tensor(length, dtype=torch.int32, device="cuda"), w_out.cuda(), ids_out.cuda(), evicted.cuda(),
                torch.cat(ko), torch.cat(vo)]
    hq = heads * case["group"]
    out = torch.zeros(sum(new), hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(sum(new), hq, dtype=torch.float64, device="cuda")
    weights = torch.zeros(sum(new), case["k"], dtype=torch.float64, device="cuda") if case["op"] == "found" else None
    w_out = torch.zeros_like(d["w_in"], dtype=torch.float64) if "w_in" in d else None
    first, tok = 0, 0
    for s in range(case["n_seqs"]):
        keys, values = d["keys"][first:first + held[s]], d["values"][first:first + held[s]]
        first += held[s]
        if w_out is not None:
            w_out[s, :held[s]] = d["decay"] * d["w_in"][s, :held[s]].double()
        if case["op"] == "attend" and new[s] == 0:
            continue
        for h in range(heads):
            part = slice(h * case["group"], (h + 1) * case["group"])
            k, v = _exact_rows(keys[:, h:h + 1])[:, 0], _exact_rows(values[:, h:h + 1])[:, 0]
            if case["op"] == "attend":
                for t0 in range(0, new[s], 64):
                    t1 = min(t0 + 64, new[s])
                    q = d["q"][tok + t0:tok + t1, part].double()
                    z = torch.einsum("tgd,rd->tgr", q, k) * d["scale"]
                    for t in range(t0, t1):
                        z[t - t0, :, rows[s] + t + 1:] = -math.inf
                    l = torch.logsumexp(z, dim=2)
                    p = torch.exp(z - l[..., None])
                    out[tok + t0:tok + t1, part] = torch.einsum("tgr,rd->tgd", p, v)
                    lse[tok + t0:tok + t1, part] = l
                    if w_out is not None:
                        w_out[s, :held[s]] += p.sum(dim=(0, 1))
            else:
                for t0 in range(0, new[s], 128):
                    t1 = min(t0 + 128, new[s])
                    ids = d["lists"][tok + t0:tok + t1]
                    use = (ids >= 0) & (ids < rows[s])
                    at = ids.clamp(0, max(rows[s] - 1, 0))
                    if rows[s] == 0:
                        lse[tok + t0:tok + t1, part] = -math.inf
                        continue
                    z = torch.einsum("tgd,tkd->tgk", d["q"][tok + t0:tok + t1, part].double(), k[at]) * d["scale"]
                    z = z.masked_fill(~use[:, None], -math.inf)
                    l = torch.logsumexp(z, dim=2)
                    p = torch.exp(z - torch.where(l == -math.inf, 0.0, l)[..., None])
                    out[tok + t0:tok + t1, part] = torch.einsum("tgk,tkd->tgd", p, v[at])
                    lse[tok + t0:tok + t1, part] = l
                    weights[tok + t0:tok + t1] += p.sum(dim=1)
        tok += new[s]
    return [out, lse] + ([weights] if case["op"] == "found" else []) + ([w_out] if w_out is not None else [])
