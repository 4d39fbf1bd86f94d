"""The operators of paged serving, measured: a step's block tables and slot maps (page_plan), the rotated
keys and the values of its rows into their pages (page_store), causal attention over packed prompts
(attn_prompt) and attention of new tokens over the paged cache (attn_paged).

`own` false: plain torch in 32 bits. `own` true: the calls of edgeforge_b200. Sequence lengths follow
from the case alone (a fixed draw of its numbers); every value, page order and free list from the seed.
"""
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"
ROPE_THETA = 10000.0


# ---------------------------------------------------------------- cases


def listed():
    return [
        # a decode step of 8 sequences: the smallest call, latency only
        {"name": "plan_decode_8", "op": "plan", "n": 8, "longest": 1, "context": 500, "page": 16},
        # admission of a large batch: 2048 sequences, prompts of 1 to 1024 tokens behind cached prefixes
        {"name": "plan_admit_2048", "op": "plan", "n": 2048, "longest": 1024, "context": 2048, "page": 16},
        # one layer of a 64-sequence decode step at the TinyLlama heads, everything FP32 as the decoder keeps it
        {"name": "store_decode_64_f32", "op": "store", "n": 64, "longest": 1, "context": 1800, "page": 16, "heads": 32,
         "kv_heads": 4, "dim": 64, "type": "f32", "cache": "f32"},
        # a prompt batch whose FP32 projections go into a BF16 cache
        {"name": "store_prompts_f32_bf16", "op": "store", "n": 9, "longest": 4096, "context": 0, "page": 32, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "f32", "cache": "bf16"},
        # the 23-token prompt of the decode benchmark, FP32: the smallest prompt
        {"name": "prompt_23_f32", "op": "prompt", "n": 1, "longest": 23, "heads": 32, "kv_heads": 4, "dim": 64,
         "type": "f32", "fused": False},
        # a full 2048-position prompt at the TinyLlama heads, FP32
        {"name": "prompt_2048_f32", "op": "prompt", "n": 1, "longest": 2048, "heads": 32, "kv_heads": 4, "dim": 64,
         "type": "f32", "fused": False},
        # a ragged batch of prompts packed together, q, k and v views of one projection's rows
        {"name": "prompt_ragged_bf16", "op": "prompt", "n": 24, "longest": 1777, "heads": 32, "kv_heads": 4, "dim": 64,
         "type": "bf16", "fused": True},
        # one long prompt, wide heads
        {"name": "prompt_8192_bf16", "op": "prompt", "n": 1, "longest": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "type": "bf16", "fused": False},
        # one layer of a 64-sequence decode step over FP32 pages
        {"name": "decode_64_f32", "op": "paged", "n": 64, "longest": 1, "context": 4000, "page": 16, "heads": 32,
         "kv_heads": 4, "dim": 64, "type": "f32", "even": False},
        # one sequence, one token, a long cache: the work is one long axis
        {"name": "decode_131072_bf16", "op": "paged", "n": 1, "longest": 1, "context": 131071, "page": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "bf16", "even": True},
        # prompts taken in chunks: 512 new tokens of four sequences over long prefixes
        {"name": "chunk_512_bf16", "op": "paged", "n": 4, "longest": 512, "context": 7680, "page": 16, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "bf16", "even": True},
        # continuous batching: single tokens beside ragged chunks, odd group of query heads
        {"name": "mixed_f16", "op": "paged", "n": 33, "longest": 301, "context": 2999, "page": 16, "heads": 28,
         "kv_heads": 4, "dim": 128, "type": "f16", "even": False},
    ]


SCORES = 8192 * 8192 * 32  # score elements of the largest listed case (the padded square)
CACHE = 131072 * 8 * 128   # elements of the longest listed key cache
ROWS = 16384 * 32 * 128    # query elements of a row batch


def _log(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return {"heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv, "dim": rng.choice([32, 64, 64, 80, 96, 128, 128])}


def draw(rng):
    op = rng.choice(["plan", "store", "prompt", "prompt", "paged", "paged", "paged"])
    while True:
        c = {"op": op, "n": _log(rng, 1, 256)}
        if op == "plan":
            c.update(n=_log(rng, 1, 4096), longest=_log(rng, 1, 1024), context=_log(rng, 1, 4096) - 1,
                     page=rng.choice([16, 32, 64, 128]))
            if c["n"] * (c["longest"] + c["context"]) <= 6000000:
                return c
            continue
        c.update(_heads(rng))
        if op == "store":
            t = rng.choice(["f32", "f16", "bf16"])
            c.update(longest=_log(rng, 1, 8192), context=_log(rng, 1, 2048) - 1, page=rng.choice([16, 32, 64, 128]),
                     type=t, cache=rng.choice([t, "f16", "bf16"]) if t == "f32" else t)
            if sum(_lengths(c)[0]) * c["heads"] * c["dim"] <= ROWS and _slots(c) * c["kv_heads"] * c["dim"] <= CACHE:
                return c
        elif op == "prompt":
            c.update(longest=_log(rng, 1, 8192), type=rng.choice(["f32", "f16", "bf16"]), fused=rng.random() < 0.5)
            lens = _lengths(c)[0]
            cost = (2 if c["type"] == "f32" else 1) * c["n"] * c["longest"] ** 2 * c["heads"]
            if cost <= SCORES and sum(lens) * c["heads"] * c["dim"] <= ROWS:
                return c
        else:
            c.update(longest=rng.choice([1, 1, _log(rng, 1, 1024)]), context=_log(rng, 1, 65536) - 1,
                     page=rng.choice([16, 32, 64, 128]), type=rng.choice(["f32", "f16", "bf16"]), even=rng.random() < 0.3)
            cost = (2 if c["type"] == "f32" else 1) * c["n"] * c["longest"] * (c["context"] + c["longest"]) * c["heads"]
            if cost <= SCORES and c["n"] * (c["context"] + c["longest"]) * c["kv_heads"] * c["dim"] <= CACHE:
                return c


def _lengths(c):
    """(new tokens, cached tokens) of every sequence: the first has the longest of both; the others are spread over
    the logarithm, single tokens and (from four sequences on) one empty sequence among them."""
    r = random.Random("%d %d %d" % (c["n"], c["longest"], c.get("context", 0)))
    new, cached = [c["longest"]], [c.get("context", 0)]
    for i in range(1, c["n"]):
        if c.get("even"):
            new.append(c["longest"])
            cached.append(c["context"])
            continue
        single = c["op"] == "paged" and r.random() < 0.6
        new.append(1 if single or c["longest"] == 1 else _log(r, 1, c["longest"]))
        cached.append(_log(r, 1, c.get("context", 0) + 1) - 1 if r.random() < 0.5 else r.randint(0, c.get("context", 0)))
    if c["n"] >= 4 and c["longest"] > 1 and not c.get("even"):
        new[2] = 0
    return new, cached


def _pages(c):
    """Pages of every sequence before and after the step."""
    new, cached = _lengths(c)
    p = c["page"]
    return [(k + p - 1) // p for k in cached], [(k + m + p - 1) // p for k, m in zip(cached, new)]


def _slots(c):
    return (sum(_pages(c)[1]) + 3) * c["page"]


def _pad(c):
    """Rows behind the last sequence: a batch padded to a round size, as a captured step is."""
    return 5 if c["n"] % 2 and c["n"] > 1 else 0


def work(c):
    new, cached = _lengths(c)
    rows = sum(new)
    if c["op"] == "plan":
        before, after = _pages(c)
        fresh = sum(after) - sum(before)
        return {"bytes": 8 * c["n"] + 8 * fresh + 4 * c["n"] + 8 * (rows + _pad(c)) + 8 * c["n"], "flops": 0}
    h, kv, d, es = c["heads"], c["kv_heads"], c["dim"], BYTES[c["type"]]
    if c["op"] == "store":
        es2 = BYTES[c["cache"]]
        return {"bytes": rows * (h + 2 * kv) * d * (es + es2) + rows * (8 + 4 * d), "flops": rows * (h + kv) * d * 3}
    if c["op"] == "prompt":
        return {"bytes": rows * (2 * h + 2 * kv) * d * es, "flops": 4 * d * h * sum(m * (m + 1) // 2 for m in new)}
    seen = sum(m * k + m * (m + 1) // 2 for m, k in zip(new, cached))
    held = sum(m + k for m, k in zip(new, cached) if m)
    return {"bytes": rows * 2 * h * d * es + held * 2 * kv * d * es, "flops": 4 * d * h * seen}


# ---------------------------------------------------------------- what a program has in hand


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _table(c, gen, pages):
    """Block tables over a shuffled pool: (table [n, widest], the pages nobody holds, pool size)."""
    after = _pages(c)[1]
    pool = sum(after) + 3
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((c["n"], max(1, max(after))), -1, dtype=torch.int32, device=DEV)
    held = torch.tensor(pages, device=DEV)
    table[torch.arange(table.shape[1], device=DEV)[None, :] < held[:, None]] = order[: sum(pages)]
    return table, order[sum(pages):].contiguous(), pool


def prepare(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    new, cached = _lengths(c)
    rows, pad = sum(new), _pad(c)
    s = {"case": c}
    if c["op"] == "plan":
        table, free, pool = _table(c, gen, _pages(c)[0])
        s.update(table=table, free=free, pool=pool, cached=_int(cached), new=_int(new))
        s.update(slots=_int([0] * (rows + pad)), positions=_int([0] * (rows + pad)), cu=_int([0] * (c["n"] + 1)),
                 kv_len=_int([0] * c["n"]), taken=_int([0]))
        return s
    h, kv, d, t = c["heads"], c["kv_heads"], c["dim"], TYPES[c["type"]]

    def values(*shape, dtype=t, scale=1.0):
        return torch.randn(*shape, generator=gen, device=DEV).mul_(scale).to(dtype)

    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    s["cu"] = _int(cu)
    if c["op"] == "store":
        table, _, pool = _table(c, gen, _pages(c)[1])
        pos = torch.cat([torch.arange(k, k + m) for m, k in zip(new, cached)] + [torch.full((pad,), -1)]).to(DEV)
        seq = torch.repeat_interleave(torch.arange(c["n"]), torch.tensor(new)).to(DEV)
        slots = torch.full((rows + pad,), -1, dtype=torch.int32, device=DEV)
        p = c["page"]
        slots[:rows] = table[seq, pos[:rows] // p] * p + (pos[:rows] % p).to(torch.int32)
        ct = TYPES[c["cache"]]
        far = max(k + m for m, k in zip(new, cached))
        angle = torch.arange(far, device=DEV, dtype=torch.float64)[:, None] * ROPE_THETA ** (
            -torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        s.update(q=values(rows + pad, h, d), k=values(rows + pad, kv, d), v=values(rows + pad, kv, d), slots=slots,
                 positions=pos.to(torch.int32), cos=angle.cos().float().contiguous(), sin=angle.sin().float().contiguous(),
                 k_cache=torch.zeros(pool, p, kv, d, dtype=ct, device=DEV),
                 v_cache=torch.zeros(pool, p, kv, d, dtype=ct, device=DEV),
                 q_out=torch.zeros(rows + pad, h, d, dtype=ct, device=DEV))
        return s
    out = torch.zeros(rows + pad, h, d, dtype=t, device=DEV)
    if c["op"] == "prompt":
        if c["fused"]:
            x = values(rows + pad, h + 2 * kv, d)
            x[:, :h] *= 2
            q, k, v = x[:, :h], x[:, h : h + kv], x[:, h + kv :]
        else:
            q, k, v = values(rows + pad, h, d, scale=2.0), values(rows + pad, kv, d), values(rows + pad, kv, d)
        s.update(q=q, k=k, v=v, out=out)
        return s
    table, _, pool = _table(c, gen, _pages(c)[1])
    s.update(q=values(rows + pad, h, d, scale=2.0), k_cache=values(pool, c["page"], kv, d),
             v_cache=values(pool, c["page"], kv, d), table=table, kv_len=_int([m + k for m, k in zip(new, cached)]), out=out)
    return s


# ---------------------------------------------------------------- one pass


def run(s):
    return {"plan": _plan, "store": _store, "prompt": _prompt, "paged": _paged}[s["case"]["op"]](s)


def _plan(s):
    p = s["case"]["page"]
    if own:
        import edgeforge_b200 as efg

        efg.page_plan(s["table"], s["slots"], s["positions"], s["cu"], s["kv_len"], s["taken"], s["cached"], s["new"],
                      s["free"], s["pool"], p)
        return {k: s[k] for k in ("table", "slots", "positions", "cu", "kv_len", "taken")}
    table, cached, new = s["table"].long(), s["cached"].long(), s["new"].long()
    have, held = (cached + p - 1) // p, (cached + new + p - 1) // p
    need = held - have
    first = need.cumsum(0) - need
    free = s["free"].long()
    j = torch.arange(table.shape[1], device=DEV)[None, :]
    fresh = free[(first[:, None] + j - have[:, None]).clamp(0, free.numel() - 1)]
    table = torch.where((j >= have[:, None]) & (j < held[:, None]), fresh, table)
    ends = new.cumsum(0)
    row = torch.arange(s["slots"].numel(), device=DEV)
    live = row < ends[-1]
    seq = torch.searchsorted(ends, row, right=True).clamp(max=ends.numel() - 1)
    pos = cached[seq] + row - (ends - new)[seq]
    slot = table[seq, (pos // p).clamp(0, table.shape[1] - 1)] * p + pos % p
    out = {"table": table, "slots": torch.where(live, slot, -1), "positions": torch.where(live, pos, -1),
           "cu": torch.cat([torch.zeros_like(ends[:1]), ends]), "kv_len": cached + new, "taken": need.sum()[None]}
    return {k: v.to(torch.int32) for k, v in out.items()}


def _store(s):
    if own:
        import edgeforge_b200 as efg

        efg.page_store(s["q_out"], s["k_cache"], s["v_cache"], s["q"], s["k"], s["v"], s["slots"], s["positions"], s["cos"],
                       s["sin"])
        return [s["q_out"], s["k_cache"], s["v_cache"]]
    slots, pos, kc, vc = s["slots"].long(), s["positions"].long(), s["k_cache"], s["v_cache"]
    live = slots >= 0
    a = s["q"].shape[2] // 2
    cos, sin = s["cos"][pos.clamp(min=0)][:, None, :], s["sin"][pos.clamp(min=0)][:, None, :]

    def turn(x):
        x = x.float()
        return torch.cat([x[..., :a] * cos - x[..., a:] * sin, x[..., a:] * cos + x[..., :a] * sin], -1).to(kc.dtype)

    # a padding row writes what the first row writes, to the first row's slot
    at = torch.where(live, slots, slots[0])
    pick = lambda x: torch.where(live[:, None, None], x, x[:1])  # noqa: E731
    kc.view(-1, *kc.shape[2:])[at] = pick(turn(s["k"]))
    vc.view(-1, *vc.shape[2:])[at] = pick(s["v"].to(vc.dtype))
    return [torch.where(live[:, None, None], turn(s["q"]), s["q_out"]), kc, vc]


def _softmax_product(q, k, v, seen):
    """q [n, l, kv, g, d], k and v [n, s, kv, d], seen [n, l, s]: the weighted values; zeros where a row sees nothing."""
    score = torch.einsum("nlkgd,nskd->nkgls", q, k) * q.shape[-1] ** -0.5
    score = torch.where(seen[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.einsum("nkgls,nskd->nlkgd", e / torch.where(total == 0, 1.0, total), v)


def _by_sequence(cu, longest, rows):
    """Row of every (sequence, step), and the sequence and step of every row."""
    step = torch.arange(longest, device=DEV)
    at = (cu[:-1, None] + step[None, :]).clamp(max=rows - 1)
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return step, at, row, seq.clamp(max=cu.numel() - 2)


def _unpack(o, cu, row, seq, out):
    o = o.flatten(2, 3)[seq, (row - cu[seq]).clamp(0, o.shape[1] - 1)].to(out.dtype)
    return torch.where((row < cu[-1])[:, None, None], o, out)


def _prompt(s):
    if own:
        import edgeforge_b200 as efg

        efg.attn_prompt(s["out"], s["q"], s["k"], s["v"], s["cu"])
        return s["out"]
    c, cu = s["case"], s["cu"].long()
    step, at, row, seq = _by_sequence(cu, c["longest"], s["q"].shape[0])
    length = cu[1:] - cu[:-1]
    seen = (step[None, :, None] >= step[None, None, :]) & (step < length[:, None])[:, None, :]
    q = s["q"].float()[at].unflatten(2, (c["kv_heads"], -1))
    return _unpack(_softmax_product(q, s["k"].float()[at], s["v"].float()[at], seen), cu, row, seq, s["out"])


def _paged(s):
    c = s["case"]
    if own:
        import edgeforge_b200 as efg

        efg.attn_paged(s["out"], s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["kv_len"], c["longest"])
        return s["out"]
    cu, kv_len, table = s["cu"].long(), s["kv_len"].long(), s["table"].long().clamp(min=0)
    step, at, row, seq = _by_sequence(cu, c["longest"], s["q"].shape[0])
    k, v = (x[table].flatten(1, 2).float() for x in (s["k_cache"], s["v_cache"]))
    pos = (kv_len - (cu[1:] - cu[:-1]))[:, None] + step[None, :]
    place = torch.arange(k.shape[1], device=DEV)
    seen = (place <= pos[:, :, None]) & (place < kv_len[:, None, None])
    q = s["q"].float()[at].unflatten(2, (c["kv_heads"], -1))
    return _unpack(_softmax_product(q, k, v, seen), cu, row, seq, s["out"])


# ---------------------------------------------------------------- from the definitions, in 64 bits


def exact(c, seed):
    if c["op"] == "plan":
        return None
    s = prepare(c, seed)
    new, cached = _lengths(c)
    if c["op"] == "store":
        p, a = c["page"], c["dim"] // 2
        q_out, kc, vc = s["q_out"].double(), s["k_cache"].double().flatten(0, 1), s["v_cache"].double().flatten(0, 1)
        rows = sum(new)
        where, pos = s["slots"][:rows].long(), s["positions"][:rows].long()
        phase = torch.complex(s["cos"].double()[pos], s["sin"].double()[pos])[:, None, :]
        for x, to, at in ((s["q"], q_out, torch.arange(rows, device=DEV)), (s["k"], kc, where)):
            x = x[:rows].double()
            z = torch.complex(x[..., :a], x[..., a:]) * phase
            to[at, :, :a], to[at, :, a:] = z.real, z.imag
        vc[where] = s["v"][:rows].double()
        return [q_out, kc.unflatten(0, (-1, p)), vc.unflatten(0, (-1, p))]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    g = h // kv
    out = s["out"].double()
    t0 = 0
    for i, m in enumerate(new):
        if m == 0:
            continue
        if c["op"] == "prompt":
            n, k, v = m, s["k"][t0 : t0 + m], s["v"][t0 : t0 + m]
        else:
            n = m + cached[i]
            pages = s["table"][i, : -(-n // c["page"])].long()
            k, v = (x[pages].flatten(0, 1)[:n] for x in (s["k_cache"], s["v_cache"]))
        k, v = k.double().transpose(0, 1), v.double().transpose(0, 1)
        hide = torch.ones(m, n, dtype=torch.bool, device=DEV).triu(n - m + 1)
        for j in range(h):
            w = s["q"][t0 : t0 + m, j].double() @ k[j // g].T / d**0.5
            w.masked_fill_(hide, float("-inf"))
            out[t0 : t0 + m, j] = torch.softmax(w, -1) @ v[j // g]
        t0 += m
    return out
