"""Step planning and the rotated store into pages on the GPU, against plain forms (attn_reference.py)."""
from __future__ import annotations

import random

import numpy as np
import pytest

import edgeforge_b200 as efg
from attn_reference import EPS, plan, rotate

pytestmark = pytest.mark.gpu


def _t(torch, a, dtype=None):
    return torch.tensor(np.asarray(a), dtype=dtype or torch.int32, device="cuda")


def _plan(torch, cached, new, table, free, pool, ps, n_rows):
    n = len(new)
    st = {"table": _t(torch, np.asarray(table, np.int32)), "slots": _t(torch, [7] * n_rows), "positions": _t(torch, [7] * n_rows),
          "cu": _t(torch, [7] * (n + 1)), "kv_len": _t(torch, [7] * n), "taken": _t(torch, [7])}
    efg.page_plan(st["table"], st["slots"], st["positions"], st["cu"], st["kv_len"], st["taken"], _t(torch, cached),
                  _t(torch, new), _t(torch, free), pool, ps)
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in st.items()}


def _setting(r, n, longest, context, ps, spare=2):
    cached = [r.randint(0, context) for _ in range(n)]
    new = [r.choice([0, 1, r.randint(0, longest)]) for _ in range(n)]
    have = [-(-c // ps) for c in cached]
    held = [-(-(c + m) // ps) for c, m in zip(cached, new)]
    pool = sum(held) + spare
    order = r.sample(range(pool), pool)
    table = np.full((n, max([1] + held)), -1, np.int32)
    at = 0
    for s in range(n):
        table[s, : have[s]] = order[at : at + have[s]]
        at += have[s]
    return cached, new, table, order[at:], pool


@pytest.mark.parametrize("n,longest,context,ps,pad", [(1, 1, 0, 16, 0), (8, 1, 500, 16, 0), (3, 200, 40, 16, 9),
                                                      (511, 3, 70, 1, 1), (512, 40, 7, 32, 0), (513, 5, 90, 64, 600),
                                                      (1500, 300, 300, 16, 5), (2, 5000, 3, 128, 0), (5, 0, 33, 16, 4), (2047, 2, 20, 16, 0),
                                                      (2048, 3, 40, 8, 3), (2049, 9, 9, 16, 0), (5000, 4, 100, 32, 1)])
def test_plan(cuda, n, longest, context, ps, pad):
    import torch

    cached, new, table, free, pool = _setting(random.Random(n + longest), n, longest, context, ps)
    want = plan(cached, new, table, free, ps, sum(new) + pad)
    got = _plan(torch, cached, new, table, free, pool, ps, sum(new) + pad)
    for k in want:
        np.testing.assert_array_equal(got[k], want[k], err_msg=k)
    assert efg.device_error() == 0


def test_plan_without_sequences_or_rows(cuda):
    import torch

    got = _plan(torch, [], [], np.zeros((0, 3)), [1, 2], 8, 16, 4)
    assert got["cu"].tolist() == [0] and got["taken"].tolist() == [0] and got["slots"].tolist() == [-1] * 4
    got = _plan(torch, [5, 0], [0, 0], [[0], [-1]], [], 8, 16, 0)
    assert got["cu"].tolist() == [0, 0, 0] and got["kv_len"].tolist() == [5, 0]
    assert efg.device_error() == 0


def test_plan_that_does_not_fit(cuda):
    """Not enough pages: served in order until one does not fit; then only those that need none."""
    import torch

    got = _plan(torch, [0, 0, 3, 16], [16, 33, 4, 16], [[-1] * 3, [-1] * 3, [5, -1, -1], [6, -1, -1]], [9, 8, 7], 10, 16, 69)
    assert efg.device_error() == 5  # EFG_ENOMEM
    assert got["cu"].tolist() == [0, 16, 49, 53, 69] and got["taken"].tolist() == [1]
    assert got["kv_len"].tolist() == [16, 0, 7, 0]
    assert got["slots"].tolist() == list(range(144, 160)) + [-1] * 33 + [83, 84, 85, 86] + [-1] * 16
    assert got["positions"].tolist() == list(range(16)) + [-1] * 33 + [3, 4, 5, 6] + [-1] * 16
    assert got["table"].tolist() == [[9, -1, -1], [-1] * 3, [5, -1, -1], [6, -1, -1]]
    assert efg.device_error() == 0  # cleared


def test_plan_with_bad_lengths_and_pages(cuda):
    import torch

    # a negative length, a table too narrow, an existing page and a free page outside the pool
    got = _plan(torch, [-1, 0, 1, 0], [2, 17, 1, 1], [[-1], [-1], [77], [-1]], [-5, 3], 10, 16, 21)
    assert efg.device_error() == 1
    assert got["cu"].tolist() == [0, 2, 19, 20, 21]
    assert got["kv_len"].tolist() == [0, 0, 2, 1] and got["slots"].tolist() == [-1] * 21
    # more rows than the caller has room for
    got = _plan(torch, [0, 0], [6, 6], [[-1], [-1]], [1, 2], 10, 16, 8)
    assert efg.device_error() == 1
    assert got["cu"].tolist() == [0, 6, 8] and got["slots"].tolist() == list(range(16, 22)) + [32, 33]


TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


@pytest.mark.parametrize("kind,cache", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows,heads,kv,dim,strided", [(1, 1, 1, 2, False), (5, 32, 4, 64, False), (37, 7, 1, 80, True),
                                                       (130, 6, 2, 30, True), (64, 8, 8, 128, True), (9, 3, 3, 256, False)])
def test_store(cuda, kind, cache, rows, heads, kv, dim, strided):
    """Rotation and store against float64. The rotation makes three FP32 roundings (two products, one
    sum; each at most 2^-24 of a term no larger than |a| + |b|), then one to the cache's type; values are
    rounded once. Rows with slot or position -1 and all other slots stay as they were."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows)
    dt, ct = getattr(torch, TYPES[kind]), getattr(torch, TYPES[cache])
    x = torch.randn(rows, heads + 2 * kv + (1 if strided else 0), dim, generator=g, device="cuda").to(dt)
    q, k, v = x[:, :heads], x[:, heads : heads + kv], x[:, heads + kv : heads + 2 * kv]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    ps, pool, far = 16, rows // 16 + 3, 300
    r = random.Random(rows)
    slots = r.sample(range(pool * ps), rows)
    pos = [r.randrange(far) for _ in range(rows)]
    if rows > 4:
        slots[1], (slots[3], pos[3]) = -1, (-1, -1)
    ang = np.arange(far)[:, None] * 0.7 ** np.arange(dim // 2)[None, :]
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    kc = torch.full((pool, ps, kv, dim), 3.0, dtype=ct, device="cuda")
    vc = torch.full((pool, ps, kv, dim), 4.0, dtype=ct, device="cuda")
    qo = torch.full((rows, heads, dim), 5.0, dtype=ct, device="cuda")
    F = torch.float32
    efg.page_store(qo, kc, vc, q, k, v, _t(torch, slots), _t(torch, pos), _t(torch, cos, F), _t(torch, sin, F))
    torch.cuda.synchronize()
    assert efg.device_error() == 0
    p = np.array(pos)
    u = EPS[cache] / 2
    D = lambda t: t.double().cpu().numpy()  # noqa: E731

    def near(got, want, mag):
        assert (np.abs(got - want) <= u * np.abs(want) + 2.0**-22 * mag + (2.0**-25 if cache == "f16" else 0)).all()

    live = p >= 0
    for src, got in ((q, D(qo)), (k, None)):
        w = rotate(D(src)[live], p[live], cos, sin)
        a = np.abs(D(src)[live])
        mag = a + np.roll(a, dim // 2, -1)
        if got is not None:
            near(got[live], w, mag)
            assert (got[~live] == 5.0).all()
        else:
            at = np.array(slots)[live]
            st = at >= 0
            flat = D(kc).reshape(-1, kv, dim)
            near(flat[at[st]], w[st], mag[st])
            rest = np.ones(len(flat), bool)
            rest[at[st]] = False
            assert (flat[rest] == 3.0).all()
            fv = D(vc).reshape(-1, kv, dim)
            np.testing.assert_array_equal(fv[at[st]], D(v.to(ct))[live][st])
            assert (fv[rest] == 4.0).all()


def test_store_in_place_without_rotation_and_bad_slots(cuda):
    import torch

    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(4, h, 64, generator=g, device="cuda") for h in (4, 2, 2))
    ang = torch.rand(8, 32, generator=g, device="cuda")
    cos, sin = ang.cos(), ang.sin()
    want, kc, vc = torch.empty_like(q), torch.zeros(2, 16, 2, 64, device="cuda"), torch.zeros(2, 16, 2, 64, device="cuda")
    slots, pos = _t(torch, [0, 1, 2, 3]), _t(torch, [0, 3, 7, 2])
    efg.page_store(want, kc, vc, q, k, v, slots, pos, cos, sin)
    mine = q.clone()
    efg.page_store(mine, kc, vc, mine, k, v, slots, pos, cos, sin)  # q_out is q
    assert torch.equal(mine, want)
    efg.page_store(None, kc, vc, None, k, v, slots, pos)  # keys and values only, as they are
    assert torch.equal(kc.view(-1, 2, 64)[:4], k) and torch.equal(vc.view(-1, 2, 64)[:4], v)
    assert efg.device_error() == 0
    before = kc.clone()
    efg.page_store(None, kc, vc, None, k, v, _t(torch, [32, -1, 2, 2**31 - 1]), pos)  # slots outside the cache
    efg.page_store(None, kc, vc, None, k, v, slots, _t(torch, [8, 8, 8, 8]), cos, sin)  # positions outside the table
    assert efg.device_error() == 1 and torch.equal(kc, before)


def test_step_runs_on_its_stream_and_in_a_graph(cuda):
    """A whole step (plan, store, attention over the pages) captured once and replayed with other
    lengths, beside the same calls made directly."""
    import torch

    n, heads, kv, dim, ps, wide = 3, 8, 2, 64, 16, 6
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = 12
    q, k, v = (torch.randn(rows, h, dim, generator=g, device="cuda") for h in (heads, kv, kv))
    ang = torch.rand(200, dim // 2, generator=g, device="cuda")
    cos, sin = ang.cos(), ang.sin()
    free = _t(torch, list(range(2, 18)))
    cached, new = _t(torch, [0, 0, 0]), _t(torch, [3, 0, 5])

    def fresh():
        return {"table": torch.full((n, wide), -1, dtype=torch.int32, device="cuda"), "slots": _t(torch, [0] * rows),
                "positions": _t(torch, [0] * rows), "cu": _t(torch, [0] * (n + 1)), "kv_len": _t(torch, [0] * n),
                "taken": _t(torch, [0]), "kc": torch.full((18, ps, kv, dim), float("nan"), device="cuda"),
                "vc": torch.full((18, ps, kv, dim), float("nan"), device="cuda"), "qo": torch.zeros_like(q),
                "out": torch.full_like(q, 9.0)}

    def step(s):
        efg.page_plan(s["table"], s["slots"], s["positions"], s["cu"], s["kv_len"], s["taken"], cached, new, free, 18, ps)
        efg.page_store(s["qo"], s["kc"], s["vc"], q, k, v, s["slots"], s["positions"], cos, sin)
        efg.attn_paged(s["out"], s["qo"], s["kc"], s["vc"], s["table"], s["cu"], s["kv_len"], 8)

    a, b = fresh(), fresh()
    step(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(b)
    graph.replay()
    torch.cuda.synchronize()
    for key in a:
        assert torch.equal(torch.nan_to_num(a[key].float(), 77), torch.nan_to_num(b[key].float(), 77)), key
    assert torch.isfinite(a["out"]).all() and (a["out"][8:] == 9.0).all()
    cached.copy_(_t(torch, [3, 0, 5]))
    new.copy_(_t(torch, [1, 4, 1]))
    free.copy_(_t(torch, list(range(4, 18)) + [0, 1]))
    step(a)
    graph.replay()
    torch.cuda.synchronize()
    for key in ("table", "slots", "kv_len", "out"):
        assert torch.equal(a[key], b[key]), key
    assert efg.device_error() == 0
