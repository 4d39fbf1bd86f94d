"""Attention over packed prompts and over the paged cache on the GPU, against float64 (attn_reference.py
states the error that is allowed and why)."""
from __future__ import annotations

import random

import numpy as np
import pytest

import edgeforge_b200 as efg
from attn_reference import attend, tolerance

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
KINDS = list(TYPES)


def _i(torch, a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _d(t):
    return t.double().cpu().numpy()


def _cu(lens):
    return [0] + np.cumsum(lens).tolist()


def _held(kind, got, *expected):
    want, tol = expected[0], tolerance(kind, *expected)
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), float(off.max()))


def _prompt(torch, kind, lens, heads, kv, dim, pad=0, strided=False, seed=0, scale=None, qscale=1.0):
    dt = getattr(torch, TYPES[kind])
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(lens) + pad
    if strided:
        x = torch.randn(rows, heads + 2 * kv, dim, generator=g, device="cuda").to(dt)
        q, k, v = x[:, :heads], x[:, heads : heads + kv], x[:, heads + kv :]
    else:
        q, k, v = (torch.randn(rows, h, dim, generator=g, device="cuda").to(dt) for h in (heads, kv, kv))
    q = q * qscale if qscale != 1 else q
    out = torch.full((rows, heads, dim), 7.0, dtype=dt, device="cuda")
    efg.attn_prompt(out, q, k, v, _i(torch, _cu(lens)), scale=scale)
    torch.cuda.synchronize()
    return q, k, v, out


def _check_prompt(kind, lens, q, k, v, out, scale=None):
    scale = scale if scale is not None else float(np.float32(q.shape[2] ** -0.5))
    Q, K, V, O = _d(q), _d(k), _d(v), _d(out)
    for a, b in zip(_cu(lens)[:-1], _cu(lens)[1:]):
        if b > a:
            _held(kind, O[a:b], *attend(Q[a:b], K[a:b], V[a:b], scale))
    assert (O[_cu(lens)[-1]:] == 7.0).all()
    assert efg.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,heads,kv,dim", [
    ([1], 4, 4, 64), ([23], 32, 4, 64), ([130], 2, 1, 128), ([300], 8, 1, 64), ([129, 1, 0, 64, 255, 0], 4, 2, 64),
    ([2, 3, 1, 1, 5], 14, 2, 128), ([257], 3, 1, 80), ([96, 200], 6, 2, 32), ([70], 5, 5, 96), ([33], 12, 1, 16),
    ([65, 5], 2, 2, 256), ([40], 3, 3, 20), ([50, 9], 2, 1, 7), ([17], 40, 1, 64), ([128, 128], 16, 2, 128),
    ([9], 130, 1, 64), ([200], 7, 1, 8)])
def test_prompt(cuda, kind, lens, heads, kv, dim):
    import torch

    q, k, v, out = _prompt(torch, kind, lens, heads, kv, dim)
    _check_prompt(kind, lens, q, k, v, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_long(cuda, kind, dim):
    import torch

    lens = [700, 1, 515]
    q, k, v, out = _prompt(torch, kind, lens, 4, 2, dim, pad=3, seed=2)
    _check_prompt(kind, lens, q, k, v, out)


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_strided_padded_and_scaled(cuda, kind):
    import torch

    lens = [150, 0, 31]
    q, k, v, out = _prompt(torch, kind, lens, 4, 2, 64, pad=6, strided=True, seed=3, scale=0.3)
    _check_prompt(kind, lens, q, k, v, out, scale=float(np.float32(0.3)))
    q, k, v, out = _prompt(torch, kind, lens, 4, 2, 64, seed=4, scale=-0.2)
    _check_prompt(kind, lens, q, k, v, out, scale=float(np.float32(-0.2)))
    q, k, v, out = _prompt(torch, kind, lens, 4, 2, 64, seed=4, scale=0.0)  # every visible key the same weight
    _check_prompt(kind, lens, q, k, v, out, scale=0.0)


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_with_large_scores(cuda, kind):
    """Scores of several hundred: the softmax is close to one key, the running maximum moves often."""
    import torch

    lens = [260]
    q, k, v, out = _prompt(torch, kind, lens, 4, 2, 64, seed=5, qscale=64.0)
    _check_prompt(kind, lens, q, k, v, out)


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_rising_scores(cuda, kind):
    """Keys whose scores rise along the sequence, so that every block of keys has a new maximum."""
    import torch

    dt = getattr(torch, TYPES[kind])
    n, dim = 600, 64
    q = torch.ones(n, 2, dim, device="cuda", dtype=dt)
    k = (torch.arange(n, device="cuda")[:, None, None] / 16 * torch.ones(1, 1, dim, device="cuda")).to(dt)
    v = torch.randn(n, 1, dim, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda").to(dt)
    out = torch.full((n, 2, dim), 7.0, dtype=dt, device="cuda")
    efg.attn_prompt(out, q, k, v, _i(torch, [0, n]))
    _check_prompt(kind, [n], q, k, v, out)
    k = k.flip(0).contiguous()
    efg.attn_prompt(out, q, k, v, _i(torch, [0, n]))
    _check_prompt(kind, [n], q, k, v, out)


def test_prompt_f32_over_wide_ranges(cuda):
    """F32 keeps FP32 accuracy for magnitudes that 16-bit parts cannot hold by themselves."""
    import torch

    for a, b in ((1e-6, 1e6), (1e5, 1e-5), (1.0, 1e-20), (1.0, 1e20), (1e-3, 1.0)):
        lens = [140, 9]
        g = torch.Generator(device="cuda").manual_seed(9)
        q, k, v = (torch.randn(149, h, 64, generator=g, device="cuda") for h in (4, 2, 2))
        spread = torch.exp(2 * torch.randn(149, 1, 1, generator=g, device="cuda"))  # rows of different sizes
        q, k, v = q / a, k * a * spread.clamp(max=4), v * b * spread
        out = torch.full_like(q, 7.0)
        efg.attn_prompt(out, q, k, v, _i(torch, _cu(lens)))
        _check_prompt("f32", lens, q, k, v, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_masked_places_do_not_reach_rows(cuda, kind, bad, dim):
    """NaN and infinities in the next sequence's keys and values, in the padding, and in the sequence's
    own later positions leave the rows before them as they are without them."""
    import torch

    dt = getattr(torch, TYPES[kind])
    g = torch.Generator(device="cuda").manual_seed(7)
    lens, rows = [37, 150, 60], 255
    q, k, v = (torch.randn(rows, h, dim, generator=g, device="cuda").to(dt) for h in (4, 2, 2))
    cu = _i(torch, _cu(lens))
    clean, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    efg.attn_prompt(clean, q, k, v, cu)
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    for t in (k2, v2):
        t[100:187] = bad  # from position 63 of the second sequence on
        t[247:] = bad     # padding
    q2[247:] = bad
    efg.attn_prompt(out, q2, k2, v2, cu)
    keep = list(range(100)) + list(range(187, 247))
    Q, K, V, O = _d(q), _d(k), _d(v), _d(out)
    for a, b in ((0, 37), (37, 100), (187, 247)):
        _held(kind, O[a:b], *attend(Q[a:b], K[a:b], V[a:b], float(np.float32(dim**-0.5))))
    assert torch.isfinite(out[keep]).all() and (out[247:] == 7.0).all()
    # rows that see a NaN or an infinite value are not finite
    assert not torch.isfinite(out[101:187]).all(-1).any() or bad == float("-inf")
    assert efg.device_error() == 0


def test_prompt_bad_offsets(cuda):
    """Offsets that make no sense are recorded and read nothing out of range."""
    import torch

    q = torch.randn(20, 2, 64, device="cuda")
    for cu in ([0, 30], [-5, 10], [0, 12, 8, 20], [2**31 - 1, -(2**31), 7]):
        out = torch.full_like(q, 7.0)
        efg.attn_prompt(out, q, q, q, _i(torch, cu))
        torch.cuda.synchronize()
        assert efg.device_error() == 1, cu


def _paged(torch, kind, chunks, heads, kv, dim, ps, seed=0, stale=float("nan"), pad=0, max_new=None, wide=0):
    """chunks: (new, kv_len) per sequence. Pages are shuffled; everything outside the visible positions is
    `stale`. Returns what the call gave and, per sequence, its keys and values."""
    dt = getattr(torch, TYPES[kind])
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    pages = [-(-n // ps) for _, n in chunks]
    pool = sum(pages) + 3
    order = r.sample(range(pool), pool)
    table = np.full((len(chunks), max(pages + [1]) + wide), -1, np.int32)
    kc, vc = (torch.full((pool, ps, kv, dim), stale, dtype=dt, device="cuda") for _ in range(2))
    seqs, at = [], 0
    for s, (m, n) in enumerate(chunks):
        own = order[at : at + pages[s]]
        at += pages[s]
        table[s, : pages[s]] = own
        k, v = (torch.randn(n, kv, dim, generator=g, device="cuda").to(dt) for _ in range(2))
        seqs.append((k, v))
        if n:
            slots = torch.tensor([own[j // ps] * ps + j % ps for j in range(n)], device="cuda")
            kc.view(-1, kv, dim)[slots], vc.view(-1, kv, dim)[slots] = k, v
    lens = [m for m, _ in chunks]
    q = torch.randn(sum(lens) + pad, heads, dim, generator=g, device="cuda").to(dt)
    out = torch.full_like(q, 7.0)
    args = (q, kc, vc, _i(torch, table.tolist()), _i(torch, _cu(lens)), _i(torch, [n for _, n in chunks]))
    efg.attn_paged(out, *args, max_new if max_new is not None else max(lens))
    torch.cuda.synchronize()
    return q, seqs, out, args


def _check_paged(kind, chunks, q, seqs, out):
    scale = float(np.float32(q.shape[2] ** -0.5))
    Q, O, a = _d(q), _d(out), 0
    for (m, n), (k, v) in zip(chunks, seqs):
        if m:
            _held(kind, O[a : a + m], *attend(Q[a : a + m], _d(k), _d(v), scale))
        a += m
    assert (O[a:] == 7.0).all()
    assert efg.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("chunks,heads,kv,dim,ps", [
    ([(1, 1)], 4, 4, 64, 16), ([(1, 17), (1, 300), (0, 5), (1, 0), (1, 64)], 32, 4, 64, 16),
    ([(1, 700)], 8, 1, 128, 64), ([(1, 130), (1, 129)], 14, 2, 128, 32), ([(1, 33)], 3, 3, 80, 16),
    ([(1, 100), (1, 5)], 17, 1, 64, 16), ([(1, 50)], 6, 2, 32, 1), ([(1, 90)], 4, 2, 96, 128), ([(1, 1000)] * 3, 2, 2, 64, 16),
    ([(1, 40)], 2, 1, 256, 8), ([(1, 31), (1, 2)], 3, 1, 7, 5), ([(1, 65)], 64, 1, 64, 256)])
def test_decode(cuda, kind, chunks, heads, kv, dim, ps):
    import torch

    q, seqs, out, _ = _paged(torch, kind, chunks, heads, kv, dim, ps)
    _check_paged(kind, chunks, q, seqs, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_long(cuda, kind, dim):
    """A long axis split over many workers, joined into one row."""
    import torch

    chunks = [(1, 9001), (1, 4096), (1, 1)]
    q, seqs, out, args = _paged(torch, kind, chunks, 8, 2, dim, 64, seed=1, pad=2)
    _check_paged(kind, chunks, q, seqs, out)
    again = torch.full_like(out, 7.0)
    efg.attn_paged(again, *args, 1)
    assert torch.equal(out, again)  # the same bits on every call


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("chunks,heads,kv,dim,ps", [
    ([(5, 5)], 4, 2, 64, 16), ([(130, 400), (1, 77), (0, 9), (64, 64)], 8, 2, 64, 16),
    ([(3, 260), (2, 2)], 14, 2, 128, 32), ([(100, 333)], 3, 1, 80, 64), ([(17, 1000)], 16, 1, 128, 16),
    ([(33, 40), (12, 200)], 6, 2, 96, 128), ([(9, 30)], 2, 1, 256, 16), ([(7, 20)], 3, 3, 20, 4),
    ([(40, 300), (1, 1)], 7, 7, 64, 256), ([(129, 129)], 1, 1, 128, 16), ([(2, 500), (1, 300)], 8, 4, 64, 16)])
def test_chunks(cuda, kind, chunks, heads, kv, dim, ps):
    import torch

    q, seqs, out, _ = _paged(torch, kind, chunks, heads, kv, dim, ps, pad=3, wide=2)
    _check_paged(kind, chunks, q, seqs, out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("stale", [float("nan"), float("inf"), 0.0])
def test_chunk_longer_than_its_cache_has_empty_rows(cuda, kind, stale):
    """Rows before the first position see nothing: zeros."""
    import torch

    chunks = [(20, 7), (5, 0), (3, 3)]
    q, seqs, out, _ = _paged(torch, kind, chunks, 4, 2, 64, 16, stale=stale)
    assert (out[:13] == 0).all() and (out[20:25] == 0).all()
    _check_paged(kind, chunks, q, seqs, out)


@pytest.mark.parametrize("kind", KINDS)
def test_chunk_with_infinite_later_positions(cuda, kind):
    """A chunk's rows are not reached by NaN or infinite keys and values of its later positions."""
    import torch

    chunks = [(40, 200)]
    q, seqs, out, args = _paged(torch, kind, chunks, 4, 2, 64, 16, seed=8)
    k, v = seqs[0]
    _, kc, vc, table, _, _ = args
    for bad in (float("nan"), float("inf")):
        for j in range(180, 200):
            page = int(table[0, j // 16])
            kc[page, j % 16], vc[page, j % 16] = bad, bad
        out2 = torch.full_like(out, 7.0)
        efg.attn_paged(out2, *args, 40)
        expected = attend(_d(q), _d(k), _d(v), float(np.float32(64**-0.5)))
        _held(kind, _d(out2)[:20], *(e[:20] for e in expected))
        assert not torch.isfinite(out2[20:]).any()
    assert efg.device_error() == 0


def test_shared_pages_and_one_pool_for_keys_and_values(cuda):
    """Two sequences whose tables share their prefix pages, and one tensor as both caches."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(4)
    pool = torch.randn(6, 16, 2, 64, generator=g, device="cuda")
    q = torch.randn(2, 4, 64, generator=g, device="cuda")
    table, kv_len, cu = _i(torch, [[4, 1, 3], [4, 1, 0]]), _i(torch, [40, 35]), _i(torch, [0, 1, 2])
    out = torch.empty_like(q)
    efg.attn_paged(out, q, pool, pool, table, cu, kv_len, 1)
    for s in range(2):
        rows = _d(pool[table[s].long()].flatten(0, 1))[: int(kv_len[s])]
        _held("f32", _d(out)[s : s + 1], *attend(_d(q)[s : s + 1], rows, rows, float(np.float32(64**-0.5))))
    assert efg.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 50])
def test_bad_pages_lengths_and_chunks_are_recorded(cuda, kind, m):
    """Page ids outside the pool, lengths that pass the table and chunks longer than max_new: an error word,
    no access out of range, and the other sequences right."""
    import torch

    chunks = [(m, 200), (m, 90), (m, 61)]
    q, seqs, out, args = _paged(torch, kind, chunks, 4, 2, 64, 16, seed=11)
    _check_paged(kind, chunks, q, seqs, out)
    q, kc, vc, table, cu, kv_len = args
    good = out.clone()

    def _check_rows(o, which):
        for s in which:
            k, v = seqs[s]
            want = attend(_d(q[m * s : m * s + m]), _d(k), _d(v), float(np.float32(64**-0.5)))
            _held(kind, _d(o)[m * s : m * s + m], *want)

    def again(table=table, cu=cu, kv_len=kv_len, max_new=m):
        o = torch.full_like(out, 7.0)
        efg.attn_paged(o, q, kc, vc, table, cu, kv_len, max_new)
        torch.cuda.synchronize()
        assert efg.device_error() == 1
        return o

    for page in (-1, 10**6, 2**31 - 1, -(2**31)):
        t = table.clone()
        t[1, 2] = page
        o = again(table=t)
        assert torch.equal(o[:m], good[:m]) and torch.equal(o[2 * m :], good[2 * m :])
    for n in (-3, 10**6, 2**31 - 1):
        l = kv_len.clone()
        l[0] = n
        # (the work is cut up differently without the first sequence: the same values, not the same bits)
        _check_rows(again(kv_len=l), (1, 2))
    if m > 1:
        again(max_new=m - 1)
    again(cu=_i(torch, [0, m, 5 * m, 3 * m]))


@pytest.mark.parametrize("big", [1e4, 1e8, 1e30])
@pytest.mark.parametrize("paged", [False, True])
def test_f32_outliers_take_no_digits_from_other_rows(cuda, big, paged):
    """Huge finite keys and values at positions that a row does not see, and a huge value that every row gives
    next to no weight."""
    import torch

    n, dim, at = 400, 64, 300
    g = torch.Generator(device="cuda").manual_seed(12)
    q = 1 + 0.1 * torch.randn(n, 4, dim, generator=g, device="cuda")
    k, v = (torch.randn(n, 2, dim, generator=g, device="cuda") for _ in range(2))
    k[at:], v[at:] = k[at:] * big, v[at:] * big  # the rows before do not see these
    k[5], v[5] = -2.0, v[5] * min(big, 1e6)       # seen by all rows: a weight of about 2^-24 exp(..)
    out = torch.full_like(q, 7.0)
    if paged:
        ps = 16
        table = torch.randperm(n // ps, generator=g, device="cuda").int()[None]
        kc, vc = (torch.empty(n // ps, ps, 2, dim, device="cuda") for _ in range(2))
        kc[table[0].long()], vc[table[0].long()] = k.view(-1, ps, 2, dim), v.view(-1, ps, 2, dim)
        efg.attn_paged(out, q, kc, vc, table, _i(torch, [0, n]), _i(torch, [n]), n)
    else:
        efg.attn_prompt(out, q, k, v, _i(torch, [0, n]))
    _held("f32", _d(out)[:at], *attend(_d(q)[:at], _d(k)[:at], _d(v)[:at], float(np.float32(dim**-0.5))))
    assert efg.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_long_chunks_cut_along_the_keys(cuda, kind, dim):
    """Few long chunks share the GPU: row tiles are cut along the keys and joined; NaN and infinities at a row's
    later positions reach it neither through a piece nor through the join."""
    import torch

    chunks = [(150, 2900), (0, 40), (70, 4100), (1, 900), (130, 130), (20, 7)]
    q, seqs, out, args = _paged(torch, kind, chunks, 4, 2, dim, 16, seed=13, pad=2)
    _check_paged(kind, chunks, q, seqs, out)
    again = torch.full_like(out, 7.0)
    efg.attn_paged(again, *args, 150)
    assert torch.equal(out, again)
    _, kc, vc, table, _, _ = args
    for bad in (float("nan"), float("inf")):
        for j in range(2800, 2900):
            kc[int(table[0, j // 16]), j % 16] = vc[int(table[0, j // 16]), j % 16] = bad
        efg.attn_paged(again, *args, 150)
        k, v = seqs[0]
        want = attend(_d(q)[:50], _d(k)[:2800], _d(v)[:2800], float(np.float32(dim**-0.5)))
        _held(kind, _d(again)[:50], *want)
        assert not torch.isfinite(again[50:150]).any()
        _check_paged(kind, chunks[1:], q[150:], seqs[1:], again[150:])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.4])
def test_paged_with_other_scales(cuda, kind, scale):
    import torch

    for chunks in ([(1, 300), (1, 20)], [(40, 333), (3, 3)]):
        q, seqs, out, args = _paged(torch, kind, chunks, 8, 2, 64, 16, seed=14)
        efg.attn_paged(out, *args, max(m for m, _ in chunks), scale=scale)
        Q, O, a = _d(q), _d(out), 0
        for (m, n), (k, v) in zip(chunks, seqs):
            _held(kind, O[a : a + m], *attend(Q[a : a + m], _d(k), _d(v), float(np.float32(scale))))
            a += m
    assert efg.device_error() == 0


def _c_call(torch, args, max_new, work, work_bytes):
    """efg_attn_paged through the C interface, with a workspace of the test's choice."""
    from edgeforge_b200 import _lib

    q, kc, vc, table, cu, kv_len = args
    out = torch.full_like(q, 7.0)
    kind = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[q.dtype]
    block = _lib.ATTN_PAGED.pack(kind, q.shape[2] ** -0.5, out.data_ptr(), q.data_ptr(), q.shape[1] * q.shape[2],
                                 kc.data_ptr(), vc.data_ptr(), kc.shape[0], kc.shape[1], table.data_ptr(),
                                 table.shape[1], cu.data_ptr(), kv_len.data_ptr(), kv_len.numel(), q.shape[0], max_new,
                                 q.shape[1], kc.shape[2], q.shape[2], work, work_bytes)
    return _lib.load().efg_attn_paged(block, torch.cuda.current_stream().cuda_stream), out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 200])
def test_workspace_is_asked_for_and_checked(cuda, kind, m):
    import torch

    from edgeforge_b200 import _lib

    chunks = [(m, 5000), (1, 100)]
    q, seqs, out, args = _paged(torch, kind, chunks, 4, 2, 64, 16, seed=15)
    q, kc, vc, table, cu, kv_len = args
    kinds = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    need = _lib.load().efg_attn_paged_workspace(_lib.ATTN_PAGED.pack(
        kinds[q.dtype], 1.0, 0, 0, 0, 0, 0, 0, 16, 0, table.shape[1], 0, 0, 2, q.shape[0], m, 4, 2, 64, 0, 0))
    assert need > 0
    work = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    for ptr, size in ((0, 0), (0, need), (work.data_ptr(), need - 1), (work.data_ptr() + 8, need)):
        status, o = _c_call(torch, args, m, ptr, size)
        torch.cuda.synchronize()
        assert status == 1 and (o == 7.0).all()  # EFG_EINVAL, nothing queued
    work[need:] = 77
    status, o = _c_call(torch, args, m, work.data_ptr(), need)
    torch.cuda.synchronize()
    assert status == 0 and torch.equal(o, out) and (work[need:] == 77).all()
    _check_paged(kind, chunks, q, seqs, o)


@pytest.mark.parametrize("kind", KINDS)
def test_two_calls_at_once_and_a_graph_of_them(cuda, kind):
    """Decode steps and chunks on two streams, and both captured in one graph, as the calls one by one."""
    import torch

    calls = []
    for chunks, seed in (([(1, 9000), (1, 70)], 16), ([(180, 3000), (2, 50)], 17), ([(1, 400)] * 40, 18)):
        q, _, out, args = _paged(torch, kind, chunks, 8, 2, 64, 16, seed=seed)
        calls.append((args, max(m for m, _ in chunks), out))
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [torch.full_like(o, 7.0) for _, _, o in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, (args, m, _), o in zip(streams, calls, outs):
            with torch.cuda.stream(st):
                efg.attn_paged(o, *args, m)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o, (_, _, want) in zip(outs, calls))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        for st, (args, m, _), o in zip(streams, calls, outs):
            st.wait_stream(main)
            with torch.cuda.stream(st):
                efg.attn_paged(o, *args, m)
            main.wait_stream(st)
    for _ in range(3):
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o, (_, _, want) in zip(outs, calls))
    assert efg.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,dim,ps", [(1, 128, 128), (20, 128, 128), (100, 128, 128), (5, 128, 160)])
def test_cache_of_more_than_2_to_the_31_elements(cuda, kind, m, dim, ps):
    """Rows stored to and read from pages whose elements lie past 2^31 of the pool."""
    import torch

    dt = getattr(torch, TYPES[kind])
    kv, n = 2, 300
    pages = 2**31 // (ps * kv * dim) + 8
    kc, vc = (torch.empty(pages, ps, kv, dim, dtype=dt, device="cuda") for _ in range(2))
    table = _i(torch, [[pages - 1, 0, pages - 2]])
    g = torch.Generator(device="cuda").manual_seed(19)
    k, v, q = (torch.randn(x, h, dim, generator=g, device="cuda").to(dt) for x, h in ((n, kv), (n, kv), (m, 4)))
    slots = _i(torch, [int(table[0, j // ps]) * ps + j % ps for j in range(n)])
    efg.page_store(None, kc, vc, None, k, v, slots, slots.clone())
    out = torch.full_like(q, 7.0)
    efg.attn_paged(out, q, kc, vc, table, _i(torch, [0, m]), _i(torch, [n]), m)
    _held(kind, _d(out), *attend(_d(q), _d(k), _d(v), float(np.float32(dim**-0.5))))
    assert efg.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,dim", [(1, 64), (100, 64), (1, 128), (30, 128), (100, 20)])
def test_without_pages_and_without_positions(cuda, kind, m, dim):
    """An empty pool and a table without columns: rows that see nothing are zeros; a length there is an error."""
    import torch

    dt = getattr(torch, TYPES[kind])
    q = torch.randn(2 * m, 4, dim, device="cuda").to(dt)
    cache = torch.empty(0, 16, 2, dim, dtype=dt, device="cuda")
    for wide in (0, 2):
        table = torch.full((2, wide), -1, dtype=torch.int32, device="cuda")
        out = torch.full_like(q, 7.0)
        efg.attn_paged(out, q, cache, cache, table, _i(torch, [0, m, 2 * m]), _i(torch, [0, 0]), m)
        assert (out == 0).all() and efg.device_error() == 0
        efg.attn_paged(out, q, cache, cache, table, _i(torch, [0, m, 2 * m]), _i(torch, [0, 5]), m)
        torch.cuda.synchronize()
        assert (out[:m] == 0).all() and efg.device_error() == 1


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,heads,kv", [(1, 64, 8), (30, 64, 64), (50, 64, 8)])
def test_queries_of_more_than_2_to_the_31_elements(cuda, kind, m, heads, kv):
    """The last sequences' rows lie past 2^31 elements of q and out; the ones before see nothing."""
    import torch

    dt = getattr(torch, TYPES[kind])
    dim, ps, n = 128, 16, 70
    before = 2**31 // (heads * dim) // m + 2  # sequences of m rows and no position
    rows = (before + 2) * m
    q = torch.zeros(rows, heads, dim, dtype=dt, device="cuda")
    out = torch.full_like(q, 7.0)
    g = torch.Generator(device="cuda").manual_seed(20)
    q[-2 * m :] = torch.randn(2 * m, heads, dim, generator=g, device="cuda").to(dt)
    k, v = (torch.randn(10, ps, kv, dim, generator=g, device="cuda").to(dt) for _ in range(2))
    table = torch.zeros(before + 2, 5, dtype=torch.int32, device="cuda")
    table[-2:] = _i(torch, [[3, 1, 4, 0, 9], [2, 6, 5, 8, 7]])
    kv_len = torch.zeros(before + 2, dtype=torch.int32, device="cuda")
    kv_len[-2:] = n
    cu = torch.arange(before + 3, dtype=torch.int32, device="cuda") * m
    efg.attn_paged(out, q, k, v, table, cu, kv_len, m)
    assert efg.device_error() == 0
    for s in (0, 1):
        at = table[before + s].long()
        a = (before + s) * m
        want = attend(_d(q[a : a + m]), _d(k[at].flatten(0, 1)[:n]), _d(v[at].flatten(0, 1)[:n]), float(np.float32(dim**-0.5)))
        _held(kind, _d(out[a : a + m]), *want)
    assert float(out[: before * m].abs().max()) == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("m,dim", [(3, 64), (3, 128), (8, 80), (20, 64), (40, 128), (100, 64), (100, 128), (70, 20)])
def test_the_largest_values_at_later_positions(cuda, kind, sign, m, dim):
    """Later positions hold the type's largest or lowest value, in a prompt and over pages."""
    import torch

    dt = getattr(torch, TYPES[kind])
    g = torch.Generator(device="cuda").manual_seed(21)
    n, heads, kv, ps, see = 160, 4, 2, 16, 2  # the last m - see positions hold it
    q, k, v = (torch.randn(x, h, dim, generator=g, device="cuda").to(dt) for x, h in ((m, heads), (n, kv), (n, kv)))
    far = n - m + see
    k[far:] = v[far:] = sign * torch.finfo(dt).max
    scale = float(np.float32(dim**-0.5))
    table = torch.randperm(n // ps, generator=g, device="cuda").int()[None]
    kc, vc = (torch.empty(n // ps, ps, kv, dim, dtype=dt, device="cuda") for _ in range(2))
    kc[table[0].long()], vc[table[0].long()] = k.view(-1, ps, kv, dim), v.view(-1, ps, kv, dim)
    out = torch.full_like(q, 7.0)
    efg.attn_paged(out, q, kc, vc, table, _i(torch, [0, m]), _i(torch, [n]), m)
    want = attend(_d(q)[:see], _d(k)[:far], _d(v)[:far], scale)
    _held(kind, _d(out)[:see], *want)
    efg.attn_prompt(out, q, k[n - m :], v[n - m :], _i(torch, [0, m]))
    want = attend(_d(q)[:see], _d(k)[n - m : far], _d(v)[n - m : far], scale)
    _held(kind, _d(out)[:see], *want)
    assert efg.device_error() == 0
