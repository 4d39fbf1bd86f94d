"""Paged serving without a GPU: the index arithmetic that the kernels run (efg_paged.cuh, compiled for
the host) on good and bad lengths and page ids, and the calls that are refused before any device work."""
from __future__ import annotations

import ctypes as C
import random
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent

HOST = r"""
#include "efg_paged.cuh"
using namespace efg;
extern "C" {
void need(int32_t c, int32_t f, int64_t ps, int64_t mp, int64_t* out) {
  const SeqNeed n = seq_need(c, f, ps, mp);
  out[0] = n.rows; out[1] = n.have; out[2] = n.need; out[3] = n.valid;
}
int served(int64_t need, int valid, int64_t first, int64_t n_free) {
  return seq_served(SeqNeed{0, 0, need, valid != 0}, first, n_free);
}
int ok(int32_t page, int64_t n) { return page_ok(page, n); }
int32_t visible(int32_t r, int32_t e, int32_t k) { return visible_keys(r, e, k); }
int64_t find(const int32_t* cu, int64_t n, int64_t row) { return find_sequence(cu, n, row); }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "host.cpp").write_text(HOST)
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-shared", "-fPIC", "-I", str(ROOT / "edgeforge_b200" / "csrc"),
                    str(d / "host.cpp"), "-o", str(d / "host.so")], check=True)
    lib = C.CDLL(str(d / "host.so"))
    i64 = C.c_int64
    lib.need.argtypes = [C.c_int32, C.c_int32, i64, i64, C.c_void_p]
    lib.served.argtypes = [i64, C.c_int, i64, i64]
    lib.ok.argtypes = [C.c_int32, i64]
    lib.visible.argtypes, lib.visible.restype = [C.c_int32] * 3, C.c_int32
    lib.find.argtypes, lib.find.restype = [C.c_void_p, i64, i64], i64
    return lib


def _need(lib, *a):
    out = np.zeros(4, np.int64)
    lib.need(*a, out.ctypes.data)
    return tuple(int(v) for v in out)


def test_needs(host):
    assert _need(host, 0, 0, 16, 4) == (0, 0, 0, 1)
    assert _need(host, 16, 1, 16, 4) == (1, 1, 1, 1)
    assert _need(host, 15, 1, 16, 4) == (1, 1, 0, 1)
    assert _need(host, 0, 64, 16, 4) == (64, 0, 4, 1)
    assert _need(host, 0, 65, 16, 4) == (65, 0, 0, 0)  # more positions than the table holds
    assert _need(host, -1, 5, 16, 4) == (5, 0, 0, 0)
    assert _need(host, 5, -1, 16, 4) == (0, 0, 0, 0)
    big = 2**31 - 1
    assert _need(host, big, big, 16, big) == (big, 2**27, 2**27, 1)  # no 32-bit overflow
    assert host.served(3, 1, 5, 8) and not host.served(4, 1, 5, 8)
    assert host.served(0, 1, 100, 8) and not host.served(0, 0, 0, 8)


def test_pages_and_visible_positions(host):
    assert host.ok(0, 1) and not host.ok(1, 1) and not host.ok(-1, 5) and not host.ok(0, 0)
    assert host.visible(0, 1, 1) == 1
    assert host.visible(12, 14, 100) == 99
    assert host.visible(10, 14, 3) == 0  # a chunk longer than its cache: the first rows see nothing
    assert host.visible(13, 14, 3) == 3
    assert host.visible(10, 14, 0) == 0
    top = 2**31 - 256
    assert host.visible(0, top, 0) == 0 and host.visible(0, 1, top) == top  # no 32-bit overflow at the limits
    assert host.visible(top - 1, top, top) == top and host.visible(0, top, top) == 1


def test_find_sequence_stays_in_bounds(host):
    r = random.Random(1)
    for trial in range(300):
        n = r.choice([1, 2, 5, 33])
        good = trial % 2 == 0
        cu = [0]
        for _ in range(n):
            cu.append(cu[-1] + r.choice([0, 0, 1, 7]) if good else r.randint(-2**31, 2**31 - 1))
        a = np.array(cu, np.int32)
        for row in range(-1, max(cu[-1], 3) + 2 if good else 20):
            s = host.find(a.ctypes.data, n, row)
            assert -1 <= s <= n
            if good:
                assert s == max((i for i in range(n + 1) if cu[i] <= row), default=-1)


def test_c_refusals(efg_lib):
    """Refused on the host, before a device is looked for (there is none here)."""
    lib = efg_lib.load()
    P = 4096  # never dereferenced

    def said(code, text):
        assert code == 1
        assert text in lib.efg_last_error().decode(), lib.efg_last_error()

    from edgeforge_b200._lib import ATTN_PAGED, ATTN_PROMPT, PAGE_PLAN, PAGE_STORE

    def call(fn, block, **fields):
        return lambda **k: fn(block.pack(*({**fields, **k}[n] or 0 for n in block.names)), None)

    plan = call(lib.efg_page_plan, PAGE_PLAN, block_table=P, max_pages=4, slots=P, positions=P, n_rows=8, cu=P, kv_len=P,
                taken=P, cached=P, new=P, n_seqs=2, free=P, n_free=8, n_pages=16, page_size=16)
    assert lib.efg_page_plan(None, None) == 1
    said(plan(cu=None), "null pointer")
    said(plan(free=None), "null pointer")
    said(plan(block_table=None), "null pointer")
    said(plan(slots=None), "null pointer")
    said(plan(page_size=0), "page size 0")
    said(plan(n_pages=2**30), "2^31 slots")
    said(plan(n_rows=2**31), "out of range")
    A = {n: 2**16 * (i + 1) for i, n in enumerate(("block_table", "slots", "positions", "cu", "kv_len", "taken", "cached", "new", "free"))}
    said(plan(**{**A, "kv_len": A["cached"]}), "overlaps")
    said(plan(**{**A, "kv_len": A["new"] + 4}), "overlaps")
    said(plan(**{**A, "positions": A["slots"] + 28}), "overlaps")
    said(plan(**{**A, "taken": A["cu"] + 8}), "overlaps")
    said(plan(**{**A, "block_table": A["free"] + 28}), "overlaps")

    store = call(lib.efg_page_store, PAGE_STORE, type=2, cache_type=2, q_out=P, k_cache=P, v_cache=P, n_slots=64, q=P,
                 q_stride=512, k=P, k_stride=128, v=P, v_stride=128, slots=P, positions=P, n_rows=3, cos=P, sin=P,
                 max_pos=64, heads=8, kv_heads=2, head_dim=64)
    said(store(type=3), "unknown type 3")
    said(store(cache_type=1), "the cache has the rows' type")
    said(store(type=1, cache_type=0), "the cache has the rows' type")
    said(store(head_dim=63), "not an even number")
    said(store(head_dim=0), "not an even number")
    said(store(kv_heads=0), "key heads")
    said(store(q=None), "come together")
    said(store(sin=None), "come together")
    said(store(k_stride=127), "shorter than a row")
    said(store(slots=None), "null pointer")
    A = {"q_out": 2**16, "k_cache": 2**18, "v_cache": 2**19, "q": 2**20, "k": 2**21, "v": 2**22}
    said(store(), "an output overlaps an input")
    said(store(**{**A, "q_out": 2**20 + 2}), "an output overlaps an input")  # not q itself
    said(store(**{**A, "q_out": 2**20, "q_stride": 513}), "an output overlaps an input")  # rows apart
    said(store(**{**A, "type": 0, "q_out": 2**20}), "an output overlaps an input")  # another type
    said(store(**{**A, "k_cache": 2**21 + (2 * 128 + 127) * 2}), "an output overlaps an input")
    said(store(**{**A, "v_cache": 2**22 - 64 * 128 * 2 + 2}), "an output overlaps an input")
    said(store(**{**A, "v_cache": 2**18}), "outputs overlap")
    said(store(**{**A, "q_out": 2**18 + 64 * 128 * 2 - 2}), "outputs overlap")
    assert store(n_rows=0) == 0  # nothing to do

    prompt = call(lib.efg_attn_prompt, ATTN_PROMPT, type=2, scale=0.125, out=P, q=P, q_stride=512, k=P, k_stride=128, v=P,
                  v_stride=128, cu=P, n_seqs=1, n_rows=5, heads=8, kv_heads=2, head_dim=64)
    said(prompt(type=4), "unknown type 4")
    said(prompt(head_dim=257), "not in 1..256")
    said(prompt(heads=7), "do not divide")
    said(prompt(kv_heads=0), "do not divide")
    said(prompt(q_stride=511), "shorter than a row")
    said(prompt(v_stride=100), "shorter than a row")
    said(prompt(scale=float("nan")), "not finite")
    said(prompt(scale=float("inf")), "not finite")
    said(prompt(cu=None), "null pointer")
    said(prompt(n_rows=2**31), "out of range")
    Q, K, V = 2**20, 2**21, 2**22
    said(prompt(), "out overlaps an input")
    said(prompt(out=Q - 5 * 512 * 2 + 2, q=Q, k=K, v=V), "out overlaps an input")
    said(prompt(out=K + (4 * 128 + 127) * 2, q=Q, k=K, v=V), "out overlaps an input")
    said(prompt(out=V, q=Q, k=K, v=V), "out overlaps an input")
    assert prompt(n_rows=0) == 0 and prompt(n_seqs=0) == 0

    paged = call(lib.efg_attn_paged, ATTN_PAGED, type=2, scale=0.125, out=P, q=P, q_stride=512, k_cache=P, v_cache=P,
                 n_pages=16, page_size=16, block_table=P, max_pages=4, cu=P, kv_len=P, n_seqs=1, n_rows=5, max_new=5,
                 heads=8, kv_heads=2, head_dim=64, workspace=0, workspace_bytes=0)
    said(paged(page_size=0), "page size 0")
    said(paged(n_pages=2**28), "2^31 slots")
    said(paged(max_pages=2**28), "2^31 slots")
    said(paged(max_new=2**31), "max_new")
    said(paged(block_table=None), "null pointer")
    said(paged(v_cache=None), "null pointer")
    said(paged(heads=9), "do not divide")
    said(paged(), "out overlaps an input")
    said(paged(out=K + (16 * 16 * 128 - 1) * 2, q=Q, k_cache=K, v_cache=V), "out overlaps an input")
    said(paged(out=V - 2, q=Q, k_cache=K, v_cache=V), "out overlaps an input")
    assert paged(n_rows=0) == 0 and paged(max_new=0) == 0
    assert lib.efg_attn_paged_workspace(None) == 0


def test_python_refusals(efg_lib):
    torch = pytest.importorskip("torch")
    E = efg_lib.EdgeForgeError
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(E, match="current CUDA device"):
        efg_lib.attn_prompt(z(4, 2, 8), z(4, 2, 8), z(4, 1, 8), z(4, 1, 8), i(2))
    with pytest.raises(E, match="current CUDA device"):
        efg_lib.attn_paged(z(4, 2, 8), z(4, 2, 8), z(3, 16, 1, 8), z(3, 16, 1, 8), i(1, 3), i(2), i(1), 4)
    with pytest.raises(E, match="current CUDA device"):
        efg_lib.page_plan(i(2, 4), i(8), i(8), i(3), i(2), i(1), i(2), i(2), i(4), 16, 16)
    with pytest.raises(E, match="come together"):
        efg_lib.page_store(None, z(3, 16, 1, 8), z(3, 16, 1, 8), z(4, 2, 8), z(4, 1, 8), z(4, 1, 8), i(4), i(4))
    with pytest.raises(E, match="back to back"):
        efg_lib.page_store(None, z(3, 16, 2, 8), z(3, 16, 2, 8), None, z(4, 8, 2).transpose(1, 2), z(4, 2, 8), i(4), i(4))
