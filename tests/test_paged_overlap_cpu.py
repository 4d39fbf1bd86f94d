"""Memory that a paged call writes and memory that it reads or writes elsewhere: every overlap is refused before any
device work, and what only touches is not."""
from __future__ import annotations

import pytest

from edgeforge_b200._lib import ATTN_PAGED, ATTN_PROMPT, PAGE_STORE

FAR = 2**24  # no two arrays of these calls reach each other at this distance


@pytest.fixture(autouse=True)
def _no_device():
    """The addresses are made up: what is not refused must end at the missing device."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("runs where there is no GPU")



def _call(fn, block, fields):
    return fn(block.pack(*(fields[n] or 0 for n in block.names)), None)


def _refused(lib, fn, block, fields, **moved):
    code = _call(fn, block, {**fields, **moved})
    return code == 1 and "overlap" in lib.efg_last_error().decode()


def _spread(names):
    return {n: FAR * (i + 1) for i, n in enumerate(names)}


STORE = ("q_out", "k_cache", "v_cache", "q", "k", "v", "slots", "positions", "cos", "sin")
STORE_BYTES = {"q_out": 3 * 512 * 2, "k_cache": 64 * 128 * 2, "v_cache": 64 * 128 * 2, "slots": 12, "positions": 12,
               "cos": 64 * 32 * 4, "sin": 64 * 32 * 4}


@pytest.mark.parametrize("out", ["q_out", "k_cache", "v_cache"])
@pytest.mark.parametrize("read", ["slots", "positions", "cos", "sin"])
def test_store(efg_lib, out, read):
    lib = efg_lib.load()
    f = dict(type=2, cache_type=2, n_slots=64, q_stride=512, k_stride=128, v_stride=128, n_rows=3, max_pos=64, heads=8,
             kv_heads=2, head_dim=64, **_spread(STORE))
    args = lib, lib.efg_page_store, PAGE_STORE, f
    assert not _refused(*args)
    assert _refused(*args, **{out: f[read]})
    assert _refused(*args, **{read: f[out] + STORE_BYTES[out] - 4})
    assert _refused(*args, **{read: f[out] - STORE_BYTES[read] + 4})
    assert not _refused(*args, **{read: f[out] + STORE_BYTES[out]})
    assert not _refused(*args, **{read: f[out] - STORE_BYTES[read]})


@pytest.mark.parametrize("at,hits", [(0, True), (-5 * 512 * 2 + 2, True), (3 * 4, False), (8, True)])
def test_prompt(efg_lib, at, hits):
    lib = efg_lib.load()
    f = dict(type=2, scale=0.125, q_stride=512, k_stride=128, v_stride=128, n_seqs=2, n_rows=5, heads=8, kv_heads=2,
             head_dim=64, **_spread(("out", "q", "k", "v", "cu")))
    args = lib, lib.efg_attn_prompt, ATTN_PROMPT, f
    assert not _refused(*args)
    assert _refused(*args, out=f["cu"] + at) == hits


PAGED = ("out", "q", "k_cache", "v_cache", "block_table", "cu", "kv_len", "workspace")


def _paged_fields():
    return dict(type=2, scale=0.125, q_stride=512, n_pages=16, page_size=16, max_pages=16, n_seqs=3, n_rows=5, max_new=5,
                heads=8, kv_heads=2, head_dim=64, workspace_bytes=2**20, **_spread(PAGED))


@pytest.mark.parametrize("read,size", [("block_table", 3 * 16 * 4), ("cu", 16), ("kv_len", 12)])
def test_paged(efg_lib, read, size):
    lib = efg_lib.load()
    f = _paged_fields()
    args = lib, lib.efg_attn_paged, ATTN_PAGED, f
    n_out = 5 * 512 * 2
    assert not _refused(*args)
    assert _refused(*args, out=f[read])
    assert _refused(*args, out=f[read] + size - 2)
    assert _refused(*args, out=f[read] - n_out + 2)
    assert not _refused(*args, out=f[read] + size)
    assert not _refused(*args, out=f[read] - n_out)


@pytest.mark.parametrize("other,size", [("out", 5 * 512 * 2), ("q", 5 * 512 * 2), ("k_cache", 256 * 128 * 2),
                                        ("v_cache", 256 * 128 * 2), ("block_table", 3 * 16 * 4), ("cu", 16), ("kv_len", 12)])
def test_workspace(efg_lib, other, size):
    lib = efg_lib.load()
    f = _paged_fields()
    args = lib, lib.efg_attn_paged, ATTN_PAGED, f
    assert _refused(*args, workspace=f[other])
    assert _refused(*args, workspace=f[other] - 2**20 + 4)
    assert _refused(*args, **{other: f["workspace"] + 2**20 - 4})
    assert not _refused(*args, **{other: f["workspace"] + 2**20})
    assert not _refused(*args, workspace=f[other] - 2**20)
    assert not _refused(*args, **{other: f["workspace"] - size})
    assert not _refused(*args, workspace=0, workspace_bytes=0)
