"""Sequences at the limit of what a cache can hold: 2^31 - 256 positions."""
from __future__ import annotations

import ctypes as C
import subprocess
from pathlib import Path

import pytest

import edgeforge_b200 as efg

ROOT = Path(__file__).resolve().parent.parent
TOP = 2**31 - 256


def test_needs_at_the_limit(tmp_path):
    (tmp_path / "h.cpp").write_text('#include "efg_paged.cuh"\nextern "C" int ok(int32_t c, int32_t n, int64_t p, int64_t m) '
                                    "{ const auto s = efg::seq_need_held(c, n, p, m); "
                                    "return s.valid ? 1 : s.need || s.have || s.rows != (n > 0 ? n : 0) ? -1 : 0; }\n")
    subprocess.run(["g++", "-std=c++20", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared",
                    "-fPIC", "-I", str(ROOT / "edgeforge_b200" / "csrc"), str(tmp_path / "h.cpp"), "-o", str(tmp_path / "h.so")],
                   check=True)
    lib = C.CDLL(str(tmp_path / "h.so"))
    lib.ok.argtypes = [C.c_int32, C.c_int32, C.c_int64, C.c_int64]
    for p in (1, 16, 100, 2**20, 2**30):
        assert lib.ok(TOP - 1, 1, p, 2**31 - 1) == 1 and lib.ok(0, TOP, p, 2**31 - 1) == 1
        assert lib.ok(TOP, 1, p, 2**31 - 1) == 0 and lib.ok(2**31 - 1, 2**31 - 1, p, 2**31 - 1) == 0
        assert lib.ok(-1, 1, p, 2**31 - 1) == 0 and lib.ok(p, 1, p, 1) == 0
    assert lib.ok(2**31 - 1, 1, 2**20, 4096) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cached,new", [(2**31 - 1, 1), (2**31 - 3, 3), (TOP, 1), (2**31 - 1, 2**31 - 1)])
def test_a_sequence_past_the_limit_is_not_served(cuda, cached, new):
    """Its length would be negative and its positions those of padding rows; the sequence after it is served."""
    import torch

    def i(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    ps, wide, n_rows = 2**20, 4096, 8
    table = torch.zeros(2, wide, dtype=torch.int32, device="cuda")
    slots, pos, cu, kv_len, taken = i([7] * n_rows), i([7] * n_rows), i([7] * 3), i([7] * 2), i([7])
    rows = min(new, n_rows)
    efg.page_plan(table, slots, pos, cu, kv_len, taken, i([cached, 0]), i([new, 2]), i([1000, 1001]), 2047, ps)
    torch.cuda.synchronize()
    assert efg.device_error() == 1 and efg.device_error() == 0
    assert kv_len.tolist() == [0, 2] and taken.tolist() == [1]
    live = min(2, n_rows - rows)
    assert slots.tolist() == [-1] * rows + [1000 * ps, 1000 * ps + 1][:live] + [-1] * (n_rows - rows - live)
    assert pos.tolist() == [-1] * rows + [0, 1][:live] + [-1] * (n_rows - rows - live)


@pytest.mark.gpu
@pytest.mark.parametrize("at", [TOP - 1, 2**31 - 2**20])
def test_a_sequence_at_the_limit_is_served(cuda, at):
    import torch

    def i(a):
        return torch.tensor(a, dtype=torch.int32, device="cuda")

    ps, page = 2**20, 2000
    table = torch.full((1, 4096), page, dtype=torch.int32, device="cuda")
    slots, pos, cu, kv_len, taken = i([7]), i([7]), i([7] * 2), i([7]), i([7])
    efg.page_plan(table, slots, pos, cu, kv_len, taken, i([at]), i([1]), i([page]), 2047, ps)
    torch.cuda.synchronize()
    assert efg.device_error() == 0
    assert kv_len.tolist() == [at + 1] and pos.tolist() == [at] and slots.tolist() == [page * ps + at % ps]
