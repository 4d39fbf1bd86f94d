"""What the paged calls' device-side checks find (pages that run out, bad slots, pages and lengths) is reported by
device_error and by nothing else: every other call gives its usual results while the report waits."""
from __future__ import annotations

import numpy as np
import pytest

import edgeforge_b200 as efg
from edgeforge_b200 import QType
from test_decode_gpu import medium  # noqa: F401  (a small decoder that has both modes, and the oracle's logits)

pytestmark = pytest.mark.gpu
TOL = 1e-4  # of the decoder's logits
ENOMEM, EINVAL = 5, 1


def _i(torch, a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _out_of_pages(torch):
    table, slots, pos = _i(torch, [[-1, -1]]), _i(torch, [0] * 20), _i(torch, [0] * 20)
    efg.page_plan(table, slots, pos, _i(torch, [0, 0]), _i(torch, [0]), _i(torch, [0]), _i(torch, [0]), _i(torch, [20]),
                  _i(torch, [3]), 8, 16)


def _bad_slot(torch):
    k = torch.ones(1, 1, 8, device="cuda")
    cache = torch.zeros(1, 4, 1, 8, device="cuda")
    efg.page_store(None, cache, cache.clone(), None, k, k, _i(torch, [4]), _i(torch, [0]))


def _bad_page(torch):
    q = torch.ones(1, 1, 64, device="cuda")
    cache = torch.zeros(1, 16, 1, 64, device="cuda")
    efg.attn_paged(torch.empty_like(q), q, cache, cache, _i(torch, [[9]]), _i(torch, [0, 1]), _i(torch, [3]), 1)


def _bad_offsets(torch):
    q = torch.ones(40, 1, 64, device="cuda")
    efg.attn_prompt(torch.empty_like(q), q, q, q, _i(torch, [0, 50]))


FINDINGS = [(_out_of_pages, ENOMEM), (_bad_slot, EINVAL), (_bad_page, EINVAL), (_bad_offsets, EINVAL)]


def _packed(torch, qt, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(rows)
    W = torch.empty(rows * cols // 32 * (18 if qt == QType.Q4_0 else 34), dtype=torch.uint8, device="cuda")
    efg.quantize_rows(qt, torch.randn(rows, cols, generator=g, device="cuda") * 0.02, rows, cols, W, True)
    return W, torch.randn(64, cols, generator=g, device="cuda")


@pytest.mark.parametrize("find,code", FINDINGS)
def test_matvec_gemm_and_sharded_calls_go_on(cuda, find, code):
    import torch

    rows, cols = 8192, 4096
    comm = efg.Comm(efg.Comm.unique_id(), 1, 0)
    try:
        for qt in (QType.Q4_0, QType.Q8_0):
            W, X = _packed(torch, qt, rows, cols)
            gemm = efg.gemm_q4_0 if qt == QType.Q4_0 else efg.gemm_q8_0

            def all_of_them():
                y, z, Y = (torch.full((n, rows), float("nan"), device="cuda") for n in (1, 1, 64))
                efg.matvec(qt, y[0], W, X[0], rows, cols)
                efg.matvec_sharded(qt, z[0], W, X[0], rows, cols, comm)
                gemm(Y, W, X, rows, cols, 64)
                torch.cuda.synchronize()
                return torch.cat([y, z, Y])

            want = all_of_them()
            assert torch.isfinite(want).all() and efg.device_error() == 0
            find(torch)
            for _ in range(5):
                assert torch.equal(all_of_them(), want)
            assert efg.device_error() == code and efg.device_error() == 0
    finally:
        comm.close()


@pytest.mark.parametrize("persistent", [True, False])
@pytest.mark.parametrize("find,code", FINDINGS)
def test_the_decoder_goes_on(cuda, medium, persistent, find, code):  # noqa: F811
    """And it does not take the report away from the call that it belongs to."""
    import torch

    efq, prompt, forced, ref = medium
    with efg.Decoder(efq, 64) as dec:
        dec.persistent = persistent
        find(torch)
        torch.cuda.synchronize()
        for i, t in enumerate(prompt):
            logits = dec.forward(int(t), i)
        assert np.abs(logits - ref[0]).max() <= TOL
        tokens = dec.generate(prompt, len(forced), forced=forced).tokens
        np.testing.assert_array_equal(np.array(tokens), np.argmax(ref, axis=1))
        dec.reset()
        assert np.abs(dec.prefill(prompt) - ref[0]).max() <= TOL
        dec.set_slots(2)
        logits, _ = dec.step_slots([1], [int(prompt[0])], [0])
        assert np.isfinite(logits).all()
    assert efg.device_error() == code and efg.device_error() == 0


def test_attention_goes_on_and_the_first_finding_is_kept(cuda):
    import torch

    g = torch.Generator(device="cuda").manual_seed(2)
    for kind in (torch.float32, torch.bfloat16):
        q, k, v = (torch.randn(300, h, 64, generator=g, device="cuda").to(kind) for h in (4, 2, 2))
        want, out = torch.empty_like(q), torch.empty_like(q)
        efg.attn_prompt(want, q, k, v, _i(torch, [0, 300]))
        _out_of_pages(torch)
        _bad_page(torch)
        efg.attn_prompt(out, q, k, v, _i(torch, [0, 300]))
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert efg.device_error() == ENOMEM and efg.device_error() == 0
