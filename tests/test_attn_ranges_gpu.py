"""FP32 attention over wide ranges of values, element by element against float64 (attn_reference.py states the error
that is allowed and why; no term is added to it here)."""
from __future__ import annotations

import numpy as np
import pytest

import edgeforge_b200 as efg
from attn_reference import attend, tolerance

pytestmark = pytest.mark.gpu
MAX = float(np.finfo(np.float32).max)


def _i(torch, a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _d(t):
    return t.double().cpu().numpy()


def _held(got, *expected):
    want, tol = expected[0], tolerance("f32", *expected)
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), float(off.max()))


def _call(torch, q, k, v, ps=16):
    """The chunk q after all but its own of the positions of k and v: as a prompt where it has them all, over shuffled
    pages otherwise."""
    m, n, dim = q.shape[0], k.shape[0], q.shape[2]
    out = torch.full_like(q, 7.0)
    if m == n:
        efg.attn_prompt(out, q, k, v, _i(torch, [0, m]))
    else:
        pages = -(-n // ps)
        table = torch.randperm(pages, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").int()[None]
        kc, vc = (torch.full((pages, ps, k.shape[1], dim), float("nan"), device="cuda") for _ in range(2))
        at = torch.arange(n, device="cuda")
        slots = table[0].long()[at // ps] * ps + at % ps
        kc.view(-1, k.shape[1], dim)[slots], vc.view(-1, k.shape[1], dim)[slots] = k, v
        efg.attn_paged(out, q, kc, vc, table, _i(torch, [0, m]), _i(torch, [n]), m)
    torch.cuda.synchronize()
    assert efg.device_error() == 0
    return _d(out)


def _inputs(torch, m, n, dim, seed, heads=4, kv=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = 1 + 0.1 * torch.randn(m, heads, dim, generator=g, device="cuda")
    k, v = (torch.randn(n, kv, dim, generator=g, device="cuda") for _ in range(2))
    return q, k, v


@pytest.mark.parametrize("what", ["values", "keys", "both"])
@pytest.mark.parametrize("big", [1e8, 1e13, 1e30, MAX])
@pytest.mark.parametrize("m,n,see,dim", [(64, 64, 40, 64), (400, 400, 300, 64), (100, 100, 3, 20), (100, 1500, 40, 64),
                                         (100, 4000, 70, 64), (20, 20, 9, 64), (64, 64, 40, 128), (4, 300, 2, 64)])
def test_huge_later_positions(cuda, what, big, m, n, see, dim):
    """Huge finite keys or values from the position behind row see - 1 on: the rows before see none of them, whether
    they fill a key tile, lie in the first one or are all that one piece of the keys holds."""
    import torch

    q, k, v = _inputs(torch, m, n, dim, 31)
    far = n - m + see
    for t in {"values": (v,), "keys": (k,), "both": (k, v)}[what]:
        t[far:] = (t[far:].sign() if big == MAX else t[far:]) * big
    out = _call(torch, q, k, v)
    _held(out[:see], *attend(_d(q)[:see], _d(k)[:far], _d(v)[:far], float(np.float32(dim**-0.5))))


def _check(torch, q, k, v):
    _held(_call(torch, q, k, v), *attend(_d(q), _d(k), _d(v), float(np.float32(q.shape[2] ** -0.5))))


SIZES = [(200, 200, 64), (64, 64, 64), (150, 1500, 64), (100, 100, 20), (20, 20, 64), (90, 90, 128), (4, 300, 64)]


@pytest.mark.parametrize("big", [1e3, 1e6, 1e8, 1e10, 1e30])
@pytest.mark.parametrize("m,n,dim", SIZES)
def test_a_large_channel_of_values(cuda, big, m, n, dim):
    """One dim of all values is far larger than the others: every element keeps FP32 accuracy, with the large dim also
    of another size at later positions, and with one dim of zeros."""
    import torch

    q, k, v = _inputs(torch, m, n, dim, 32)
    v[:, :, 3] *= big
    _check(torch, q, k, v)
    v[n - m // 2 :, :, 3] *= 1e4
    v[:, 1, 7] = 0
    _check(torch, q, k, v)


@pytest.mark.parametrize("first,second", [(1e-12, 1.0), (1.0, 1e-12), (1.0, 1e9), (1e-30, 1e30)])
@pytest.mark.parametrize("m,n,dim", SIZES)
def test_values_of_two_sizes(cuda, first, second, m, n, dim):
    """Positions of one size, then positions of another, in all dims and in every second one."""
    import torch

    for step in (1, 2):
        q, k, v = _inputs(torch, m, n, dim, 33)
        half = n - m // 2
        v[:half, :, ::step] *= first
        v[half:, :, ::step] *= second
        _check(torch, q, k, v)


@pytest.mark.parametrize("bits", [20, 26, 30, 40, 60, 100])
@pytest.mark.parametrize("where", [5, 130])
@pytest.mark.parametrize("m,n,dim", [(200, 200, 64), (150, 1500, 64), (100, 400, 32), (200, 200, 128), (4, 300, 64)])
def test_a_huge_value_of_next_to_no_weight(cuda, bits, where, m, n, dim):
    """A value of 2^bits whose weight is near 2^-bits: what it adds is as large as the rest, and its weight has to be
    as exact as theirs."""
    import torch

    q, k, v = _inputs(torch, m, n, dim, 34)
    k[where] = -bits * np.log(2) / dim**0.5
    v[where] *= 2.0**bits
    _check(torch, q, k, v)


def test_a_value_far_below_the_others_of_its_dim(cuda):
    """Rows that see nothing else than a key whose value is tiny in a few dims, also with zeros about."""
    import torch

    q, k, v = _inputs(torch, 150, 150, 64, 35)
    for d, small in ((0, 1e-9), (1, 1e-15), (2, 1e-30), (3, 0.0)):
        v[:30, :, d] *= small
    v[60:90, :, 5] = 0
    _check(torch, q, k, v)


def test_rows_that_take_longer_alone_than_a_wait_may(cuda):
    """The last rows of a long prompt see a key far above the others and are computed alone, one after another (32 a
    warp, about 3 s; a wait gives up after 2): the rest of the CTA waits for them, and every row is there."""
    import torch

    n, dim = 2**19, 64
    g = torch.Generator(device="cuda").manual_seed(36)
    q, k, v = (torch.randn(n, 1, dim, generator=g, device="cuda") for _ in range(3))
    k[n - 130] = 1e8
    out = torch.full_like(q, float("nan"))
    efg.attn_prompt(out, q, k, v, _i(torch, [0, n]))
    torch.cuda.synchronize()
    assert efg.device_error() == 0
    assert torch.isfinite(out).all()
    scale = float(np.float32(dim**-0.5))
    for r in (5, 1000, 300001, n - 300, n - 131, n - 130, n - 77, n - 1):
        want = attend(_d(q[r : r + 1]), _d(k[: r + 1]), _d(v[: r + 1]), scale)
        _held(_d(out[r : r + 1]), *want)


@pytest.mark.parametrize("share", [0.02, 0.5, 0.98])
@pytest.mark.parametrize("m,n,dim,spread", [(200, 200, 64, 3.0), (129, 129, 60, 8.0), (150, 2700, 64, 8.0), (64, 64, 12, 8.0),
                                            (90, 90, 128, 8.0), (3, 2800, 64, 8.0)])
def test_values_with_zeros(cuda, share, m, n, dim, spread):
    """Dims where the keys that weigh most have a value of zero: what keys of next to no weight add is all there is.
    Weights are held within 2^-48 of the row's largest (include/efg.h), which over n keys is n 2^-48 max |v|."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(37)
    q, k, v = (torch.randn(x, h, dim, generator=g, device="cuda") for x, h in ((m, 4), (n, 2), (n, 2)))
    q = q * spread / dim**0.5 * 2
    v[torch.rand(v.shape, generator=g, device="cuda") > share] = 0
    out = _call(torch, q, k, v)
    want = attend(_d(q), _d(k), _d(v), float(np.float32(dim**-0.5)))
    assert (np.abs(out - want[0]) <= tolerance("f32", *want) + 2.0**-48 * want[3]).all()
