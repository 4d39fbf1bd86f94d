"""Plain 64-bit forms of the paged serving operators, and the error that their kernels may make.

A kernel rounds the output once (u = eps / 2 of its type, relative), a 16-bit one also each softmax
weight (u again, relative to the weight). Everything else is FP32: with A = sum_j w_j |v_j| and
B = max_j scale sum_d |q_d k_jd|, a score is off by at most (d + 4) 2^-24 B (d products and sums; F32
operands split for the tensor cores leave out at most 2^-21 of a product, counted as 8 steps more), a
weight by twice that plus 2^-21 (exponential, running maximum, normalisation), and a sum over n weights
by (n / 8 + 40) 2^-24 of A: no kernel adds more than n / 8 products one after the other outside the
tensor cores, whose sums over 16 or more products are at least as good as one FP32 chain over n / 8.
F16 holds a weight of at most 2^-14 of the largest within 2^-25 of it, which over n weights is at most
n 2^-25 max |v|.
"""
from __future__ import annotations

import numpy as np

EPS = {"f32": 2.0**-23, "f16": 2.0**-10, "bf16": 2.0**-7}


def attend(q, k, v, scale, last=None):
    """q [m][h][d], k and v [n][kv][d] in float64; row i sees keys 0 .. n - m + i. Returns (out, tolerance
    without the type's own roundings as a multiple of A, A, n max |v|)."""
    m, h, d = q.shape
    n, kv, _ = k.shape
    g = h // kv
    out = np.zeros((m, h, d))
    A = np.zeros((m, h, d))
    rel, tiny = np.zeros((m, h, 1)), np.zeros((m, h, 1))
    for i in range(m):
        c = n - m + i + 1
        if c <= 0:
            continue
        for a in range(kv):
            qq = q[i, a * g : (a + 1) * g]
            s = qq @ k[:c, a].T * scale
            B = (np.abs(qq) @ np.abs(k[:c, a]).T).max(-1, keepdims=True) * abs(scale)
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[i, a * g : (a + 1) * g] = w @ v[:c, a]
            A[i, a * g : (a + 1) * g] = w @ np.abs(v[:c, a])
            rel[i, a * g : (a + 1) * g] = 2 * (d + 12) * 2.0**-24 * B + 2.0**-21 + (c / 8 + 40) * 2.0**-24
            tiny[i, a * g : (a + 1) * g] = c * np.abs(v[:c, a]).max()
    return out, rel, A, tiny


def tolerance(kind, out, rel, A, tiny):
    u = EPS[kind] / 2
    if kind == "f32":
        return u * np.abs(out) + A * rel
    return u * np.abs(out) + A * (rel + u) + (2.0**-25 * (1 + tiny) if kind == "f16" else 0.0)


def plan(cached, new, table, free, page_size, n_rows):
    """The step plan in plain Python, every sequence served. Returns a dict of int32 arrays."""
    table = np.array(table, np.int32)
    slots, positions, cu, taken = [], [], [0], 0
    for s, (c, m) in enumerate(zip(cached, new)):
        have, held = -(-c // page_size), -(-(c + m) // page_size)
        for j in range(have, held):
            table[s, j] = free[taken]
            taken += 1
        for t in range(c, c + m):
            slots.append(int(table[s, t // page_size]) * page_size + t % page_size)
            positions.append(t)
        cu.append(cu[-1] + m)
    pad = [-1] * (n_rows - cu[-1])
    return {"table": table, "slots": np.array(slots + pad, np.int32), "positions": np.array(positions + pad, np.int32),
            "cu": np.array(cu, np.int32), "kv_len": np.array([c + m for c, m in zip(cached, new)], np.int32),
            "taken": np.array([taken], np.int32)}


def rotate(x, pos, cos, sin):
    """Half-split rotation of x [rows][heads][d] in float64 by table rows cos[pos], sin[pos]."""
    a = x.shape[-1] // 2
    c, s = cos[pos][:, None, :].astype(np.float64), sin[pos][:, None, :].astype(np.float64)
    return np.concatenate([x[..., :a] * c - x[..., a:] * s, x[..., a:] * c + x[..., :a] * s], -1)
