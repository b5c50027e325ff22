"""64-bit restatements of the training-step operators, for the tests.

Plain numpy, written from the operators' formulas; nothing here is used by the
package.  Where a result hangs on the order of fp32 roundings (the 8-bit
moments' codes) the restatement is in numpy float32, operation by operation.
"""

from __future__ import annotations

import numpy as np

U = 2.0 ** -24          # half a unit of fp32, relative
BLOCK, TOP = 256, 256.0


def norm_and_factor(grads, max_norm):
    total = sum(float(np.sum(np.square(g.astype(np.float64)))) for g in grads)
    norm = float(np.sqrt(total))
    factor = np.nan if not np.isfinite(total) else max_norm / norm if norm > max_norm else 1.0
    return norm, factor


def adamw(p, g, m, v, *, t, lr, beta1, beta2, eps, decay, scale=1.0):
    """(p, m, v, bounds): the step in 64 bits, and how far an fp32 step may be
    from each: every operation rounds by at most U relative to its result, the
    rounded constants by U each."""
    p, g, m, v = (a.astype(np.float64) for a in (p, g, m, v))
    g = g * scale
    parts_m = np.abs(beta1 * m) + np.abs((1 - beta1) * g)
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    rate, root = lr / (1 - beta1 ** t), 1 / np.sqrt(1 - beta2 ** t)
    denom = np.sqrt(v) * root + eps
    move = rate * m / denom
    new = p * (1 - lr * decay) - move
    # m: scale, product with a rounded constant, sum; v: two more products
    bm, bv = 5 * U * parts_m, 8 * U * v + 2e-45
    # p: its own product and difference; the move inherits m's, half of v's
    # and seven roundings of its own
    bp = 3 * U * np.abs(p) + rate / denom * bm + 12 * U * np.abs(move) + U * np.abs(new)
    return new, m, v, (bp, bm, bv)


def mix32(x):
    x = np.asarray(x, dtype=np.uint32)
    with np.errstate(over="ignore"):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(16))


def step_key(seed, t):
    k = mix32(np.uint32((seed & 0xFFFFFFFF) ^ 0x9E3779B9))
    for word in (seed >> 32, t & 0xFFFFFFFF, t >> 32):
        k = mix32(k ^ np.uint32(word))
    return k


def random_words(key, first_block, n):
    """32 bits for each of a tensor's n values; its blocks are counted from
    `first_block` on through the list."""
    i = np.arange(n, dtype=np.uint64)
    with np.errstate(over="ignore"):
        lane = (np.uint64(first_block * 32) + i // np.uint64(8)).astype(np.uint32)
        x = mix32(mix32(lane) + key) + (i % np.uint64(8)).astype(np.uint32) * np.uint32(0x9E3779B9)
        x = (x ^ (x >> np.uint32(17))) * np.uint32(0xBB67AE85)
    return x ^ (x >> np.uint32(15))


def e4m3_values():
    """The value of every e4m3 code 0..127 (127 is NaN)."""
    c = np.arange(128)
    e, f = c >> 3, c & 7
    val = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    val[127] = np.nan
    return val


def opened(codes, tops):
    """Codes (uint8) and tops to fp32 values, as the step reads them."""
    table = e4m3_values().astype(np.float32)
    mag = table[codes & 127]
    unit = (tops * np.float32(1 / TOP)).astype(np.float32)
    val = mag * np.repeat(unit, BLOCK)[:codes.size]
    return np.where(codes & 128, -val, val).astype(np.float32)


def closed(x, random16, second):
    """fp32 values to (codes, tops), each rounded up or down by 16 random bits."""
    n = x.size
    blocks = -(-n // BLOCK)
    pad = np.zeros(blocks * BLOCK, dtype=np.float32)
    pad[:n] = x
    tops = np.abs(pad).reshape(blocks, BLOCK).max(1)
    tops = np.where(tops < np.float32(2.0 ** -100), np.float32(0), tops).astype(np.float32)
    inv = np.zeros_like(tops)
    inv[tops > 0] = (np.float32(1) / tops[tops > 0]) * np.float32(TOP)
    a = (np.abs(x) * np.repeat(inv, BLOCK)[:n]).astype(np.float32)
    low = a < np.float32(2.0 ** -6)
    lifted = (a + np.where(low, np.float32(2.0 ** -6), np.float32(0))).astype(np.float32)
    bits = lifted.view(np.uint32) + ((random16.astype(np.uint32) << np.uint32(4)) + np.uint32(8))
    code = (bits >> np.uint32(20)).astype(np.int64) - 960 - 8 * low
    if second:
        code = np.where(x > 0, np.maximum(code, 1), code)
    code = code | np.where(x < 0, 128, 0)
    return code.astype(np.uint8), tops


def moments32(m, v, g, *, beta1, beta2, scale):
    """The new moments in fp32, each operation rounded on its own."""
    f = np.float32
    b1, r1, b2, r2 = f(beta1), f(1 - beta1), f(beta2), f(1 - beta2)
    g = (g.astype(np.float32) * f(scale)).astype(np.float32)
    m = (m * b1 + g * r1).astype(np.float32)
    v = (v * b2 + (g * g) * r2).astype(np.float32)
    return m, v


def _rms(a, eps):
    return 1 / np.sqrt(np.mean(a * a, axis=1, keepdims=True) + eps)


def _spread(gate, rows):
    return 1.0 if gate is None else np.repeat(gate, rows // gate.shape[0], axis=0)


def block_norm(x, h, gate, post, pre, *, post_norm=True, pre_norm=True, eps=1e-6, offset=0.0,
               a=1.0, b=1.0):
    """(y, z, post_rstd, pre_rstd) and the parts' magnitudes |a x| + |b gate u|."""
    rows = x.shape[0]
    q = None
    parts = np.abs(a * x)
    y = x
    if h is not None:
        u = h
        if post_norm:
            q = _rms(h, eps)
            u = h * q * (1.0 if post is None else post + offset)
        branch = b * _spread(gate, rows) * u
        y = a * x + branch
        parts = np.abs(a * x) + np.abs(branch)
    else:
        parts = np.abs(x)
    z = r = None
    if pre_norm:
        r = _rms(y, eps)
        z = y * r * (1.0 if pre is None else pre + offset)
    return y, z, None if q is None else q[:, 0], None if r is None else r[:, 0], parts


def block_norm_grads(y, h, gate, post, pre, q, r, dy, dz, *, offset=0.0, a=1.0, b=1.0):
    """The gradients, and for each a sum of the magnitudes that it is made of
    (what its rounding errors are relative to).  q, r: the statistics, or None
    without that norm."""
    rows, width = y.shape
    w = 1.0 if pre is None else pre + offset
    v = 1.0 if post is None else post + offset
    d = np.zeros_like(y) if dy is None else dy
    d_abs = np.abs(d)
    out = {}
    if r is not None:
        r = r[:, None]
        n, t = y * r, dz * w
        d = d + r * (t - n * np.mean(t * n, axis=1, keepdims=True))
        d_abs = d_abs + r * (np.abs(t) + np.abs(n) * np.mean(np.abs(t * n), axis=1, keepdims=True))
        out["dpre_weight"] = ((dz * n).sum(0), np.abs(dz * n).sum(0))
    if h is None:  # y is x
        out["dx"] = (d, d_abs)
        return out
    out["dx"] = (a * d, np.abs(a) * d_abs)
    g = _spread(gate, rows)
    e, e_abs = b * g * d, np.abs(b * g) * d_abs
    if q is None:
        k = h
        out["dh"] = (e, e_abs)
    else:
        k = h * q[:, None]
        out["dpost_weight"] = ((e * k).sum(0), (e_abs * np.abs(k)).sum(0))
        ev, ev_abs = e * v, e_abs * np.abs(v)
        out["dh"] = (q[:, None] * (ev - k * np.mean(ev * k, axis=1, keepdims=True)),
                     q[:, None] * (ev_abs + np.abs(k)
                                   * np.mean(ev_abs * np.abs(k), axis=1, keepdims=True)))
    if gate is not None:
        runs = gate.shape[0]
        both = [(b * d * k * v), (np.abs(b) * d_abs * np.abs(k * v))]
        out["dgate"] = tuple(s.reshape(runs, rows // runs, width).sum(1) for s in both)
    return out
