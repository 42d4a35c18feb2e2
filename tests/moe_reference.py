"""64-bit references of the mixture-of-experts operators and of the linear
with an epilogue, with elementwise error bounds of the library's arithmetic
(test infrastructure).

The bounds follow the arithmetic in include/mlq.h, not a measurement:
* a value x in a block with largest magnitude A is carried either as 31-bit
  fixed point (half a step: below 1.01 * 2^-31 A; for q4 the block holds 16-fold
  values too, so 2^-27 A) or, with many rows, as two fp16 values (each rounding 2^-11
  relative: 2^-22 |x|, and at most 2^-39 of the largest of its 64 values where the
  second is subnormal).  A weight is then two fp16 values too: 2^-22 |w| (and
  q4_1 one fp32 rounding), 2^-39 of the largest of the row's 64; and the
  product of both second values, below 2^-22 |x w|, is left out.  The sum of all
  these covers either form;
* integer sums of a block are exact.  The fp32 steps round by 2^-24 relative
  each: per block one conversion of the integer sum, one product and one sum, then a
  few for the parts of the K axis, and 5 in a block's sum of x (q4) -- counted as
  (blocks + 16) roundings of the sum of magnitudes (each sum's partial values stay
  below it).  With many rows the sums of 64 values are made by the matrix unit,
  which may truncate: 12 instructions, 2^-22 of those magnitudes each, 48
  roundings more in all."""
from __future__ import annotations

import math

import numpy as np

EPS = 2.0 ** -24
BLOCK = {"q8_0": 34, "q4_0": 18, "q4_1": 20}


def bytes_of(fmt, rows, cols):
    return rows * ((cols + 31) // 32) * BLOCK[fmt]


def random_blocks(rng, fmt, rows, cols):
    """Packed blocks with random codes (every code value occurs) and scales of
    weights near N(0, 0.02); codes past `cols` are random too: x is zero there."""
    nb = (cols + 31) // 32
    raw = rng.integers(0, 256, (rows * nb, BLOCK[fmt]), dtype=np.uint8)
    if fmt == "q8_0":
        raw[:, 2:][raw[:, 2:] == 128] = 129
        d = rng.uniform(1e-4, 6e-4, rows * nb)
    else:
        d = rng.uniform(2e-3, 9e-3, rows * nb)
    d = (d * rng.choice([-1.0, 1.0], rows * nb)).astype(np.float16)
    raw[:, 0:2] = d.view(np.uint8).reshape(-1, 2)
    if fmt == "q4_1":
        m = rng.uniform(-0.06, 0.06, rows * nb).astype(np.float16)
        raw[:, 2:4] = m.view(np.uint8).reshape(-1, 2)
    return raw.reshape(-1)


def dequantize64(fmt, blocks, rows, cols):
    """(weights, magnitudes that the kernel sums) as float64 [rows, cols]."""
    nb = (cols + 31) // 32
    raw = np.ascontiguousarray(blocks).reshape(rows * nb, BLOCK[fmt])
    d = raw[:, 0:2].copy().view(np.float16).astype(np.float64)
    if fmt == "q8_0":
        w = raw[:, 2:].copy().view(np.int8) * d
        mag = np.abs(w)
    else:
        code = raw[:, BLOCK[fmt] - 16:]
        code = np.concatenate((code & 15, code >> 4), 1).astype(np.float64)
        if fmt == "q4_0":
            w = (code - 8) * d
            mag = (code + 8) * np.abs(d)  # summed as c x and 8 x apart
        else:
            m = raw[:, 2:4].copy().view(np.float16).astype(np.float64)
            w = code * d + m
            mag = code * np.abs(d) + np.abs(m)  # summed as d c x and m x apart
    return w.reshape(rows, nb * 32)[:, :cols], mag.reshape(rows, nb * 32)[:, :cols]


def block_max(x, size=32):
    """Per element, the largest magnitude of its block."""
    r, n = x.shape
    nb = (n + size - 1) // size
    p = np.zeros((r, nb * size))
    p[:, :n] = np.abs(x)
    return np.repeat(p.reshape(r, nb, size).max(2), size, 1)[:, :n]


def product(x, fmt, blocks, out, dx=None):
    """x W^T in float64 and its bound; dx: an elementwise error of x already there."""
    w, mag = dequantize64(fmt, blocks, out, x.shape[1])
    xa = np.abs(x) + (0 if dx is None else dx)
    step = (3 * 2.0 ** -22 + EPS) * xa + 1.01 * 2.0 ** -27 * block_max(xa) + 2.0 ** -39 * block_max(xa, 64)
    nb = (x.shape[1] + 31) // 32
    bound = step @ np.abs(w).T + 2.0 ** -39 * (xa @ block_max(np.abs(w), 64).T)
    bound += (nb + 64) * EPS * ((xa + step) @ mag.T)
    if dx is not None:
        bound = bound + dx @ np.abs(w).T
    return x @ w.T, bound


def experts(x, ids, weights, residual, fmt, fmt_down, gate, up, down, n_experts, hidden, out):
    """y and its bound; gate/up/down: packed stacks."""
    rows, k = ids.shape
    x = x.astype(np.float64)
    y = np.zeros((rows, out))
    mag = np.zeros((rows, out))
    bound = np.zeros((rows, out))
    per = lambda f, o, i: bytes_of(f, o, i)  # noqa: E731
    for e in np.unique(ids):
        if e < 0 or e >= n_experts:
            continue
        r, j = np.nonzero(ids == e)
        gb = per(fmt, hidden, x.shape[1])
        db = per(fmt_down, out, hidden)
        g, dg = product(x[r], fmt, gate[e * gb:(e + 1) * gb], hidden)
        u, du = product(x[r], fmt, up[e * gb:(e + 1) * gb], hidden)
        sg = g / (1 + np.exp(-g))
        h = sg * u
        # |silu'| <= 1.1; the fp32 steps of silu and the product: 8 roundings
        dh = 1.1 * dg * np.abs(u) + np.abs(sg) * du + 1.1 * dg * du + 8 * EPS * (np.abs(h) + 1.1 * dg * (np.abs(u) + du))
        d, dd = product(h, fmt_down, down[e * db:(e + 1) * db], out, dh)
        w = weights[r, j].astype(np.float64)[:, None]
        np.add.at(y, r, d * w)
        np.add.at(mag, r, np.abs(d * w))
        np.add.at(bound, r, dd * np.abs(w))
    bound += (k + 2) * EPS * (mag + bound)
    if residual is not None:
        y = y + residual
        bound += EPS * np.abs(y)
    return y, bound + 1e-37


def act64(v, name):
    if name == "silu":
        return v / (1 + np.exp(-v))
    if name == "gelu":
        return v * 0.5 * np.vectorize(math.erfc)(-v / math.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if name == "relu":
        return np.where(v < 0, 0, v)
    if name == "sigmoid":
        return 1 / (1 + np.exp(-v))
    return v


def epilogue(x, fmt, blocks, out, bias=None, act="none", row_scale=None, residual=None):
    v, b = product(x.astype(np.float64), fmt, blocks, out)
    if bias is not None:
        v = v + bias
        b = b + EPS * (np.abs(v) + b)
    y = act64(v, act)
    if act not in ("none", "relu"):
        # every activation's slope is below 1.15; its own fp32 steps: at most 16 roundings of the value, and of the
        # exponent (times the slope there: below 1)
        b = 1.15 * b + 16 * EPS * (np.abs(y) + 1)
    if row_scale is not None:
        y = y * row_scale[:, None]
        b = b * np.abs(row_scale[:, None]) + EPS * np.abs(y)
    if residual is not None:
        y = y + residual
        b = b + EPS * np.abs(y)
    return y, b + 1e-37


def digits_bound(x, w):
    """How far a logit of 31-bit fixed point digits can be from the exact one.
    A row's unit is a power of two below 2 amax / 2139062016 (the largest magnitude
    becomes more than half of that); every value is off by half a unit at
    most, which meets the other side's magnitudes; of the 16 products of
    digits three are left out: at most 2 * 2^14 * 2^8 + 2^14 units of both per
    element, and the product of both halves."""
    x, w = np.abs(x.astype(np.float64)), np.abs(w.astype(np.float64))
    ux, uw = x.max(1)[:, None] * 2 / 2139062016, w.max(1)[None] * 2 / 2139062016
    return 0.5 * ux * w.sum(1) + 0.5 * uw * x.sum(1)[:, None] + x.shape[1] * ux * uw * (2.0 ** 23 + 2.0 ** 14 + 0.25)


def route(x, w, top_k, bias=None, scoring="softmax", renormalize=True, scale=1.0):
    logits = x.astype(np.float64) @ w.astype(np.float64).T
    if scoring == "softmax":
        s = np.exp(logits - logits.max(1, keepdims=True))
        s = s / s.sum(1, keepdims=True)
    else:
        s = 1 / (1 + np.exp(-logits))
    c = s if bias is None else s + bias.astype(np.float64)
    ids = np.argsort(-c, axis=1, kind="stable")[:, :top_k]
    p = np.take_along_axis(s, ids, 1)
    masked = np.take_along_axis(c, ids, 1) == -np.inf
    p = np.where(masked, 0, p)
    if renormalize:
        total = p.sum(1, keepdims=True)
        p = np.divide(p, total, out=np.zeros_like(p), where=total != 0)
    return np.where(masked, -1, ids).astype(np.int32), p * scale, logits
