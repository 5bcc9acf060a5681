"""Plain 64-bit forms of the MXFP4 format and the grouped products (numpy, on the host), and
the inputs and tolerances of their tests."""
from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
#: half a step of a result type, relative to the value, and of its smallest values
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
HALF_TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}


def mx_encode(x):
    """(codes [..., K/2], scales [..., K/32]) of float values, by the definition: the scale by
    comparison with powers of two, an element by its distance to every level."""
    x = np.asarray(x, np.float64)
    b = x.reshape(-1, 32)
    amax = np.abs(b).max(axis=1)
    bad = ~np.isfinite(b).all(axis=1)
    safe = np.where(bad | (amax == 0), 1.0, amax)
    e = np.frexp(safe)[1] - 1 - 2
    byte = np.where(amax == 0, 0, np.maximum(e + 127, 0))
    t = np.where(bad[:, None], 0.0, np.abs(np.where(np.isfinite(b), b, 0.0)) * np.exp2(127.0 - byte)[:, None])
    d = np.abs(t[..., None] - LEVELS)
    near = d == d.min(axis=-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = code + 8 * np.signbit(b)
    code[bad] = 0
    byte = np.where(bad, 255, byte)
    code = code.reshape(x.shape).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.astype(np.uint8).reshape(x.shape[:-1] + (-1,))


def mx_decode(codes, scales):
    """float64 values of MXFP4 codes and scale bytes."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1,))
    v = np.where(c >= 8, -1.0, 1.0) * LEVELS[c & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(scales.shape + (32,)) * s[..., None]).reshape(v.shape)


def bounds(offsets, P):
    """[(first row, end)] of the groups: clamped into [0, P], the first from row 0."""
    o = np.clip(np.asarray(offsets, np.int64), 0, P)
    o[0] = 0
    return [(int(a), int(b)) for a, b in zip(o[:-1], o[1:])]


def forward(x, w, offsets):
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    y = np.zeros((x.shape[0], w.shape[1]))
    for e, (a, b) in enumerate(bounds(offsets, x.shape[0])):
        y[a:b] = x[a:b] @ w[e].T
    return y


def dgrad(dy, w, offsets):
    return forward(dy, np.swapaxes(np.asarray(w, np.float64), 1, 2), offsets)


def wgrad(dy, x, offsets, E):
    dy, x = np.asarray(dy, np.float64), np.asarray(x, np.float64)
    dw = np.zeros((E, dy.shape[1], x.shape[1]))
    for e, (a, b) in enumerate(bounds(offsets, x.shape[0])):
        dw[e] = dy[a:b].T @ x[a:b]
    return dw


def tolerance(ref, mags, n, dtype):
    """How far a result of `dtype` may be from the 64-bit one: n products (exact in fp32 for
    16-bit operands) added up in fp32 in any order, each addition off by at most a step
    (2^-23) of a partial sum that the sum of magnitudes bounds, then half a step of the
    result's type."""
    s = n * 2.0 ** -23 * mags
    return s + HALF_STEP[dtype] * (np.abs(ref) + s) + HALF_TINY[dtype]


def offsets_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def round_to(v, dtype):
    """float64 values rounded to a result type (through fp32, exact for the integers of the
    exact tests)."""
    import torch
    t = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype]
    return torch.from_numpy(np.asarray(v, np.float64)).float().to(t)
