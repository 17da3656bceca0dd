"""AdamW with 8-bit moments (numpy restatement).

TEST INFRASTRUCTURE ONLY (see `oracle/__init__.py`).

`store_*` / `load_*` restate the codes with fp32 arithmetic rounded after every operation, so
that the kernel's codes and scales must agree bit for bit; `step64` is the definition in 64 bits.
"""

from __future__ import annotations

import numpy as np

from oracle.philox import philox4x32_10

BLOCK = 128
TINY = np.float32(2.0**-100)


def bits(P, inner, *, tensor, step, seed, member_base=0):
    """(P, inner) 32 random bits per element; step: one per member."""
    group = np.arange((inner + 3) // 4, dtype=np.uint64)[None].astype(np.uint32)
    member = (np.arange(P, dtype=np.uint64)[:, None] + member_base).astype(np.uint32)
    when = np.asarray(step, dtype=np.uint64).reshape(-1, 1).astype(np.uint32)
    words = philox4x32_10(*np.broadcast_arrays(group, np.uint32(tensor), member, when),
                          np.uint32(seed & 0xFFFFFFFF), np.uint32(seed >> 32))
    return np.stack(words, -1).reshape(P, -1)[:, :inner]


def _blocks(x):
    P, inner = x.shape
    nb = -(-inner // BLOCK)
    return np.pad(x, ((0, 0), (0, nb * BLOCK - inner))).reshape(P, nb, BLOCK)


def _scale(x, top):
    big = np.abs(x).max(-1)
    scale = (big * (np.float32(1) / np.float32(top))).astype(np.float32)
    scale = np.where(big < TINY, np.float32(0), scale)
    scale = np.where(np.isfinite(big), scale, np.float32(np.nan))
    with np.errstate(divide='ignore', invalid='ignore'):
        inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0)).astype(np.float32)
    return scale, inv[..., None]


def store_first(m, r16):
    """(P, inner) fp32 and 16 random bits each -> (uint8 codes, fp32 scales)."""
    inner = m.shape[1]
    x, r = _blocks(m), _blocks(r16).astype(np.uint32)
    with np.errstate(invalid='ignore', over='ignore'):
        scale, inv = _scale(x, 448.0)
        y = np.minimum(np.abs(x) * inv, np.float32(448))
        normal = ((y.view(np.uint32) + (r << 4)) >> 20).astype(np.int64) - (120 << 3)
        small = np.where(y < 1, y * np.float32(512) + r.astype(np.float32) / np.float32(65536), 0).astype(np.int64)
    code = np.where(y >= np.float32(2.0**-6), normal, small) + np.where(x < 0, 128, 0)
    code = np.where(inv > 0, code, 0)
    return code.astype(np.uint8).reshape(len(m), -1)[:, :inner], scale


def store_root(u, r16):
    inner = u.shape[1]
    x, r = _blocks(u), _blocks(r16).astype(np.uint32)
    with np.errstate(invalid='ignore', over='ignore'):
        scale, inv = _scale(x, 1.9375)
        y = np.minimum(x * inv, np.float32(1.9375))
        code = np.clip(((y.view(np.uint32) + (r << 3)) >> 19).astype(np.int64) - (112 << 4), 1, 255)
    code = np.where((x > 0) & (inv > 0), code, 0)
    return code.astype(np.uint8).reshape(len(u), -1)[:, :inner], scale


def load_first(codes, scales):
    """fp32 first moments of uint8 codes (P, inner) and scales (P, blocks)."""
    c = codes.astype(np.int64)
    e, f = c >> 3 & 15, c & 7
    v = np.where(e > 0, (8.0 + f) * 2.0 ** (e - 10), f * 2.0**-9) * np.where(c > 127, -1.0, 1.0)
    return v.astype(np.float32) * np.repeat(scales, BLOCK, 1)[:, : codes.shape[1]]


def load_root(codes, scales):
    c = codes.astype(np.int64)
    v = np.where(c > 0, (16.0 + c % 16) * 2.0 ** (c // 16 - 19), 0.0)
    return v.astype(np.float32) * np.repeat(scales, BLOCK, 1)[:, : codes.shape[1]]


def moments32(m, u, g, b1, b2, one_m_b1, one_m_b2):
    """The new (m, u) in fp32, one rounding per operation; betas as fp32 columns or scalars."""
    with np.errstate(over='ignore', invalid='ignore'):
        m = m * b1 + g * one_m_b1
        u = np.sqrt((u * u) * b2 + (g * g) * one_m_b2)
    return m.astype(np.float32), u.astype(np.float32)


def step64(p, g, m, u, *, lr, b1, b2, eps, wd, t):
    """The new parameter in 64 bits, and the size of its update."""
    p, g, m, u = (x.astype(np.float64) for x in (p, g, m, u))
    m = b1 * m + (1 - b1) * g
    v = b2 * u * u + (1 - b2) * g * g
    update = lr * (m / (1 - b1**t)) / (np.sqrt(v / (1 - b2**t)) + eps)
    return p * (1 - lr * wd) - update, np.abs(update)
