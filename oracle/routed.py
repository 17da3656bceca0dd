"""Routing, row moves, ragged linear layers and 4-bit rows in 64 bits, from their definitions (torch, any device)."""

from __future__ import annotations

import math

import torch


def route(logits, k, renormalize):
    """(weight, expert, position, offsets, importance) of scores (T, E); weight and importance carry gradients."""
    z = logits.double()
    T, E = z.shape
    expert = torch.argsort(-z.detach(), dim=1, stable=True)[:, :k]
    chosen = z.gather(1, expert)
    there = chosen.detach() > -math.inf
    some = there[:, :1]
    p = torch.softmax(torch.where(some, z, 0.0), 1) * some
    w = torch.softmax(torch.where(some, chosen, 0.0), 1) * some if renormalize else p.gather(1, expert)
    flat = torch.where(there, expert, E).flatten()
    order = torch.argsort(flat, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(T * k, device=z.device)
    counts = torch.bincount(flat, minlength=E + 1)
    return w, torch.where(there, expert, -1), position.view(T, k), torch.cumsum(counts, 0) - counts, p.sum(0)


def dispatch(x, position, used):
    T, k = position.shape
    out = x.new_zeros(T * k, x.shape[1])
    for j in range(k):
        at = position[:, j].long()
        out[at] = torch.where((at < used)[:, None], x, 0)
    return out


def combine(y, weight, position, used):
    T, k = position.shape
    out = torch.zeros(T, y.shape[1], dtype=torch.float64, device=y.device)
    for j in range(k):
        at = position[:, j].long()
        term = torch.where((at < used)[:, None], y[at].double(), 0.0)
        out += term if weight is None else term * weight[:, j, None].double()
    return out


def ragged_linear(x, w, b, edges, in_f=None, out_f=None, relu=False, dy=None, y=None):
    """Forward: (y, bound), `bound` the sums of magnitudes.  With dy: (dx, dw, db) and their sums of magnitudes; `y` is
    the output whose sign the gradient goes by."""
    P, N, K = w.shape
    R = x.shape[0]
    new = lambda *s: torch.zeros(s, dtype=torch.float64, device=x.device)  # noqa: E731
    out = [new(R, N)] if dy is None else [new(R, K), new(P, N, K), new(P, N)]
    bound = [torch.zeros_like(t) for t in out]
    for m in range(P):
        a, e = edges[m], edges[m + 1]
        i = K if in_f is None else int(in_f[m])
        o = N if out_f is None else int(out_f[m])
        xm, wm = x[a:e, :i].double(), w[m, :o, :i].double()
        if dy is None:
            bias = 0.0 if b is None else b[m, :o].double()
            t = xm @ wm.T + bias
            out[0][a:e, :o] = t.relu() if relu else t
            bound[0][a:e, :o] = xm.abs() @ wm.abs().T + (0.0 if b is None else bias.abs())
        else:
            g = dy[a:e, :o].double()
            if relu:
                g = torch.where(y[a:e, :o] > 0, g, 0.0)
            for to, f in ((out, lambda t: t), (bound, torch.abs)):
                to[0][a:e, :i] = f(g) @ f(wm)
                to[1][m, :o, :i] = f(g).T @ f(xm)
                to[2][m, :o] = f(g).sum(0)
    return out, bound


FP4_BLOCK = {'nvfp4': 16, 'mxfp4': 32}
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _floor_log2(x):
    return torch.frexp(x)[1] - 1


def _pow2(n):
    return torch.ldexp(torch.ones(n.shape, dtype=torch.float64), n.cpu()).to(n.device)


def _e4m3(t):
    """Non-negative numbers up to 448 to e4m3: nearest, ties to even."""
    step = _pow2(torch.clamp(_floor_log2(t.clamp(min=2.0 ** -10)), min=-6) - 3)
    return torch.round(t / step) * step


def fp4_round(x, format, n=None):
    """(values, block scales, row scales) of (..., K) rows in 4 bits, in fp64; columns from `n` on count as zeros."""
    x = x.double()
    K, size = x.shape[-1], FP4_BLOCK[format]
    if n is not None:
        x = torch.where(torch.arange(K, device=x.device) < n, x, 0.0)
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, 0.0)
    b = torch.nn.functional.pad(x, (0, -K % size)).unflatten(-1, (-1, size))
    big = b.abs().amax(-1)
    if format == 'mxfp4':
        power = torch.clamp(_floor_log2(big.clamp(min=2.0 ** -130)) - 2, min=-100)
        scale, row = _pow2(power), torch.ones_like(big[..., 0])
    else:
        top = big.amax(-1).clamp(min=2.0 ** -130)
        row = _pow2(torch.clamp(-_floor_log2(2688.0 / top), min=-100))
        scale = _e4m3(big / 6.0 / row[..., None]) * row[..., None]
    q = torch.where(scale[..., None] > 0, b.abs() / scale[..., None], 0.0)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    up = torch.searchsorted(middle, q.contiguous(), right=True)   # the middle goes up
    down = torch.searchsorted(middle, q.contiguous(), right=False)  # the middle goes down
    code = torch.where(up % 2 == 0, up, down)  # the even one of the two
    value = torch.sign(b) * grid[code] * scale[..., None]
    row = torch.where(finite, row, math.nan)
    value = value.flatten(-2)[..., :K] * torch.where(finite, 1.0, math.nan)[..., None]
    return value, scale, row


def fp4_unpack(codes, scales, row_scale, K, format):
    """The values of rows (R, K) from their stored form: codes (R, pitch), scales (tiles, tiles of blocks, 512)."""
    R, size = codes.shape[0], FP4_BLOCK[format]
    byte = scales.cpu().long()
    code = codes.cpu().long()
    r = torch.arange(R)[:, None]
    c = torch.arange(K)[None]
    nibble = (code[r, c // 2] >> (4 * (c % 2))) & 15
    block = c // size
    s = byte[r // 128, block // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + block % 4]
    if format == 'mxfp4':
        scale = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s - 127)
    else:
        e, f = s >> 3 & 15, s & 7
        scale = torch.where(e > 0, torch.ldexp(1 + f.double() / 8, e - 7), f.double() / 512)
    value = torch.tensor(_GRID, dtype=torch.float64)[nibble & 7] * torch.where(nibble > 7, -1.0, 1.0)
    return value * scale * row_scale.cpu().double()[:, None]
