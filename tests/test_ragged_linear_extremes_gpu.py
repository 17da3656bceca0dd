"""fp32 linear layers over ragged groups of rows with infinities, NaN and the largest numbers in the members' own rows."""

import math

import pytest
import torch

from oracle import routed
from tabpack_b200 import ops

pytestmark = pytest.mark.gpu

U24 = 2.0 ** -24
# sizes of the members' batches, features in, features out
SHAPES = [
    ([12], 17, 8),
    ([300, 0, 80], 128, 136),      # both gradients in one launch
    ([40, 90], 1500, 70),          # the K loop in pieces
    ([4100], 64, 40),              # rows split over CTAs
    ([700, 30, 650], 77, 333),
    ([1500, 900, 2100], 1100, 1040),  # CTA pairs
    ([1100, 0] * 10, 520, 520),
]


def sums(n):
    """As for finite numbers: six sums of n products, each step of 16 added with less than two units in the last place of 24 bits."""
    return (6 * (n / 16 + 2) * 2 + 8) * 2 * U24


def data(sizes, K, N, seed, widths):
    edges = [2]
    for s in sizes:
        edges.append(edges[-1] + s)
    R, P = edges[-1] + 3, len(sizes)
    gen = torch.Generator(device='cuda').manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    d = dict(x=normal(R, K), w=normal(P, N, K) * K ** -0.5, b=normal(P, N), dy=normal(R, N), saved=torch.relu(normal(R, N)),
             edges=edges, offsets=torch.tensor(edges, dtype=torch.int32, device='cuda'), in_f=None, out_f=None)
    d['x'][:2] = d['dy'][R - 3:] = math.inf
    if widths:
        d['in_f'] = torch.randint(8, K + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
        d['out_f'] = torch.randint(8, N + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
    return d


def compare(got, want, mag, n):
    """The same infinities and NaN, and finite numbers as near as ever."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    finite = want.isfinite()
    assert ((got - want).abs()[finite] <= (want.abs() * U24 + mag * sums(n))[finite]).all()


def check(d, relu):
    kw = dict(in_features=d['in_f'], out_features=d['out_f'], relu=relu)
    N, K = d['w'].shape[1:]
    rows = max(b - a for a, b in zip(d['edges'], d['edges'][1:]))
    y = ops.ragged_linear_forward(d['x'], d['w'], d['b'], d['offsets'], **kw)
    (want,), (mag,) = routed.ragged_linear(d['x'], d['w'], d['b'], d['edges'], d['in_f'], d['out_f'], relu)
    compare(y, want, mag, K)
    saved = d['saved'] if relu else None
    got = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], saved, d['offsets'], **kw)
    want, mag = routed.ragged_linear(d['x'], d['w'], None, d['edges'], d['in_f'], d['out_f'], relu, d['dy'], d['saved'])
    for g, t, m, n in zip(got, want, mag, (N, rows, rows)):
        compare(g, t, m, n)
    # each gradient by itself
    dx, _, _ = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], saved, d['offsets'], need_dw=False, need_db=False, **kw)
    _, dw, _ = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], saved, d['offsets'], need_dx=False, need_db=False, **kw)
    compare(dx, want[0], mag[0], N)
    compare(dw, want[1], mag[1], rows)


@pytest.mark.parametrize('widths', [False, True])
@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_infinities_and_nan(shape, relu, widths):
    sizes, K, N = SHAPES[shape]
    d = data(sizes, K, N, shape, widths)
    for m, (a, e) in enumerate(zip(d['edges'], d['edges'][1:])):
        w = d['w'][m]
        w[1], w[2, 0], w[3, :4] = 1.0, 0.0, 0.5  # weights that one bf16 holds, and none at all
        w[4] = 1.0 + 2.0 ** -10  # ... whose second part has the other sign
        w[5, 6], w[6, 6] = math.inf, -math.inf
        if e - a < 9:
            continue
        x, dy = d['x'][a:e], d['dy'][a:e]
        x[0, 0], x[1, 1], x[2, 0], x[2, 3], x[3, 2] = math.inf, -math.inf, math.inf, -math.inf, math.nan
        x[4, 6] = 0.0  # against an infinite weight
        dy[5, 0], dy[6, 1], dy[7, 2], dy[7, 3] = math.inf, -math.inf, math.inf, math.inf
        dy[8, 4] = math.nan
    check(d, relu)


@pytest.mark.parametrize('widths', [False, True])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_the_largest_numbers(shape, widths):
    sizes, K, N = SHAPES[shape]
    d = data(sizes, K, N, 100 + shape, widths)
    d['w'].clamp_(-0.9, 0.9)
    top = torch.finfo(torch.float32).max
    for a, e in zip(d['edges'], d['edges'][1:]):
        if e - a < 9:
            continue
        x, dy = d['x'][a:e], d['dy'][a:e]
        # each alone among small ones, so that no sum of the definition overflows
        x[0], x[1], x[2], dy[:3] = 0.0, 0.0, 0.1, 0.01 * dy[:3].clamp(-4, 4)
        x[0, 5], x[1, 6] = top, -3.397e38
        dy[2, 3] = top
        x[2, 7] = -0.9
    check(d, False)
