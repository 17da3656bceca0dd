"""Linear layers over ragged groups of rows, against 64 bits."""

import math

import pytest
import torch

from oracle import routed
from tabpack_b200 import ops
from tabpack_b200.nn import LinearPack

pytestmark = pytest.mark.gpu

U24 = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float32]


def sums(n, dtype):
    """Bound of a sum of n products on the tensor core relative to the sum of their magnitudes: a step of 16 products
    is added with less than two units in the last place of 24 bits (it does not round to nearest).  fp32 operands take six such
    sums, and leave out products below 2^-24 (three of them, and the parts' own remainders)."""
    steps = n / 16 + 2
    return steps * 2 * 2 * U24 if dtype == torch.bfloat16 else (6 * steps * 2 + 8) * 2 * U24


def data(sizes, K, N, dtype, seed=0, widths=False, head=3, tail=5, poison=True):
    P, R = len(sizes), sum(sizes) + head + tail
    edges = [head]
    for s in sizes:
        edges.append(edges[-1] + s)
    gen = torch.Generator(device='cuda').manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    d = dict(x=normal(R, K).to(dtype), w=(normal(P, N, K) * K ** -0.5).to(dtype), b=normal(P, N),
             dy=normal(R, N).to(dtype), saved=torch.relu(normal(R, N)).to(dtype), edges=edges,
             offsets=torch.tensor(edges, dtype=torch.int32, device='cuda'), in_f=None, out_f=None)
    if widths:
        d['in_f'] = torch.randint(1, K + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
        d['out_f'] = torch.randint(1, N + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
    if poison:  # nothing beyond a member's rows and widths takes part
        d['x'][:head] = d['dy'][:head] = math.nan
        d['x'][R - tail:] = d['dy'][R - tail:] = math.inf
        if widths:
            for m in range(P):
                a, e, i, o = edges[m], edges[m + 1], int(d['in_f'][m]), int(d['out_f'][m])
                d['x'][a:e, i:] = d['w'][m, :, i:] = d['w'][m, o:] = d['dy'][a:e, o:] = math.nan
                d['b'][m, o:] = math.nan
    return d


def check(d, relu, dtype):
    kw = dict(in_features=d['in_f'], out_features=d['out_f'], relu=relu)
    K, N = d['w'].shape[2], d['w'].shape[1]
    eps = torch.finfo(dtype).eps / 2 * 1.01
    y = ops.ragged_linear_forward(d['x'], d['w'], d['b'], d['offsets'], **kw)
    (want,), (mag,) = routed.ragged_linear(d['x'], d['w'], d['b'], d['edges'], d['in_f'], d['out_f'], relu)
    assert y.dtype == dtype and y.shape == want.shape
    assert ((y.double() - want).abs() <= want.abs() * eps + mag * sums(K, dtype)).all()
    got = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], d['saved'] if relu else None, d['offsets'], **kw)
    want, mag = routed.ragged_linear(d['x'], d['w'], None, d['edges'], d['in_f'], d['out_f'], relu, d['dy'], d['saved'])
    rows = max(b - a for a, b in zip(d['edges'], d['edges'][1:]))
    for name, g, t, m, e, n in zip(('dx', 'dw', 'db'), got, want, mag, (eps, U24, U24), (N, rows, rows)):
        bound = m * (sums(n, dtype) if name != 'db' else (n / 8 + 64) * U24)
        assert ((g.double() - t).abs() <= t.abs() * e + bound).all(), name
    assert got[0].dtype == dtype and got[1].dtype == got[2].dtype == torch.float32
    return y, got


SHAPES = [
    # sizes of the members' batches, features in, features out
    ([1], 1, 1), ([0, 0], 16, 8), ([5], 17, 3),
    ([0, 1, 17, 130, 0, 256, 300], 200, 264),     # partial tiles, members without rows
    ([129, 127, 128, 1], 64, 64),                 # on and beside a tile's edge
    ([700, 3, 650], 77, 33),                      # rows off 16-byte boundaries
    ([2] * 70, 64, 33),                           # more members than a warp holds, few rows each
    ([100, 0, 0, 5, 33, 1, 0, 2], 520, 130),      # few rows a member, one with many
    ([1], 4096, 520),                             # one row, the K loop over a cluster
    ([1500, 900, 2100], 1100, 1040),              # CTA pairs
    ([9001], 309, 190),                           # rows split over CTAs and into pieces
]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('widths', [False, True])
@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_forward_and_backward(shape, relu, widths, dtype):
    sizes, K, N = SHAPES[shape]
    check(data(sizes, K, N, dtype, seed=shape, widths=widths), relu, dtype)


@pytest.mark.parametrize('K', [2047, 2049, 5000])
def test_long_sums_in_fp32(K):
    d = data([40, 90], K, 70, torch.float32, seed=K)
    y, _ = check(d, True, torch.float32)
    # no further from 64 bits than a plain fp32 product by more than a few times
    (want,), _ = routed.ragged_linear(d['x'], d['w'], d['b'], d['edges'], relu=True)
    assert ((y.double() - want).norm() / want.norm()).item() < 1e-5


def test_long_batches():
    d = data([30011, 4097, 8], 96, 40, torch.bfloat16, seed=1)
    _, (_, dw, _) = check(d, False, torch.bfloat16)
    want, _ = routed.ragged_linear(d['x'], d['w'], None, d['edges'], dy=d['dy'])
    # the pieces of a sum keep what the tensor core's own rounding would lose over 30011 rows
    assert ((dw.double() - want[1]).norm() / want[1].norm()).item() < 1e-5


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes,K,N', [([4100], 64, 40), ([2600, 1500], 130, 70), ([300, 0, 80], 128, 128)])
def test_gradients_of_few_tiles(sizes, K, N, dtype):
    # both gradients in one launch, the rows in parts; each by itself is as near to the exact one
    d = data(sizes, K, N, dtype, seed=4)
    check(d, True, dtype)
    kw = dict(relu=True, need_db=False)
    dx, none, _ = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], d['saved'], d['offsets'], need_dw=False, **kw)
    assert none is None
    none, dw, _ = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], d['saved'], d['offsets'], need_dx=False, **kw)
    assert none is None
    (x, w, _), (x_mag, w_mag, _) = routed.ragged_linear(d['x'], d['w'], None, d['edges'], relu=True, dy=d['dy'], y=d['saved'])
    eps = torch.finfo(dtype).eps / 2 * 1.01
    assert ((dx.double() - x).abs() <= x.abs() * eps + x_mag * sums(N, dtype)).all()
    assert ((dw.double() - w).abs() <= w.abs() * U24 + w_mag * sums(max(sizes), dtype)).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('widths', [False, True])
def test_members_without_rows_between_long_ones(widths, dtype):
    # more tiles than CTAs, so that one CTA goes from a sum in pieces to a tile that is zero
    check(data([1100, 0] * 20, 520, 520, dtype, widths=widths), False, dtype)


@pytest.mark.parametrize('dtype', DTYPES)
def test_one_member_without_rows_and_one_row(dtype):
    check(data([0], 24, 16, dtype, head=2, tail=0), False, dtype)
    d = data([3, 4], 24, 16, dtype, head=0, tail=0)
    empty = ops.ragged_linear_forward(d['x'][:0], d['w'], d['b'], torch.zeros(3, dtype=torch.int32, device='cuda'))
    assert empty.shape == (0, 16)
    dx, dw, db = ops.ragged_linear_backward(d['dy'][:0], d['x'][:0], d['w'], None, torch.zeros(3, dtype=torch.int32,
                                                                                               device='cuda'))
    assert dx.shape == (0, 24) and not dw.any() and not db.any()


def test_offsets_out_of_range_are_cut():
    d = data([4, 6], 24, 16, torch.bfloat16, head=0, tail=0)
    for offsets in ([-5, 4, 10 ** 6], [0, 4, 10]):
        y = ops.ragged_linear_forward(d['x'], d['w'], d['b'], torch.tensor(offsets, device='cuda'))
        assert torch.equal(y, ops.ragged_linear_forward(d['x'], d['w'], d['b'], d['offsets']))
    # members of negative length have no rows
    y = ops.ragged_linear_forward(d['x'], d['w'], d['b'], torch.tensor([8, 3, 10], device='cuda'))
    assert torch.equal(y[3:], ops.ragged_linear_forward(d['x'], d['w'], d['b'],
                                                        torch.tensor([3, 3, 10], device='cuda'))[3:])


@pytest.mark.parametrize('rows,cols,stride,first', [(1, 1, 9, 8), (7, 5, 5, 0), (1000, 1003, 1003, 0), (33, 515, 600, 1), (3, 4095, 4099, 3)])
def test_rows_are_moved_onto_boundaries(rows, cols, stride, first):
    flat = torch.randn(first + rows * stride + 8, device='cuda').bfloat16()
    x = flat[first: first + rows * stride].view(rows, stride)[:, :cols]
    x[0, 0] = math.nan
    out, wide = ops._align_rows(x, stride, rows, cols, 0)
    assert wide % 8 == 0 and wide - cols < 8
    assert torch.equal(out[:, :cols].view(torch.int16), x.contiguous().view(torch.int16)) and not out[:, cols:].any()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('first', [0, 1, 4, 8])
def test_strided_operands(first, dtype):
    d = data([30, 50], 40, 24, dtype)
    wide = torch.full((88, 72), 7.0, device='cuda').to(dtype)
    x, dy = wide.clone()[:, first: first + 40], wide.clone()[:, first: first + 24]
    x.copy_(d['x'])
    dy.copy_(d['dy'])
    w = torch.zeros(2, 24, 56, device='cuda').to(dtype)[..., first: first + 40]
    w.copy_(d['w'])
    for a, b in ((x, d['x']), (x.T.contiguous().T, d['x'])):
        assert torch.equal(ops.ragged_linear_forward(a, w, d['b'], d['offsets']),
                           ops.ragged_linear_forward(b, d['w'], d['b'], d['offsets']))
    got = ops.ragged_linear_backward(dy, x, w, None, d['offsets'])
    for a, b in zip(got, ops.ragged_linear_backward(d['dy'], d['x'], d['w'], None, d['offsets'])):
        assert torch.equal(a, b)


@pytest.mark.parametrize('need', [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 0, 0)])
@pytest.mark.parametrize('dtype', DTYPES)
def test_some_of_the_gradients(need, dtype):
    d = data([200, 90], 40, 100, dtype)
    kw = dict(need_dx=need[0], need_dw=need[1], need_db=need[2])
    every = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], d['saved'], d['offsets'], relu=True)
    for n, g, e in zip(need, ops.ragged_linear_backward(d['dy'], d['x'], d['w'], d['saved'], d['offsets'], relu=True, **kw),
                       every):
        assert (g is None) if not n else torch.equal(g, e)


def test_without_a_bias_and_with_nan():
    d = data([30, 50], 40, 24, torch.bfloat16, head=0, tail=0)
    (want,), _ = routed.ragged_linear(d['x'], d['w'], None, d['edges'])
    got = ops.ragged_linear_forward(d['x'], d['w'], None, d['offsets'])
    torch.testing.assert_close(got.double(), want, rtol=2.0 ** -8, atol=1e-5)
    d['x'][10, 3] = math.nan
    for dtype in DTYPES:
        y = ops.ragged_linear_forward(d['x'].to(dtype), d['w'].to(dtype), None, d['offsets'], relu=True)
        assert y[10].isnan().all() and not y[torch.arange(80) != 10].isnan().any()


@pytest.mark.parametrize('dtype', DTYPES)
def test_gradient_against_differences(dtype):
    """sum(y c) is linear in x, w and b: a difference is the gradient but for the forward's roundings."""
    d = data([20, 30], 24, 16, dtype, head=0, tail=0)
    dx, dw, db = ops.ragged_linear_backward(d['dy'], d['x'], d['w'], None, d['offsets'])
    gen = torch.Generator(device='cuda').manual_seed(2)
    for name, grad in (('x', dx), ('w', dw), ('b', db)):
        step = torch.randn(grad.shape, generator=gen, device='cuda').to(d[name].dtype)
        moved = dict(d)
        moved[name] = d[name] + step
        real = (moved[name].double() - d[name].double())
        y0, y1 = (ops.ragged_linear_forward(t['x'], t['w'], t['b'], t['offsets']).double() for t in (d, moved))
        diff = ((y1 - y0) * d['dy'].double()).sum().item()
        want = (grad.double() * real).sum().item()
        # each y and each dx is rounded once
        noise = ((y0.abs() + y1.abs()) * d['dy'].double().abs()).sum().item() + (grad.double() * real).abs().sum().item()
        assert abs(diff - want) <= noise * (torch.finfo(dtype).eps / 2 + 1e-6)


def test_results_are_the_same_each_time_in_graphs_and_on_streams():
    d = data([700, 0, 90, 5000], 96, 72, torch.bfloat16, head=0, tail=0)
    x, offsets = d['x'], d['offsets']

    def step():
        y = ops.ragged_linear_forward(x, d['w'], d['b'], offsets, relu=True)
        return [y, *ops.ragged_linear_backward(d['dy'], x, d['w'], y, offsets, relu=True)]

    first = step()
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.normal_()
    offsets.copy_(torch.tensor([0, 10, 3000, 3001, 5790], dtype=torch.int32))  # other groups, the same graph
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    for a, b in zip(other, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize('autocast', [True, False])
@pytest.mark.parametrize('out', [48, 45])
def test_layer_with_gradients(autocast, out):
    torch.manual_seed(3)
    layer = LinearPack([20, 33, 9], [out, 7, 30], max_in_features=33, max_out_features=out, pack_size=3).cuda()
    edges = [0, 40, 41, 190]
    offsets = torch.tensor(edges, device='cuda')
    x = torch.randn(200, 33, device='cuda', requires_grad=True)
    with torch.autocast('cuda', dtype=torch.bfloat16, enabled=autocast):
        y = layer.forward_rows(x, offsets, relu=True)
    dtype = torch.bfloat16 if autocast else torch.float32
    assert y.dtype == dtype and y.shape == (200, out)
    c = torch.randn_like(y)
    y.backward(c)
    xr, wr = x.detach().to(dtype), layer.weight.detach().to(dtype)
    args = xr, wr, layer.bias.detach(), edges, layer.in_features, layer.out_features
    (want,), _ = routed.ragged_linear(*args, relu=True)
    torch.testing.assert_close(y.detach().double(), want, rtol=torch.finfo(dtype).eps, atol=1e-5)
    (dx, dw, db), _ = routed.ragged_linear(*args, relu=True, dy=c, y=y)
    torch.testing.assert_close(x.grad.double(), dx, rtol=torch.finfo(dtype).eps, atol=1e-5)
    torch.testing.assert_close(layer.weight.grad.double(), dw, rtol=1e-5, atol=1e-4)
    torch.testing.assert_close(layer.bias.grad.double(), db, rtol=1e-5, atol=1e-4)
    # the weights' copy follows an update
    with torch.no_grad():
        layer.weight.mul_(2.0)
        layer.bias.zero_()
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=autocast):
            again = layer.forward_rows(x, offsets)
        (want,), _ = routed.ragged_linear(xr, layer.weight.to(dtype), None, edges, layer.in_features, layer.out_features)
        torch.testing.assert_close(again.double(), want, rtol=torch.finfo(dtype).eps, atol=1e-5)


def test_layer_agrees_with_equal_batches():
    torch.manual_seed(4)
    layer = LinearPack([64, 40], [72, 56], max_in_features=64, max_out_features=72, pack_size=2).cuda()
    x = torch.randn(2, 50, 64, device='cuda').bfloat16()
    x[1, :, 40:] = 0
    y = layer(x)
    rows = layer.forward_rows(x.flatten(0, 1), torch.tensor([0, 50, 100], device='cuda'))
    torch.testing.assert_close(rows.view_as(y).float(), y.float(), rtol=2.0 ** -7, atol=1e-5)


def test_refusals():
    d = data([4, 6], 24, 16, torch.bfloat16, head=0, tail=0)
    x, w, b, o = d['x'], d['w'], d['b'], d['offsets']
    for args, error in (((x.float(), w, b, o), TypeError), ((x[:, :8], w, b, o), ValueError), ((x, w[0], b, o), ValueError),
                        ((x, w, b.bfloat16(), o), TypeError), ((x, w, b, o[:2]), ValueError), ((x, w, b, o.float()), TypeError),
                        ((x, w, b, o.cpu()), ValueError), ((x.cpu(), w, b, o), RuntimeError), ((x, w[:0], b, o), ValueError),
                        ((x.half(), w.half(), b, o), TypeError), ((x, w.cpu(), b, o), ValueError)):
        with pytest.raises(error):
            ops.ragged_linear_forward(*args)
    with pytest.raises(ValueError):
        ops.ragged_linear_forward(x, w, b, o, in_features=o)
    with pytest.raises(ValueError):
        ops.ragged_linear_backward(d['dy'], x, w, None, o, relu=True)
    with pytest.raises(ValueError):
        ops.ragged_linear_backward(d['dy'][:5], x, w, None, o)
    layer = LinearPack(24, 16, pack_size=2).cuda()
    with pytest.raises(ValueError):
        layer.forward_rows(x[None], o)
    with pytest.raises(RuntimeError):
        layer.forward_rows(x.cpu(), o)
