"""Routing of rows to members and the moves of rows, against 64 bits."""

import math

import pytest
import torch

from oracle import routed
from tabpack_b200 import nn as pnn
from tabpack_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


def scores(T, E, dtype, seed, masked=0.0, levels=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    z = 2.0 * torch.randn(T, E, generator=gen, device='cuda')
    if levels:
        z = torch.round(z * levels) / levels
    if masked:
        z.masked_fill_(torch.rand(T, E, generator=gen, device='cuda') < masked, -math.inf)
    return z.to(dtype)


def weight_tolerance(z, E):
    """exp(z - max) as 2^(z log2(e) + c): the exponent's rounding is 2^-24 of at most |z - max| log2(e) (the rounding
    of c is common to a row), ex2.approx is off by 2^-22; a weight has one such term above and their sum below, and the sum of
    E terms over 32 lanes and 5 exchanges rounds (E / 32 + 5) times by 2^-24."""
    finite = torch.where(torch.isfinite(z.float()), z.float(), 0.0)
    spread = (finite.amax() - finite.amin()).item() * 1.5
    return 2 * (2.0 ** -22 + spread * 2.0 ** -24) + (E / 32 + 8) * 2.0 ** -24


def check_route(z, k, renormalize):
    E = z.shape[1]
    weight, expert, position, offsets, importance = ops.route_forward(z, k, renormalize=renormalize)
    w, e, p, o, i = routed.route(z, k, renormalize)
    assert torch.equal(expert.long(), e) and torch.equal(position.long(), p) and torch.equal(offsets.long(), o)
    assert weight.dtype == importance.dtype == torch.float32 and expert.dtype == position.dtype == torch.int32
    rtol = weight_tolerance(z, E)
    torch.testing.assert_close(weight.double(), w, rtol=rtol, atol=1e-37)
    # sums over rows: a warp's rows, then warps, then blocks, each addition rounded by 2^-24 of the sum so far
    torch.testing.assert_close(importance.double(), i, rtol=rtol + (z.shape[0] / 64 + 64) * 2.0 ** -24, atol=1e-30)
    return weight, expert, position, offsets, importance


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('T,E,k,renormalize', [
    (1, 1, 1, True), (1, 64, 4, False), (7, 3, 3, True), (33, 1024, 32, True), (300, 257, 6, False),
    (129, 33, 2, True), (2000, 40, 1, False), (20001, 130, 8, True), (1025, 288, 1, True), (4097, 513, 3, False)])
def test_route(T, E, k, renormalize, dtype):
    check_route(scores(T, E, dtype, T + E), k, renormalize)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('E,k', [(2, 2), (8, 4), (24, 2), (32, 4), (33, 4), (24, 5), (64, 8), (65, 8), (100, 9), (128, 16), (129, 16), (100, 17)])
def test_rows_that_share_a_warp(E, k, dtype):
    # 4, 8, 16 and 32 lanes a row; rows with nothing, with NaN and with ties beside ordinary ones
    z = scores(3001, E, dtype, E * k, masked=0.3)
    z[::7] = -math.inf
    z[3::11] = torch.round(z[3::11])
    check_route(z, k, True)
    z[5::64, 0] = math.nan
    weight, expert, position, offsets, _ = ops.route_forward(z, k)
    rows = torch.isnan(z.float()).any(1)
    assert torch.isnan(weight[rows][expert[rows] >= 0]).all() and not torch.isnan(weight[~rows]).any()
    clean = z.clone()
    clean[rows] = -math.inf
    other = ops.route_forward(clean, k)
    assert torch.equal(weight[~rows], other[0][~rows]) and torch.equal(expert[~rows], other[1][~rows])


@pytest.mark.parametrize('T', [5, 3000])
@pytest.mark.parametrize('renormalize', [True, False])
def test_route_masked(T, renormalize):
    z = scores(T, 9, torch.float32, 3, masked=0.6)
    z[0] = -math.inf
    z[T // 2, :8] = -math.inf
    _, expert, position, offsets, _ = check_route(z, 4, renormalize)
    assert (expert[0] == -1).all() and (position[0] >= offsets[-1]).all()


@pytest.mark.parametrize('T', [40, 5000])
def test_route_ties_go_to_the_lowest_member(T):
    check_route(scores(T, 70, torch.bfloat16, 4, levels=1), 7, True)
    check_route(torch.zeros(T, 70, device='cuda'), 7, True)


def test_route_one_lane_holds_all_of_the_best():
    z = scores(50, 256, torch.float32, 5)
    z[:, 3::32] += 100.0 + torch.arange(8, device='cuda')
    check_route(z, 8, True)


def test_route_rows_that_are_not_finite():
    z = scores(100, 20, torch.float32, 6)
    plain = ops.route_forward(z, 3)
    bad = z.clone()
    bad[10, 4] = math.nan
    bad[20, 7] = math.inf
    weight, expert, _, offsets, importance = ops.route_forward(bad, 3)
    assert weight[10].isnan().all() and weight[20].isnan().all() and importance.isnan().all()
    assert expert[10, 0] == 4 and expert[20, 0] == 7
    rows = [r for r in range(100) if r not in (10, 20)]
    assert torch.equal(weight[rows], plain[0][rows]) and torch.equal(expert[rows], plain[1][rows])
    assert offsets[-1] == 300
    grad = ops.route_backward(torch.ones_like(weight), None, bad, weight, expert)
    assert grad[10].isnan().any() and not grad[rows].isnan().any()


def test_route_of_column_slices_and_empty():
    wide = scores(600, 50, torch.bfloat16, 7)
    check_route(wide[:, 3:40], 4, True)
    check_route(wide.T[:20], 4, True)
    weight, expert, position, offsets, importance = ops.route_forward(wide[:0], 2)
    assert weight.shape == expert.shape == position.shape == (0, 2) and not offsets.any() and not importance.any()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('T,E,k,renormalize,masked', [
    (1, 2, 1, False, 0), (3, 64, 4, True, 0), (500, 257, 6, False, 0.3), (77, 1024, 32, True, 0.5), (2500, 17, 3, True, 0.6)])
@pytest.mark.parametrize('which', ['both', 'weight', 'importance'])
def test_route_backward(T, E, k, renormalize, masked, dtype, which):
    z = scores(T, E, dtype, 8, masked=masked)
    gen = torch.Generator(device='cuda').manual_seed(9)
    gw = torch.randn(T, k, generator=gen, device='cuda') if which != 'importance' else None
    gi = torch.randn(E, generator=gen, device='cuda') if which != 'weight' else None
    weight, expert, *_ = ops.route_forward(z, k, renormalize=renormalize)
    got = ops.route_backward(gw, gi, z, weight, expert, renormalize=renormalize)
    z64 = z.double().requires_grad_()
    w, _, _, _, imp = routed.route(z64, k, renormalize)
    loss = 0.0
    if gw is not None:
        loss = loss + (w * gw.double()).sum()
    if gi is not None:
        loss = loss + (imp * gi.double()).sum()
    want = torch.autograd.grad(loss, z64)[0].nan_to_num()
    # terms w (g - sum w g) and p (h - sum p h): differences of numbers of the gradients' size, each off by the
    # weights' tolerance; then one rounding to the scores' type
    size = sum(g.abs().max().item() for g in (gw, gi) if g is not None)
    atol = 4 * size * (weight_tolerance(z, E) + k * 2.0 ** -23)
    torch.testing.assert_close(got.double(), want, rtol=torch.finfo(dtype).eps, atol=atol)
    assert got.dtype == dtype and got.is_contiguous()


@pytest.mark.parametrize('renormalize', [True, False])
def test_route_gradient_formula_against_differences(renormalize):
    gen = torch.Generator(device='cuda').manual_seed(10)
    z = torch.randn(6, 8, generator=gen, device='cuda', dtype=torch.float64)
    gw = torch.randn(6, 3, generator=gen, device='cuda', dtype=torch.float64)
    gi = torch.randn(8, generator=gen, device='cuda', dtype=torch.float64)

    def loss(t):
        w, _, _, _, imp = routed.route(t, 3, renormalize)
        return (w * gw).sum() + (imp * gi).sum()

    weight, expert, *_ = ops.route_forward(z.float(), 3, renormalize=renormalize)
    got = ops.route_backward(gw.float(), gi.float(), z.float(), weight, expert, renormalize=renormalize)
    h = 1e-5  # central differences: h^2 times third derivatives of order 10, and 2^-52 / h
    for r, c in ((0, 0), (1, 3), (2, 7), (5, 4)):
        up, down = z.clone(), z.clone()
        up[r, c] += h
        down[r, c] -= h
        diff = (loss(up) - loss(down)) / (2 * h)
        assert abs(diff.item() - got[r, c].item()) < 1e-5


def plan(T, k, E, seed, masked=0.0):
    z = scores(T, E, torch.float32, seed, masked=masked)
    weight, _, position, offsets, _ = ops.route_forward(z, k)
    return weight, position, offsets


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('T,k,W,masked', [
    (1, 1, 1, 0), (5, 2, 8, 0), (33, 3, 33, 0.7), (100, 5, 771, 0.6), (9, 32, 4096, 0), (64, 2, 12, 0.7), (40, 4, 8200, 0),
    (1000, 1, 100, 0.8)])
def test_row_moves(T, k, W, masked, dtype):
    weight, position, offsets = plan(T, k, 40, T + W, masked)
    used = int(offsets[-1])
    gen = torch.Generator(device='cuda').manual_seed(11)
    x = torch.randn(T, W, generator=gen, device='cuda').to(dtype)
    y = torch.randn(T * k, W, generator=gen, device='cuda').to(dtype)
    y[used:] = math.nan  # rows of no member are not read
    dout = torch.randn(T, W, generator=gen, device='cuda').to(dtype)
    assert torch.equal(ops.dispatch_rows(x, position, offsets), routed.dispatch(x, position, used))
    eps = torch.finfo(dtype).eps / 2
    mag = routed.combine(y.abs(), weight, position, used)
    for w in (weight, None):
        got = ops.combine_rows(y, w, position, offsets)
        assert got.dtype == dtype
        want = routed.combine(y, w, position, used)
        bound = (mag if w is not None else routed.combine(y.abs(), None, position, used)) * (k + 1) * 2.0 ** -23
        assert ((got.double() - want).abs() <= want.abs() * eps * 1.01 + bound).all()
    dy, dw = ops.combine_rows_backward(dout, y, weight, position, offsets)
    want = torch.zeros(T * k, W, dtype=torch.float64, device='cuda')
    want_dw = torch.zeros(T, k, dtype=torch.float64, device='cuda')
    size = torch.zeros_like(want_dw)
    for j in range(k):
        at = position[:, j].long()
        there = (at < used)[:, None]
        want[at] = torch.where(there, weight[:, j, None].double() * dout.double(), 0.0)
        terms = torch.where(there, dout.double() * y[at].double(), 0.0)
        want_dw[:, j], size[:, j] = terms.sum(1), terms.abs().sum(1)
    assert ((dy.double() - want).abs() <= want.abs() * (eps * 1.01 + 2.0 ** -24)).all()
    assert ((dw.double() - want_dw).abs() <= size * (W / 8 + 16) * 2.0 ** -24).all()
    only, none = ops.combine_rows_backward(dout, y, weight, position, offsets, need_dweight=False)
    assert none is None and torch.equal(only, dy)
    none, only = ops.combine_rows_backward(dout, y, weight, position, offsets, need_dy=False)
    assert none is None and torch.equal(only, dw)


def test_row_moves_of_strided_and_unaligned_rows():
    weight, position, offsets = plan(50, 2, 9, 12)
    wide = torch.randn(50, 130, device='cuda').bfloat16()
    for x in (wide[:, :64], wide[:, 1:65], wide[:, 2:66], wide[:, 4:68], wide[:, ::2], wide[0].expand(50, 130)):
        assert torch.equal(ops.dispatch_rows(x, position, offsets), routed.dispatch(x.contiguous(), position, 100))
    y = torch.randn(100, 130, device='cuda')
    for t in (y[:, :64], y[:, 1:65], y[:, 2:66]):
        assert torch.equal(ops.combine_rows(t, weight, position, offsets),
                           ops.combine_rows(t.contiguous(), weight, position, offsets))


def test_places_outside_the_rows_are_passed_over():
    x = torch.randn(4, 16, device='cuda')
    position = torch.tensor([[0, -1], [1, 8], [2, 2 ** 30], [3, -2 ** 31]], dtype=torch.int32, device='cuda')
    offsets = torch.tensor([0, 2, 4], dtype=torch.int32, device='cuda')
    got = ops.dispatch_rows(x, position, offsets)
    assert torch.equal(got[:4], x)
    assert torch.equal(ops.combine_rows(torch.cat([x, x]), None, position, offsets), x)
    dy, dw = ops.combine_rows_backward(x, torch.cat([x, x]), None, position, offsets)
    assert torch.equal(dy[:4], x) and not dw[:, 1].any()
    # a count of rows that is out of range is cut
    far = torch.tensor([0, 2, 10 ** 6], dtype=torch.int32, device='cuda')
    assert torch.equal(ops.combine_rows(torch.cat([x, x]), None, position, far), x)
    assert not ops.combine_rows(torch.cat([x, x]), None, position, torch.full_like(far, -3)).any()


def test_results_are_the_same_each_time():
    z = scores(30000, 100, torch.bfloat16, 13)
    first = ops.route_forward(z, 4, renormalize=False)
    for _ in range(3):
        for a, b in zip(first, ops.route_forward(z, 4, renormalize=False)):
            assert torch.equal(a, b)


def test_in_graphs_and_on_streams():
    z = scores(3000, 33, torch.float32, 14)
    x = torch.randn(3000, 24, device='cuda')

    def step():
        weight, _, position, offsets, importance = ops.route_forward(z, 2)
        rows = ops.dispatch_rows(x, position, offsets)
        out = ops.combine_rows(rows, weight, position, offsets)
        return [weight, position, offsets, importance, out, *ops.combine_rows_backward(out, rows, weight, position, offsets)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (15, 16):
        z.copy_(scores(3000, 33, torch.float32, seed))
        x.normal_()
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    for a, b in zip(other, step()):
        assert torch.equal(a, b)


def test_route_of_the_package_with_gradients():
    z = scores(200, 12, torch.float32, 17, masked=0.3).requires_grad_()
    x = torch.randn(200, 16, device='cuda', requires_grad=True)
    r = pnn.route(z, 3)
    rows = pnn.dispatch_rows(x, r)
    out = pnn.combine_rows(torch.tanh(rows), r)
    loss = (out ** 2).sum() + r.balance_loss()
    gz, gx = torch.autograd.grad(loss, (z, x))
    z64, x64 = z.detach().double().requires_grad_(), x.detach().double().requires_grad_()
    w, expert, _, offsets, imp = routed.route(z64, 3, True)
    there = (expert >= 0).double()
    out64 = (w * there).sum(1, keepdim=True) * torch.tanh(x64)
    counts = torch.diff(offsets).double()
    balance = 12 * (counts / counts.sum() * imp).sum() / 200
    wz, wx = torch.autograd.grad((out64 ** 2).sum() + balance, (z64, x64))
    # a row's copies are the same, so that the weights' gradients g are equal, G = sum 2 out tanh(x), and w (g - sum w g)
    # cancels to 0: what is left is each g's rounding (16 products and their sum, 2^-24 each) and that of sum w g, whose
    # weights are off by their tolerance, in all 2 G (17 2^-24 + tolerance)
    G = (2 * out64 * torch.tanh(x64)).abs().sum(1).max().item()
    torch.testing.assert_close(gz.double(), wz.nan_to_num(), rtol=1e-4,
                               atol=2 * G * (17 * 2.0 ** -24 + weight_tolerance(z.detach(), 12)))
    torch.testing.assert_close(gx.double(), wx, rtol=1e-5, atol=1e-5)
    assert not pnn.route(z, 3).expert.requires_grad


def test_refusals():
    z = scores(10, 5, torch.float32, 18)
    for bad, error in ((0, ValueError), (6, ValueError), (33, ValueError)):
        with pytest.raises(error):
            ops.route_forward(z, bad)
    with pytest.raises(ValueError):
        ops.route_forward(torch.zeros(3, 1025, device='cuda'), 2)
    with pytest.raises(ValueError):
        ops.route_forward(z[0], 2)
    with pytest.raises(TypeError):
        ops.route_forward(z.half(), 2)
    weight, expert, position, offsets, _ = ops.route_forward(z, 2)
    with pytest.raises(TypeError):
        ops.route_backward(weight.double(), None, z, weight, expert)
    with pytest.raises(ValueError):
        ops.route_backward(weight[:5], None, z, weight, expert)
    with pytest.raises(TypeError):
        ops.dispatch_rows(torch.zeros(10, 4, device='cuda'), position.long(), offsets)
    with pytest.raises(ValueError):
        ops.dispatch_rows(torch.zeros(11, 4, device='cuda'), position, offsets)
    with pytest.raises(ValueError):
        ops.combine_rows(torch.zeros(10, 4, device='cuda'), weight, position, offsets)
    with pytest.raises(ValueError):
        ops.combine_rows(torch.zeros(20, 4, device='cuda'), weight.cpu(), position, offsets)
    with pytest.raises(TypeError):
        ops.combine_rows_backward(torch.zeros(10, 4, device='cuda').bfloat16(), torch.zeros(20, 4, device='cuda'), weight,
                                  position, offsets)


def test_more_elements_than_31_bits():
    T, k, W = 34000, 2, 32768  # 2.2e9 elements in y
    x = torch.randn(T, W, device='cuda', dtype=torch.bfloat16)
    weight, _, position, offsets, _ = ops.route_forward(torch.randn(T, 8, device='cuda'), k)
    y = ops.dispatch_rows(x, position, offsets)
    some = torch.tensor([0, T // 2, T - 1, int(position.argmax()) // k], device='cuda')
    for j in range(k):
        assert torch.equal(y[position[some, j].long()], x[some])
    out = ops.combine_rows(y, weight, position, offsets)
    want = x[some].double() * weight[some].double().sum(1, keepdim=True)
    # a product and a sum in fp32, then one rounding to bf16
    assert ((out[some].double() - want).abs() <= want.abs() * (2.0 ** -8 + 4 * 2.0 ** -24)).all()
    del out
    dy, _ = ops.combine_rows_backward(x, y, weight, position, offsets, need_dweight=False)
    want = weight[some, 1:].double() * x[some].double()
    assert ((dy[position[some, 1].long()].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -24)).all()
