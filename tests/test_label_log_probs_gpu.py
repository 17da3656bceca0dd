"""Label log probabilities, entropies, best classes and their gradient on the GPU against the
formulas in 64 bits.

Tolerances, with u = 2^-24, z' = z - max z, S = sum exp z' >= 1, L = log S, d(C) = 64 + C / 256 the
longest chain of additions: an exponential of z' is off by (4 + 3 |z'|) u relative (the argument's
rounding, twice the exponential's own and one to spare), so S by (d + 4 + 3 E|z'|) u relative with
E|z'| <= H + L, and
    |log p error| <= u (|z'| + 3 L + |log p| + d + 8 + 3 (H + L))  =: e(z)
    |H error|     <= 2 u (d + 16) (1 + L + H) + u (H + L)^2
    |dz error|    <= |g_l| (p (e + u (4 + 3 |log p|)) + 2 u) + |g_H| p ((e + 8 u) (1 + |log p| + H) + H error)
The best classes are exact.  Outputs in bf16 add half a step.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
INF = float('inf')


@pytest.fixture(scope='module', autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')


def plain(z, labels, k, g_l, g_h):
    """64-bit values of rows z (R, C) and their tolerances."""
    C = z.shape[1]
    z64 = z.double()
    zp = z64 - z64.amax(1, keepdim=True)
    p = torch.softmax(z64, 1)
    L = torch.log(torch.exp(zp).sum(1, keepdim=True))
    lp = zp - L
    H = -torch.special.xlogy(p, p).sum(1, keepdim=True)
    d = 64 + C / 256
    e = U * (zp.abs() + 3 * L + lp.abs() + d + 8 + 3 * (H + L))
    eh = 2 * U * (d + 16) * (1 + L + H) + U * (H + L) ** 2
    hot = torch.nn.functional.one_hot(labels, C).double()
    plogp = torch.special.xlogy(p, p)
    dz = g_l[:, None] * (hot - p) - g_h[:, None] * (plogp + p * H)
    a = torch.where(p > 0, lp.abs(), 0)
    ep = torch.where(p > 0, e, 0)
    tdz = (g_l.abs()[:, None] * (p * (ep + U * (4 + 3 * a)) + 2 * U)
           + g_h.abs()[:, None] * p * ((ep + 8 * U) * (1 + a + H) + eh))
    order = torch.argsort(-z64, dim=1, stable=True)[:, :k]
    at = labels[:, None]
    return ((lp.gather(1, at)[:, 0], H[:, 0], lp.gather(1, order), order, dz),
            (e.gather(1, at)[:, 0], eh[:, 0], e.gather(1, order), tdz))


def near(got, want, tol, what, dtype=torch.float32):
    assert got.dtype == dtype, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), what
    assert torch.equal(got[~fine].double(), want[~fine]), what
    diff = (got.double() - want).abs()[fine]
    bound = (tol + torch.finfo(dtype).eps / 2 * want.abs())[fine] + 2.0**-126
    assert (diff <= bound).all(), (what, (diff - bound).max().item(), diff.max().item())


def make(lead, C, dtype, *, seed=0, scale=2.5, masked=0.0, ld=None):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    ld = C if ld is None else ld
    z = (torch.randn(*lead, ld, generator=gen, device='cuda') * scale).to(dtype)[..., :C]
    y = torch.randint(0, C, lead, generator=gen, device='cuda')
    if masked:
        off = torch.rand(z.shape, generator=gen, device='cuda') < masked
        off.scatter_(-1, y[..., None], False)
        z.masked_fill_(off, -INF)
    g_l, g_h = (torch.randn(lead, generator=gen, device='cuda') for _ in range(2))
    return z, y, g_l, g_h


def run_and_check(z, y, g_l, g_h, k=0):
    from tabpack_b200 import ops

    lp, H, top, which, stats = ops.label_log_probs_forward(z, y, top_k=k)
    dz = ops.label_log_probs_backward(g_l, g_h, z, y, stats)
    C, lead = z.shape[-1], z.shape[:-1]
    yr = y.expand(lead).reshape(-1)
    want, tol = plain(z.reshape(-1, C), yr, k, g_l.reshape(-1).double(), g_h.reshape(-1).double())
    assert lp.shape == H.shape == lead and dz.shape == z.shape and dz.is_contiguous()
    near(lp.reshape(-1), want[0], tol[0], 'log_prob')
    near(H.reshape(-1), want[1], tol[1], 'entropy')
    near(dz.reshape(-1, C), want[4], tol[3], 'dlogits', z.dtype)
    if k:
        assert torch.equal(which.reshape(-1, k), want[3]), 'top_label'
        near(top.reshape(-1, k), want[2], tol[2], 'top_log_prob')
    else:
        assert top is None and which is None


CLASSES = [1, 2, 3, 8, 10, 16, 17, 31, 32, 33, 64, 65, 100, 128, 129, 255, 256, 257, 500, 512, 513, 1000, 1023, 1024, 1025, 2048, 2051, 5000, 16384,
           32769, 51200, 131072, 200003]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('C', CLASSES)
def test_classes(C, dtype):
    run_and_check(*make((2, 5), C, dtype, seed=C), k=min(C, 7))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R', [1, 2, 3, 31, 700])
@pytest.mark.parametrize('C', [2, 10, 57, 300, 4097])
def test_rows(R, C, dtype):
    run_and_check(*make((R,), C, dtype, seed=R + C))


def test_many_rows_few_classes():
    run_and_check(*make((300, 200), 5, torch.bfloat16, seed=1))


@pytest.mark.parametrize('k', [1, 2, 5, 16, 31, 32])
@pytest.mark.parametrize('C', [32, 33, 200, 1500, 40000])
def test_best_classes(C, k):
    run_and_check(*make((3, 4), C, torch.bfloat16, seed=k), k=k)
    run_and_check(*make((3, 4), C, torch.float32, seed=k, masked=0.5), k=k)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R', [1, 2, 18, 19, 37, 38, 74, 75, 149])
def test_long_rows_of_every_split(R, dtype):
    """Row counts on both sides of each rule that spreads a row over a cluster, the best classes
    gathered in one part and spread over all, a NaN and a masked row among them."""
    from tabpack_b200 import ops

    C = 32779
    z, y, g_l, g_h = make((R,), C, dtype, seed=R)
    z[0, 8000:8032] += 20.0
    z[-1, ::500] += 20.0
    run_and_check(z, y, g_l, g_h, k=32)
    if R > 2:
        z[1], z[2, 9] = -INF, float('nan')
        lp, H, top, which, stats = ops.label_log_probs_forward(z, y, top_k=2)
        assert lp[1] == -INF and H[1] == 0 and which[1].tolist() == [0, 1]
        assert torch.isnan(lp[2]) and which[2, 0] == 9
        keep = [i for i in range(R) if i not in (1, 2)]
        want, tol = plain(z[keep], y[keep], 2, g_l[keep].double(), g_h[keep].double())
        near(lp[keep], want[0], tol[0], 'log_prob')
        assert torch.equal(which[keep], want[3])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R,C', [(1183, 4099), (1183, 8200), (1184, 1500), (1184, 16390), (1184, 32800)])
def test_long_rows_of_every_block_size(R, C, dtype):
    run_and_check(*make((R,), C, dtype, seed=C, masked=0.3), k=32)


@pytest.mark.parametrize('C', [40, 1024, 3000, 70000])
def test_best_classes_in_hard_orders(C):
    """Ascending, descending and constant rows, few distinct values, the best at the end."""
    z = torch.zeros(6, C, device='cuda')
    z[0] = torch.arange(C, device='cuda') * 1e-3
    z[1] = -z[0]
    z[3] = (torch.arange(C, device='cuda') % 3).float()
    z[4, -40:] = torch.arange(40, device='cuda').float()
    z[5, ::2], z[5, 1::2] = -0.0, 0.0
    y = torch.zeros(6, dtype=torch.int64, device='cuda')
    g = torch.ones(6, device='cuda')
    run_and_check(z, y, g, g, k=32)
    run_and_check(z.bfloat16(), y, g, g, k=32)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('C', [6, 90, 700, 9000])
def test_masked_classes(C, dtype):
    run_and_check(*make((4, 9), C, dtype, seed=C, masked=0.6), k=min(C, 6))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('C', [6, 700, 9000])
def test_lowest_values(C, dtype):
    """The type's lowest value as a mask: in some classes, and in all (a uniform row)."""
    z, y, g_l, g_h = make((5,), C, dtype, seed=C)
    low = torch.finfo(dtype).min
    z[0, 1::2] = low
    z[1] = low
    z[2] = torch.finfo(dtype).max
    z[3, 0], y[3] = low, 0
    run_and_check(z, y, g_l, g_h, k=4)


@pytest.mark.parametrize('C', [5, 300, 9000])
def test_rows_without_classes(C):
    """Nothing but -inf: log p = -inf, H = 0, a zero gradient, the first classes as the best."""
    from tabpack_b200 import ops

    z, y, g_l, g_h = make((4,), C, torch.float32, seed=C)
    z[2] = -INF
    lp, H, top, which, stats = ops.label_log_probs_forward(z, y, top_k=3)
    dz = ops.label_log_probs_backward(g_l, g_h, z, y, stats)
    assert lp[2] == -INF and H[2] == 0 and (dz[2] == 0).all()
    assert (top[2] == -INF).all() and which[2].tolist() == [0, 1, 2]
    keep = [0, 1, 3]
    run_and_check(z[keep], y[keep], g_l[keep], g_h[keep], k=3)
    assert torch.isfinite(dz).all()


@pytest.mark.parametrize('bad', [float('nan'), INF])
@pytest.mark.parametrize('C', [5, 300, 9000])
def test_nonfinite_rows(C, bad):
    from tabpack_b200 import ops

    z, y, g_l, g_h = make((4,), C, torch.float32, seed=C)
    z[1, C - 2], z[2, 0] = bad, -INF
    if y[2] == 0:
        y[2] = 1
    lp, H, top, which, stats = ops.label_log_probs_forward(z, y, top_k=3)
    dz = ops.label_log_probs_backward(g_l, g_h, z, y, stats)
    assert torch.isnan(lp[1]) and torch.isnan(H[1]) and torch.isnan(dz[1]).all() and torch.isnan(top[1]).all()
    assert which[1, 0] == C - 2
    keep = [0, 2, 3]
    run_and_check(z[keep], y[keep], g_l[keep], g_h[keep], k=3)


@pytest.mark.parametrize('C', [5, 300, 9000])
def test_ignored_and_invalid_labels(C):
    from tabpack_b200 import ops

    z, y, g_l, g_h = make((6,), C, torch.float32, seed=C)
    ref = y.clone()
    y[1], y[3], y[4] = -100, C, -1
    lp, H, _, _, stats = ops.label_log_probs_forward(z, y)
    dz = ops.label_log_probs_backward(g_l, g_h, z, y, stats)
    assert lp[1] == 0 and torch.isnan(lp[3]) and torch.isnan(lp[4])
    assert torch.isnan(dz[3]).all() and torch.isnan(dz[4]).all()
    only_h = g_l.clone()
    only_h[1] = 0
    want, tol = plain(z, ref, 0, only_h.double(), g_h.double())
    near(H, want[1], tol[1], 'entropy')
    keep = [0, 1, 2, 5]
    near(dz[keep], want[4][keep], tol[3][keep], 'dlogits')
    lp2, *_ = ops.label_log_probs_forward(z, y, ignore_index=C)
    assert lp2[3] == 0 and torch.isnan(lp2[1])
    # without the label's gradient an invalid label does not matter
    dz = ops.label_log_probs_backward(None, g_h, z, y, stats)
    want, tol = plain(z, ref, 0, torch.zeros_like(g_l).double(), g_h.double())
    near(dz, want[4], tol[3], 'dlogits of the entropy')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('C,ld', [(10, 16), (9, 16), (33, 40), (1000, 1001), (3001, 3008)])
def test_rows_of_padded_buffers(C, ld, dtype):
    run_and_check(*make((3, 7), C, dtype, seed=C, ld=ld), k=min(5, C))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('C', [16, 24, 40, 64, 96, 128, 200, 256])
def test_rows_on_different_boundaries(C, dtype):
    """Whole vectors per row, but a stride that starts the rows of one warp on different boundaries."""
    run_and_check(*make((2, 37), C, dtype, seed=C, ld=C + 1), k=min(5, C))
    run_and_check(*make((2, 37), C, dtype, seed=C, ld=C + 4))


def test_unaligned_storage_and_strided_rows():
    z, y, g_l, g_h = make((4, 6), 264, torch.bfloat16, seed=2)
    off = torch.empty(4 * 6 * 264 + 1, dtype=torch.bfloat16, device='cuda')[1:].view(4, 6, 264)
    off.copy_(z)
    run_and_check(off, y, g_l, g_h, k=3)
    run_and_check(z.transpose(0, 1), y.t(), g_l.t(), g_h.t(), k=3)
    run_and_check(z[:, ::2], y[:, ::2], g_l[:, ::2], g_h[:, ::2])
    run_and_check(z[:1].expand(4, -1, -1), y, g_l, g_h)


@pytest.mark.parametrize('C', [7, 600])
def test_shared_labels(C):
    z, y, g_l, g_h = make((4, 6), C, torch.bfloat16, seed=3)
    run_and_check(z, y[0], g_l, g_h, k=2)


@pytest.mark.parametrize('C', [10, 600, 5000])
def test_missing_and_expanded_gradients(C):
    from tabpack_b200 import ops

    z, y, g_l, g_h = make((4, 6), C, torch.float32, seed=4)
    stats = ops.label_log_probs_forward(z, y)[-1]
    zero = torch.zeros_like(g_l)
    bwd = lambda a, b: ops.label_log_probs_backward(a, b, z, y, stats)  # noqa: E731
    assert torch.equal(bwd(g_l, None), bwd(g_l, zero))
    assert torch.equal(bwd(None, g_h), bwd(zero, g_h))
    assert (bwd(None, None) == 0).all()
    one = torch.full((), 0.5, device='cuda')
    assert torch.equal(bwd(one.expand(4, 6), one.expand(4, 6)), bwd(one.repeat(4, 6), one.repeat(4, 6)))
    row = g_l[:1].expand(4, -1)
    assert torch.equal(bwd(row, row), bwd(row.contiguous(), row.contiguous()))


def test_no_rows():
    from tabpack_b200 import ops

    z = torch.empty(3, 0, 5, device='cuda')
    y = torch.empty(3, 0, dtype=torch.int64, device='cuda')
    lp, H, top, which, stats = ops.label_log_probs_forward(z, y, top_k=2)
    assert lp.shape == H.shape == (3, 0) and top.shape == which.shape == (3, 0, 2)
    assert ops.label_log_probs_backward(lp, None, z, y, stats).shape == z.shape


def test_one_row_without_leading_dimensions():
    z, y, g_l, g_h = make((), 50, torch.float32, seed=5)
    run_and_check(z, y, g_l, g_h, k=3)


def test_gradient_against_differences():
    """The kernel's gradient against central differences of the 64-bit formula, step 1e-5."""
    from tabpack_b200 import nn as tnn

    for C in (12, 300, 2500):
        z, y, a, b = make((3, 4), C, torch.float32, seed=C)
        z.requires_grad_()
        out = tnn.label_log_probs(z, y)
        (out.log_prob * a + out.entropy * b).sum().backward()
        gen = torch.Generator(device='cuda').manual_seed(1)
        v = torch.randn(z.shape, generator=gen, device='cuda', dtype=torch.float64)

        def f(s):
            lp = torch.log_softmax(z.detach().double() + s * v, -1)
            h = -(lp.exp() * lp).sum(-1)
            return (lp.gather(-1, y[..., None])[..., 0] * a + h * b).sum().item()

        slope = (f(1e-5) - f(-1e-5)) / 2e-5
        _, tol = plain(z.detach().reshape(-1, C), y.reshape(-1), 0, a.reshape(-1).double(), b.reshape(-1).double())
        room = ((tol[3].view_as(v) + U * z.grad.abs().double()) * v.abs()).sum().item()
        got = (z.grad.double() * v).sum().item()
        assert abs(got - slope) <= room + 1e-6 * (1 + abs(slope)), (C, got, slope, room)


def test_other_stream_and_graph():
    from tabpack_b200 import ops

    for C in (10, 5000):
        z, y, g_l, g_h = make((3, 50), C, torch.bfloat16, seed=6)

        def step():
            out = ops.label_log_probs_forward(z, y, top_k=4)
            return (*out[:4], ops.label_log_probs_backward(g_l, g_h, z, y, out[-1]))

        want = step()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step()
        torch.cuda.current_stream().wait_stream(s)
        for g, t in zip(got, want):
            assert torch.equal(g, t)
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(step())
            graphs.append(g)
        z.copy_(make((3, 50), C, torch.bfloat16, seed=7)[0])
        want = step()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            for a, t in zip(out, want):
                assert torch.equal(a, t)


def test_split_rows_in_a_graph_and_on_two_streams():
    """Rows spread over clusters, captured and replayed with new scores, and two such calls at once."""
    from tabpack_b200 import ops

    sets = [make((3,), 40000, torch.bfloat16, seed=s)[:2] for s in (31, 32)]
    want = [ops.label_log_probs_forward(z, y, top_k=8) for z, y in sets]
    z, y = (t.clone() for t in sets[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.label_log_probs_forward(z, y, top_k=8)
    for (zs, ys), expected in zip(sets, want):
        z.copy_(zs)
        y.copy_(ys)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (zs, ys), g in zip(streams, sets, got):
            with torch.cuda.stream(s):
                g.append(ops.label_log_probs_forward(zs, ys, top_k=8))
    torch.cuda.synchronize()
    for g, expected in zip(got, want):
        assert all(torch.equal(a, b) for out in g for a, b in zip(out, expected))


# ------------------------------------------------------------------ the function with autograd


def test_function():
    from tabpack_b200 import nn as tnn

    z, y, a, b = make((2, 9), 20, torch.bfloat16, seed=8)
    z = z.clone().requires_grad_()
    out = tnn.label_log_probs(z, y, top_k=3)
    assert out.log_prob.requires_grad and out.entropy.requires_grad
    assert not out.top_log_prob.requires_grad and not out.top_label.requires_grad
    (out.log_prob * a).sum().backward()
    want, tol = plain(z.detach().reshape(-1, 20), y.reshape(-1), 0, a.reshape(-1).double(),
                      torch.zeros(18, dtype=torch.float64, device='cuda'))
    near(z.grad.reshape(-1, 20), want[4], tol[3], 'dlogits', torch.bfloat16)
    z.grad = None
    tnn.label_log_probs(z, y).entropy.sum().backward()
    assert z.grad is not None
    grad, = torch.autograd.grad(tnn.label_log_probs(z, y).log_prob.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_refusals():
    from tabpack_b200 import ops

    z, y, g_l, g_h = make((3, 4), 10, torch.float32)
    for k in (-1, 11, 33):
        with pytest.raises(ValueError):
            ops.label_log_probs_forward(z, y, top_k=k)
    with pytest.raises(ValueError):
        ops.label_log_probs_forward(z.new_zeros(3, 40).repeat(1, 2), y[:, 0], top_k=33)
    with pytest.raises(TypeError):
        ops.label_log_probs_forward(z, y.int())
    with pytest.raises(TypeError):
        ops.label_log_probs_forward(z.half(), y)
    with pytest.raises(ValueError):
        ops.label_log_probs_forward(z, y[:, :3])
    with pytest.raises(ValueError):
        ops.label_log_probs_forward(z[..., :0], y)
    with pytest.raises(ValueError):
        ops.label_log_probs_forward(z, y.cpu())
    z, y, g_l, g_h = make((3, 4), 300, torch.float32)
    stats = ops.label_log_probs_forward(z, y)[-1]
    with pytest.raises(TypeError):
        ops.label_log_probs_backward(g_l.bfloat16(), None, z, y, stats)
    with pytest.raises(TypeError):
        ops.label_log_probs_backward(g_l[:1], None, z, y, stats)
    with pytest.raises(TypeError):
        ops.label_log_probs_backward(g_l, None, z, y, torch.zeros(2, 7, device='cuda'))


def lengths(piece, counts, vector):
    """Rows just below, at and above whole numbers of a block's or cluster's pieces."""
    return [c * piece + d for c in counts for d in (-vector - 1, -1, 0, 1, vector)]


SIZE = {torch.bfloat16: (8, 3), torch.float32: (4, 4)}  # scores of a vector, vectors of a thread in one piece


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R,parts', [(3, 8), (30, 4), (60, 2), (100, 1)])
def test_long_rows_without_best_classes(R, parts, dtype):
    """The forward that loads whole pieces without a check per vector, over clusters of 8, 4 and 2 CTAs and on
    one; rows on 16-byte boundaries and off them."""
    V, U4 = SIZE[dtype]
    piece = 256 * parts * V * U4
    for i, C in enumerate(lengths(piece, [c for c in (2, 3, 5, 7, 9) if 32768 < c * piece - 9][:2], V)):
        run_and_check(*make((R,), C, dtype, seed=C, ld=C + i % 3, masked=0.2 * (i % 2)))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R,threads,classes', [(5, 64, 4200), (5, 128, 9000), (5, 256, 17000), (1184, 64, 6000),
                                               (1184, 128, 20000), (1184, 256, 33000)])
def test_block_sizes_without_best_classes(R, threads, classes, dtype):
    """Blocks of 2, 4 and 8 warps, by the length and the number of the rows."""
    V, U4 = SIZE[dtype]
    piece = threads * V * U4
    for i, C in enumerate(lengths(piece, [classes // piece + 1], V)):
        run_and_check(*make((R,), C, dtype, seed=C, ld=C + i % 3))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('P,B,C', [(4, 6, 5000), (2, 9, 40000), (3, 20, 33001), (40, 30, 1500), (2, 1, 70000)])
def test_shared_labels_of_long_rows_with_best_classes(P, B, C, dtype):
    z, y, g_l, g_h = make((P, B), C, dtype, seed=C)
    run_and_check(z, y[0], g_l, g_h, k=9)
    run_and_check(z, y[0], g_l, g_h)


@pytest.mark.parametrize('R,C,dtype', [(36000, 60001, torch.bfloat16), (4400000, 500, torch.bfloat16),
                                       (9000000, 243, torch.float32), (220000000, 10, torch.bfloat16)])
def test_scores_beyond_32_bits(R, C, dtype):
    """The first and last rows of more than 2^31 scores: long rows, held ones with and without statistics."""
    from tabpack_b200 import ops

    few = 4
    zs, ys, g_l, g_h = make((2 * few,), C, dtype, seed=C)
    z, y = torch.zeros(R, C, dtype=dtype, device='cuda'), torch.zeros(R, dtype=torch.int64, device='cuda')
    gl, gh = torch.zeros(R, device='cuda'), torch.zeros(R, device='cuda')
    at = torch.cat([torch.arange(few, device='cuda'), torch.arange(R - few, R, device='cuda')])
    z[at], y[at], gl[at], gh[at] = zs, ys, g_l, g_h
    k = 3
    lp, H, top, which, stats = ops.label_log_probs_forward(z, y, top_k=k)
    dz = ops.label_log_probs_backward(gl, gh, z, y, stats)
    want, tol = plain(zs, ys, k, g_l.double(), g_h.double())
    near(lp[at], want[0], tol[0], 'log_prob')
    near(H[at], want[1], tol[1], 'entropy')
    near(top[at], want[2], tol[2], 'top_log_prob')
    assert torch.equal(which[at], want[3])
    near(dz[at], want[4], tol[3], 'dlogits', dtype)
    assert not dz[few: R - few].any() and (which[R // 2] == torch.arange(k, device='cuda')).all()
    del z, dz, lp, H, top, which, stats
    torch.cuda.empty_cache()
