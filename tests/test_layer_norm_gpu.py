"""Packed layer norm on the GPU against the formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32): a sum of n terms whose longest chain has d
additions is off by at most d u times the sum of magnitudes.  The row sums have chains of at most
D = 96 additions for every width tested here.  So the mean is off by D u mean|x|, the reciprocal
deviation by (D + 4) u relative, and with A = mean|x| rstd
    |xhat error| <= u (2 D + 8) (|xhat| + A)
which the bounds below carry through the formulas term by term.  The parameters' gradients are sums
over the rows, chains of at most B additions.  On top comes half a step of the output's type.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
D = 96


@pytest.fixture(scope='module', autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def plain(x, w, b, n, eps, dy=None):
    """float64 forward and backward of one member's rows, and the magnitudes of the tolerances."""
    B, W = x.shape
    y, dx, dw, db = (torch.zeros(s, dtype=torch.float64, device=x.device) for s in ((B, W), (B, W), (W,), (W,)))
    ty, tdx, tdw, tdb = (torch.zeros_like(t) for t in (y, dx, dw, db))
    x = x[:, :n].double()
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w[:n].double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b[:n].double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xhat = (x - mean) * rstd
    y[:, :n] = xhat * w + b
    size = xhat.abs() + x.abs().mean(1, keepdim=True) * rstd
    ty[:, :n] = U * ((2 * D + 8) * size * w.abs() + 2 * b.abs() + 2 * y[:, :n].abs())
    if dy is not None:
        dy = dy[:, :n].double()
        g = dy * w
        c1, c2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
        dx[:, :n] = rstd * (g - c1 - xhat * c2)
        m1, m2 = g.abs().mean(1, keepdim=True), (g.abs() * size).mean(1, keepdim=True)
        tdx[:, :n] = U * (6 * D + 40) * rstd * (g.abs() + m1 + size * m2)
        dw[:n], db[:n] = (dy * xhat).sum(0), dy.sum(0)
        tdw[:n] = U * (B + 2 * D + 16) * (dy.abs() * size).sum(0)
        tdb[:n] = U * (B + 4) * dy.abs().sum(0)
    return (y, dx, dw, db), (ty, tdx, tdw, tdb)


def check(got, want, tol, dtype, what):
    assert got.dtype == dtype, what
    diff = (got.double() - want).abs()
    bound = tol + half_step(dtype) * want.abs() + 2.0**-133
    assert torch.isfinite(got).all(), what
    assert (diff <= bound).all(), (what, (diff - bound).max().item(), diff.max().item())


def make(P, B, W, dtype, *, shared=False, ragged=True, seed=0, offset=0.5, ld=None):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    ld = W if ld is None else ld
    x = (torch.randn(*((B,) if shared else (P, B)), ld, generator=gen, device='cuda') * 1.7 + offset).to(dtype)[..., :W]
    dy = torch.randn(P, B, ld, generator=gen, device='cuda').to(dtype)[..., :W]
    w = 1 + 0.3 * torch.randn(P, W, generator=gen, device='cuda')
    b = 0.3 * torch.randn(P, W, generator=gen, device='cuda')
    n = None
    if ragged:
        n = torch.randint(1, W + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
        n[0] = W
        n[-1] = max(1, W // 3)
    return x, dy, w, b, n


def run_and_check(x, dy, w, b, n, eps=1e-5):
    from tabpack_b200 import ops

    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n, eps=eps)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n)
    P, B, W = dy.shape
    shared = x.ndim == 2
    sum_dx = tol_dx = 0
    for m in range(P):
        nm = W if n is None else int(n[m])
        want, tol = plain(x if shared else x[m], None if w is None else w[m], None if b is None else b[m], nm, eps,
                          dy[m])
        check(y[m], want[0], tol[0], x.dtype, f'y of member {m}')
        assert (y[m, :, nm:] == 0).all()
        if shared:
            sum_dx, tol_dx = sum_dx + want[1], tol_dx + tol[1] + U * (P + 1) * want[1].abs()
        else:
            check(dx[m], want[1], tol[1], x.dtype, f'dx of member {m}')
            assert (dx[m, :, nm:] == 0).all()
        check(dw[m], want[2], tol[2], torch.float32, f'dw of member {m}')
        check(db[m], want[3], tol[3], torch.float32, f'db of member {m}')
        assert (dw[m, nm:] == 0).all() and (db[m, nm:] == 0).all()
    if shared:
        assert dx.shape == x.shape
        check(dx, sum_dx, tol_dx, x.dtype, 'dx of the shared input')


WIDTHS = [1, 2, 7, 8, 33, 64, 65, 100, 256, 257, 511, 512, 768, 1000, 1024, 1025, 2040, 2049, 4096, 4100, 8192, 8200]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('W', WIDTHS)
def test_widths(W, dtype):
    run_and_check(*make(3, 5, W, dtype, seed=W))


@pytest.mark.parametrize('W', [16384, 16385, 20000])
def test_very_wide(W):
    run_and_check(*make(1, 3, W, torch.bfloat16, ragged=False, seed=1))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('P,B', [(1, 1), (1, 333), (40, 1), (5, 70), (2, 1500), (300, 3)])
@pytest.mark.parametrize('W', [48, 200, 520])
def test_rows_and_members(P, B, W, dtype):
    run_and_check(*make(P, B, W, dtype, seed=P + B))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('P,B', [(2, 1), (3, 63), (2, 64), (2, 65), (1, 1000), (70, 33)])
@pytest.mark.parametrize('W', [3, 16, 63, 64, 72, 128, 131, 136, 255, 256])
def test_narrow_rows(W, P, B, dtype):
    """Groups of 4, 8 and 16 lanes, whole and odd vectors, around a block's number of groups."""
    run_and_check(*make(P, B, W, dtype, seed=W + B))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('shared', [False, True])
@pytest.mark.parametrize('W,ld,at', [(12, 20, 0), (12, 20, 1), (12, 20, 2), (12, 20, 4), (20, 22, 0), (20, 22, 2), (10, 16, 6),
                                     (100, 104, 4), (300, 304, 2), (1204, 1206, 2), (4002, 4004, 2)])
def test_rows_on_every_boundary(W, ld, at, shared, dtype):
    """Column slices at an offset: rows on boundaries of 2, 4, 8 and 16 bytes."""
    x, dy, w, b, n = make(4, 21, ld, dtype, shared=shared, seed=W + at)
    n = (n * W // ld).clamp(min=1).to(torch.int32)
    cut = lambda t: t[..., at:at + W]  # noqa: E731
    run_and_check(cut(x), cut(dy), cut(w).contiguous(), cut(b).contiguous(), n)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('W', [24, 130, 1024])
def test_shared_input(W, dtype):
    run_and_check(*make(6, 37, W, dtype, shared=True, seed=W))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('P,B,W', [(1, 5, 70), (2, 1, 1), (7, 333, 771), (300, 3, 65), (3, 600, 1024), (2, 3, 8200)])
def test_members_of_a_shared_input(P, B, W, dtype):
    """One member (no sum), few and many, an odd and a whole number of vectors."""
    run_and_check(*make(P, B, W, dtype, shared=True, seed=P + W))


@pytest.mark.parametrize('P,B', [(0, 3), (3, 0)])
def test_shared_input_without_rows_or_members(P, B):
    from tabpack_b200 import ops

    x, stat = torch.ones(B, 8, device='cuda'), torch.ones(P, B, device='cuda')
    dx, dw, db = ops.layer_norm_backward(torch.ones(P, B, 8, device='cuda'), x, None, stat, stat)
    assert torch.equal(dx, torch.zeros(B, 8, device='cuda'))
    assert torch.equal(dw, torch.zeros(P, 8, device='cuda')) and torch.equal(db, dw)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('W,ld', [(10, 16), (100, 104), (104, 112), (300, 301), (64, 65), (2000, 2008)])
def test_rows_of_padded_buffers(W, ld, dtype):
    """Column slices of wider buffers: rows that are not packed, aligned and not; the buffer's other
    columns hold NaN, as does the padding beyond each member's width."""
    x, dy, w, b, n = make(3, 11, W, dtype, ld=ld, seed=W)
    for t in (x, dy):
        base = torch.full((3, 11, ld), float('nan'), device='cuda', dtype=dtype)
        view = base[..., :W]
        view.copy_(t)
        for m in range(3):
            view[m, :, int(n[m]):] = float('nan')
        if t is x:
            x = view
        else:
            dy = view
    for m in range(3):
        w[m, int(n[m]):] = b[m, int(n[m]):] = float('nan')
    run_and_check(x, dy, w, b, n)


def test_storage_offset_breaks_alignment():
    x, dy, w, b, n = make(2, 9, 64, torch.bfloat16, seed=3)
    flat = torch.empty(2 * 9 * 64 + 1, dtype=torch.bfloat16, device='cuda')[1:].view(2, 9, 64)
    flat.copy_(x)
    wide = torch.empty(2 * 64 + 1, device='cuda')[1:].view(2, 64)
    wide.copy_(w)
    run_and_check(flat, dy, wide, b, n)


def test_transposed_input_is_copied():
    x, dy, w, b, n = make(2, 9, 40, torch.float32, seed=4)
    run_and_check(x.transpose(1, 2).contiguous().transpose(1, 2), dy, w, b, n)


def test_expanded_gradient():
    """The gradient of y.sum(): one value for every element."""
    from tabpack_b200 import ops

    x, _, w, b, n = make(2, 9, 64, torch.float32, seed=5)
    run_and_check(x, torch.ones((), device='cuda').expand(2, 9, 64), w, b, n)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
    got = ops.layer_norm_backward(torch.ones(2, 1, 64, device='cuda').expand(2, 9, 64), x, w, mean, rstd, n_features=n)
    want = ops.layer_norm_backward(torch.ones(2, 9, 64, device='cuda'), x, w, mean, rstd, n_features=n)
    for g, t in zip(got, want):
        assert torch.equal(g, t)


@pytest.mark.parametrize('has_w,has_b', [(False, False), (True, False), (False, True)])
def test_without_parameters(has_w, has_b):
    x, dy, w, b, n = make(3, 17, 96, torch.bfloat16, seed=6)
    run_and_check(x, dy, w if has_w else None, b if has_b else None, n)


def test_large_mean():
    """Rows far from zero: the squares' sum minus the squared sum would lose every digit."""
    run_and_check(*make(2, 6, 700, torch.float32, offset=3000.0, seed=7))


def test_constant_rows():
    """No variance: y = b, and the gradient is bounded by 1 / sqrt(eps)."""
    from tabpack_b200 import ops

    x, dy, w, b, n = make(2, 6, 72, torch.float32, seed=8)
    x.fill_(0.25)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
    assert (mean == 0.25).all()
    assert torch.allclose(rstd, torch.full_like(rstd, 1e-5**-0.5), rtol=1e-6)
    for m in range(2):
        assert torch.equal(y[m, :, : int(n[m])], b[m, : int(n[m])].expand(6, -1))
    run_and_check(x, dy, w, b, n)


def test_nonfinite_rows_stay_by_themselves():
    from tabpack_b200 import ops

    x, dy, w, b, n = make(2, 40, 200, torch.bfloat16, ragged=False, seed=9)
    clean = ops.layer_norm_forward(x, w, b)[0]
    x[0, 3, 5], x[1, 7, 199] = float('nan'), float('inf')
    y = ops.layer_norm_forward(x, w, b)[0]
    bad = torch.zeros(2, 40, dtype=torch.bool, device='cuda')
    bad[0, 3] = bad[1, 7] = True
    assert torch.isnan(y[bad]).all()
    assert torch.equal(y[~bad], clean[~bad])


def test_padding_of_nonfinite_rows_is_zero():
    from tabpack_b200 import ops

    for W, dtype in ((200, torch.bfloat16), (200, torch.float32), (77, torch.float32), (3000, torch.bfloat16),
                     (9000, torch.bfloat16)):
        x, dy, w, b, n = make(2, 6, W, dtype, seed=W)
        n[0], n[1] = W - 5, W // 2
        x[0, 1, 3], x[1, 2, 0], dy[0, 4, 2] = float('nan'), float('inf'), float('nan')
        y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
        dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n)
        for m in range(2):
            k = int(n[m])
            for t in (y[m], dx[m], dw[m:m + 1], db[m:m + 1]):
                assert (t[..., k:] == 0).all()
        assert torch.isnan(y[0, 1, :k]).all() and torch.isnan(dx[0, 4, :k]).all() and torch.isnan(dw[1, :k]).all()
        assert torch.isfinite(db[1]).all() and torch.isfinite(y[0, 4]).all()


def test_widths_outside_the_row_are_clamped():
    """A width of zero leaves zeros; one beyond the row is the row."""
    from tabpack_b200 import ops

    x, dy, w, b, _ = make(3, 6, 50, torch.float32, seed=10)
    n = torch.tensor([0, 50, 60], dtype=torch.int32, device='cuda')
    full = torch.tensor([1, 50, 50], dtype=torch.int32, device='cuda')
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
    got = (y, *ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n))
    y2, mean2, rstd2 = ops.layer_norm_forward(x, w, b, n_features=full)
    want = (y2, *ops.layer_norm_backward(dy, x, w, mean2, rstd2, n_features=full))
    for g, t in zip(got, want):
        assert (g[0] == 0).all()
        assert torch.equal(g[1:], t[1:])


@pytest.mark.parametrize('P,B', [(0, 5), (3, 0)])
def test_no_rows(P, B):
    from tabpack_b200 import ops

    x = torch.empty(P, B, 16, device='cuda')
    w = torch.ones(P, 16, device='cuda')
    y, mean, rstd = ops.layer_norm_forward(x, w, w)
    dx, dw, db = ops.layer_norm_backward(torch.empty_like(y), x, w, mean, rstd)
    assert y.shape == dx.shape == (P, B, 16) and (dw == 0).all() and (db == 0).all()


def test_needs():
    from tabpack_b200 import ops

    x, dy, w, b, n = make(3, 50, 96, torch.bfloat16, seed=11)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
    want = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n)
    for need in [(True, False, False), (False, True, False), (False, False, True), (False, True, True)]:
        got = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n, need_dx=need[0], need_dw=need[1],
                                      need_db=need[2])
        for g, t, k in zip(got, want, need):
            assert (g is None) != k
            assert g is None or torch.equal(g, t)


def test_repeatable():
    from tabpack_b200 import ops

    x, dy, w, b, n = make(2, 3000, 512, torch.bfloat16, seed=12)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
    first = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n)
    for _ in range(3):
        for g, t in zip(ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n), first):
            assert torch.equal(g, t)


def test_gradient_against_differences():
    """The kernels' gradients against central differences of the 64-bit formula (step 1e-5: their
    error, about 1e-10, is far below the fp32 bounds summed over the elements)."""
    from tabpack_b200 import ops

    x, dy, w, b, n = make(2, 7, 45, torch.float32, seed=13)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n)
    gen = torch.Generator(device='cuda').manual_seed(1)
    vx, vw, vb = (torch.randn(t.shape, generator=gen, device='cuda', dtype=torch.float64) for t in (x, w, b))
    h = 1e-5

    def f(s):
        total = 0.0
        for m in range(2):
            want, _ = plain(x[m].double() + s * vx[m], w[m].double() + s * vw[m], b[m].double() + s * vb[m],
                            int(n[m]), 1e-5)
            total += (want[0] * dy[m].double()).sum().item()
        return total

    slope = (f(h) - f(-h)) / (2 * h)
    got = sum((g.double() * v).sum().item() for g, v in ((dx, vx), (dw, vw), (db, vb)))
    room = 0.0
    for m in range(2):
        _, tol = plain(x[m], w[m], b[m], int(n[m]), 1e-5, dy[m])
        for t, v, g in zip(tol[1:], (vx[m], vw[m], vb[m]), (dx[m], dw[m], db[m])):
            room += ((t + U * g.abs().double()) * v.abs()).sum().item()
    assert abs(got - slope) <= room + 1e-6 * abs(slope), (got, slope, room)


def test_other_stream_and_graph():
    """On a side stream, and captured twice into graphs that replay with new inputs."""
    from tabpack_b200 import ops

    x, dy, w, b, n = make(2, 700, 320, torch.bfloat16, seed=14)

    def step():
        y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
        return (y, *ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n))

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
    x2 = make(2, 700, 320, torch.bfloat16, seed=15)[0]
    x.copy_(x2)
    want = step()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for out in outs:
        for a, t in zip(out, want):
            assert torch.equal(a, t)


# ------------------------------------------------------------------ the module


def test_module_against_plain_autograd():
    from tabpack_b200 import nn as tnn

    widths = [40, 72, 9]
    pack = tnn.LayerNormPack(widths, max_n_features=72, pack_size=3).cuda()
    gen = torch.Generator(device='cuda').manual_seed(2)
    with torch.no_grad():
        pack.weight.copy_(1 + 0.2 * torch.randn(3, 72, generator=gen, device='cuda'))
        pack.bias.copy_(0.2 * torch.randn(3, 72, generator=gen, device='cuda'))
    x = torch.randn(3, 30, 72, generator=gen, device='cuda', requires_grad=True)
    c = torch.randn(3, 30, 72, generator=gen, device='cuda')
    y = pack(x)
    (y * c).sum().backward()
    for m, nm in enumerate(widths):
        want, tol = plain(x.detach()[m], pack.weight.detach()[m], pack.bias.detach()[m], nm, pack.eps, c[m])
        for got, t, to, what in zip((y[m], x.grad[m], pack.weight.grad[m], pack.bias.grad[m]), want, tol,
                                    ('y', 'dx', 'dw', 'db')):
            check(got.detach(), t, to, torch.float32, what)


def test_module_selection_and_replacement():
    from tabpack_b200 import nn as tnn

    pack = tnn.LayerNormPack([8, 16, 24, 32], pack_size=4).cuda().eval()
    assert pack.max_n_features == 32 and pack.pack_size == 4
    x = torch.randn(4, 5, 32, device='cuda')
    with torch.no_grad():
        pack.weight.copy_(torch.rand(4, 32, device='cuda'))
        full = pack(x)
        idx = torch.tensor([2, -4], device='cuda')
        assert torch.equal(pack(x[idx], idx), full[idx])
        with pack.temporarily_select(pack_idx=idx):
            assert pack.pack_size == 2
            assert torch.equal(pack(x[idx]), full[idx])
        assert torch.equal(pack(x), full)
        pack.replace(pack_idx=torch.tensor([1], device='cuda'), n_features=[30])
        assert pack.n_features.tolist() == [8, 30, 24, 32] and (pack.weight[1] == 1).all()
        changed = pack(x)
        assert torch.equal(changed[[0, 2, 3]], full[[0, 2, 3]]) and (changed[1, :, 16:30] != 0).any()
        pack.remove(pack_idx=torch.tensor([0], device='cuda'))
        assert pack.pack_size == 3
        assert torch.equal(pack(x[1:]), changed[1:])


def test_module_shared_rows():
    """An expanded input: y as for a copied one, and the gradient of the rows is the sum."""
    from tabpack_b200 import nn as tnn

    pack = tnn.LayerNormPack([20, 33], max_n_features=33, pack_size=2).cuda()
    rows = torch.randn(12, 33, device='cuda')
    c = torch.randn(2, 12, 33, device='cuda')
    one = rows.clone().requires_grad_()
    y1 = pack(tnn.PackView(pack_size=2).train()(one))
    (y1 * c).sum().backward()
    each = rows.expand(2, -1, -1).contiguous().requires_grad_()
    y2 = pack(each)
    (y2 * c).sum().backward()
    assert torch.equal(y1, y2)
    room = sum(plain(rows, None, None, k, pack.eps, c[m])[1][1] for m, k in enumerate([20, 33]))
    assert ((one.grad.double() - each.grad.double().sum(0)).abs() <= 2 * room + 4 * U * each.grad.abs().sum(0)).all()
    half = rows.bfloat16().requires_grad_()
    assert pack(half[None]).dtype == torch.bfloat16
    pack(half[None]).sum().backward()
    assert half.grad.dtype == torch.bfloat16 and half.grad.shape == rows.shape


def test_module_without_parameters():
    from tabpack_b200 import nn as tnn

    pack = tnn.LayerNormPack(24, elementwise_affine=False, pack_size=3).cuda()
    assert list(pack.parameters()) == []
    x = torch.randn(5, 24, device='cuda')
    y = pack(x.expand(3, -1, -1))
    assert y.shape == (3, 5, 24) and torch.equal(y[0], y[2])
    want, tol = plain(x, None, None, 24, pack.eps)
    check(y[1], want[0], tol[0], torch.float32, 'y')


def test_refusals():
    from tabpack_b200 import nn as tnn
    from tabpack_b200 import ops

    x, dy, w, b, n = make(2, 4, 16, torch.float32)
    with pytest.raises(ValueError):
        ops.layer_norm_forward(x[0, 0], w, b)
    with pytest.raises(ValueError):
        ops.layer_norm_forward(x, w[:, :8], b)
    with pytest.raises(ValueError):
        ops.layer_norm_forward(x, w, b, n_features=n[:1])
    with pytest.raises(ValueError):
        ops.layer_norm_forward(x, w, b, eps=-1.0)
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x.half(), w, b)
    with pytest.raises(TypeError):
        ops.layer_norm_forward(x, w.bfloat16(), b)
    with pytest.raises(ValueError):
        ops.layer_norm_forward(x, w.cpu(), b)
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    with pytest.raises(TypeError):
        ops.layer_norm_backward(dy.bfloat16(), x, w, mean, rstd)
    with pytest.raises(TypeError):
        ops.layer_norm_backward(dy, x, w, mean[:1], rstd)
    with pytest.raises(ValueError):
        ops.layer_norm_backward(dy[:, :3], x, w, mean, rstd)
    pack = tnn.LayerNormPack([8, 16], pack_size=2).cuda()
    with pytest.raises(ValueError):
        pack(x[0])
    with pytest.raises(ValueError):
        pack(x[..., :8])
    with pytest.raises(ValueError):
        pack(torch.zeros(3, 4, 16, device='cuda'))
    out = pack(x.requires_grad_())
    grad, = torch.autograd.grad(out.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('W,n,B,value,eps', [
    (W, n, B, 2.0**80, 1e-30) for W, n, B in [(72, 64, 40), (77, 64, 70), (300, 256, 9), (301, 256, 19), (2000, 1024, 5),
                                              (2001, 1024, 3), (4096, 4096, 7), (6000, 4096, 2), (9000, 8192, 3)]
] + [(72, 64, 40, 2.0**120, 1e-5), (77, 64, 70, 2.0**120, 1e-5)])
def test_large_constant_rows(W, n, B, value, eps, dtype):
    """Rows of one large power of two, as many columns as a power of two: mean and variance are exact, xhat is 0
    (64 x 2^120 and 8192 x 2^80 are numbers of fp32).  |mean| rstd leaves the fp32 range, so a column that is not
    part of the row, taken as x = 0, would bring in an infinity.  dx = rstd (dy w - mean(dy w)): D + 16 roundings
    of the magnitudes."""
    from tabpack_b200 import ops

    x, dy, w, b, _ = make(2, B, W, dtype, ragged=False, seed=W)
    x.fill_(value)
    k = torch.full((2,), n, dtype=torch.int32, device='cuda')
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=k, eps=eps)
    assert (mean == value).all()
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=k)
    assert torch.equal(y[..., :n], b[:, None, :n].to(dtype).expand(2, B, n)) and (y[..., n:] == 0).all()
    assert torch.equal(dw, torch.zeros_like(dw)) and (db[:, n:] == 0).all()
    dy64 = dy[..., :n].double()
    g, r = dy64 * w[:, None, :n].double(), 1 / float(eps) ** 0.5
    want = r * (g - g.mean(2, keepdim=True))
    tol = U * (D + 16) * r * (g.abs() + g.abs().mean(2, keepdim=True))
    check(dx[..., :n], want, tol, dtype, 'dx')
    check(db[:, :n], dy64.sum(1), U * (B + 4) * dy64.abs().sum(1), torch.float32, 'db')
    assert (dx[..., n:] == 0).all()


def test_large_constant_rows_of_a_shared_input():
    from tabpack_b200 import ops

    x, dy, w, b, _ = make(3, 21, 72, torch.float32, shared=True, seed=1)
    x.fill_(2.0**120)
    k = torch.full((3,), 64, dtype=torch.int32, device='cuda')
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=k)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=k)
    g = dy[..., :64].double() * w[:, None, :64].double()
    r = 1e-5**-0.5
    want = (r * (g - g.mean(2, keepdim=True))).sum(0)
    size = (r * (g.abs() + g.abs().mean(2, keepdim=True))).sum(0)
    check(dx[:, :64], want, U * (D + 20) * size, torch.float32, 'dx')
    assert (dx[:, 64:] == 0).all() and (dw == 0).all() and torch.isfinite(db).all()


@pytest.mark.parametrize('P', [2, 64])
def test_module_without_parameters_adds_a_shared_gradient_in_fp32(P):
    """bf16 rows that the members share: their gradient is rounded once, whatever the number of members."""
    from tabpack_b200 import nn as tnn

    pack = tnn.LayerNormPack(24, elementwise_affine=False, pack_size=P).cuda()
    x = torch.randn(5, 24, device='cuda').bfloat16().requires_grad_()
    dy = torch.randn(P, 5, 24, device='cuda').bfloat16()
    y = pack(x.expand(P, -1, -1))
    assert y.shape == (P, 5, 24)
    y.backward(dy)
    want = tol = 0
    for m in range(P):
        one, room = plain(x.detach(), None, None, 24, pack.eps, dy[m])
        want, tol = want + one[1], tol + room[1] + U * (P + 1) * one[1].abs()
        check(y[m].detach(), one[0], room[0], torch.bfloat16, f'y of member {m}')
    check(x.grad, want, tol, torch.bfloat16, 'dx')
    # selected members, and rows with a pack dimension of their own
    idx = torch.arange(P - 1, device='cuda')
    assert torch.equal(pack(x.detach().expand(P - 1, -1, -1), idx), y.detach()[:-1])
    assert torch.equal(pack(x.detach()[None]), y.detach()[:1])
    assert torch.equal(pack(x.detach().repeat(P, 1, 1)), y.detach())


def test_pack_size_of_a_shared_input():
    from tabpack_b200 import ops

    x, _, w, _, _ = make(3, 6, 16, torch.float32, shared=True, ragged=False, seed=2)
    one, mean, rstd = ops.layer_norm_forward(x, None, None)
    y, means, rstds = ops.layer_norm_forward(x, None, None, pack_size=3)
    assert one.shape == (1, 6, 16) and y.shape == (3, 6, 16) and means.shape == rstds.shape == (3, 6)
    for m in range(3):
        assert torch.equal(y[m], one[0]) and torch.equal(means[m], mean[0]) and torch.equal(rstds[m], rstd[0])
    assert torch.equal(ops.layer_norm_forward(x, w, None, pack_size=3)[0], ops.layer_norm_forward(x, w, None)[0])
    for args in ((x, w, None), (x.expand(3, -1, -1), None, None), (x, None, None)):
        with pytest.raises(ValueError):
            ops.layer_norm_forward(*args, pack_size=-1 if args[0].ndim == 2 and args[1] is None else 2)


# Many members, so that a member's rows are split little: a group of every number of lanes (4 to 512)
# takes 4 to 20 pairs of rows forward and 8 to 40 rows backward, several times round the rows on their way
# (3 pairs and 4 rows in bf16, 2 and 2 in fp32); on boundaries of 16 bytes and off them.
MANY_ROUNDS = [(300, 2300, 48), (300, 2301, 63), (300, 2299, 50), (300, 1100, 128), (300, 1201, 100), (300, 700, 256),
               (300, 701, 203), (300, 350, 512), (64, 1024, 512), (300, 351, 331), (300, 170, 1024), (300, 171, 771),
               (300, 90, 2048), (300, 91, 1500), (300, 50, 4096), (300, 51, 2501), (150, 40, 8192), (150, 41, 5001),
               (296, 40, 4100)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('P,B,W', MANY_ROUNDS)
def test_many_rounds(P, B, W, dtype):
    x, dy, w, b, n = make(P, B, W, dtype, seed=W + B)
    x, dy = x.clone(), dy.clone()
    for m in range(0, P, 7):
        x[m, :, int(n[m]):] = dy[m, :, int(n[m]):] = float('nan')
    run_and_check(x, dy, w, b, n)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('P,B,W', [(300, 700, 256), (300, 90, 2048)])
def test_many_rounds_of_rows_apart(P, B, W, dtype):
    """Rows of a wider buffer, on every boundary that they can start on."""
    for ld, at in ((W + 8, 8), (W + 4, 4), (W + 2, 2), (W + 1, 1)):
        x, dy, w, b, n = make(P, B, ld, dtype, seed=ld)
        n = (n * W // ld).clamp(min=1).to(torch.int32)
        cut = lambda t: t[..., at:at + W]  # noqa: E731
        run_and_check(cut(x), cut(dy), cut(w).contiguous(), cut(b).contiguous(), n)


@pytest.mark.parametrize('P,B,W,dtype', [(2, 140000, 8000, torch.bfloat16), (3, 1000000, 771, torch.float32),
                                         (3, 80000, 9001, torch.bfloat16)])
def test_elements_beyond_32_bits(P, B, W, dtype):
    """The last rows of more than 2^31 elements, forward and backward, and the parameters' gradients where only
    those rows have one."""
    from tabpack_b200 import ops

    few = 5
    xs, dys, w, b, n = make(P, few, W, dtype, seed=W)
    x, dy = (torch.zeros(P, B, W, dtype=dtype, device='cuda') for _ in range(2))
    x[:, B - few:], dy[:, B - few:] = xs, dys
    y, mean, rstd = ops.layer_norm_forward(x, w, b, n_features=n)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd, n_features=n)
    for m in range(P):
        k = int(n[m])
        want, tol = plain(xs[m], w[m], b[m], k, 1e-5, dys[m])
        check(y[m, B - few:], want[0], tol[0], dtype, 'y')
        check(dx[m, B - few:], want[1], tol[1], dtype, 'dx')
        check(dw[m], want[2], tol[2], torch.float32, 'dw')
        check(db[m], want[3], tol[3], torch.float32, 'db')
        assert torch.equal(y[m, B // 2, :k], b[m, :k].to(dtype)) and not dx[m, : B - few].any()
    del x, dy, y, dx, mean, rstd
    torch.cuda.empty_cache()
