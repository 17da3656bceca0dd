"""Members whose in_features are 0: y = relu(b), no gradient but the bias's."""

import pytest
import torch

from oracle import routed
from tabpack_b200 import ops

pytestmark = pytest.mark.gpu

# sizes of the members' batches, features in, features out: few rows (its K loop on one CTA and over a cluster), many, CTA pairs
SHAPES = [([2, 5, 1, 0], 40, 24), ([3, 1, 2], 4096, 136), ([300, 150, 700], 200, 333), ([130, 257, 100, 33], 64, 40),
          ([2100, 1500, 900], 1104, 1040)]


def data(sizes, K, N, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    P, edges = len(sizes), [1]
    for s in sizes:
        edges.append(edges[-1] + s)
    in_f = torch.randint(1, K + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
    out_f = torch.randint(N // 2, N + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
    in_f[1] = 0
    return normal(edges[-1] + 2, K), normal(P, N, K) * K ** -0.5, normal(P, N), edges, in_f, out_f


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('biased', [False, True])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_ragged_linear(shape, biased, relu, dtype):
    x, w, b, edges, in_f, out_f = data(*SHAPES[shape], shape)
    x, w, b = x.to(dtype), w.to(dtype), b if biased else None
    offsets = torch.tensor(edges, dtype=torch.int32, device='cuda')
    kw = dict(in_features=in_f, out_features=out_f, relu=relu)
    y = ops.ragged_linear_forward(x, w, b, offsets, **kw)
    (want,), _ = routed.ragged_linear(x, w, b, edges, in_f, out_f, relu)
    rows = slice(edges[1], edges[2])
    assert torch.equal(y[rows], want[rows].to(dtype))
    other = in_f.clone()
    other[1] = 1
    again = ops.ragged_linear_forward(x, w, b, offsets, in_features=other, out_features=out_f, relu=relu)
    for m in (0, 2):
        assert torch.equal(y[edges[m]:edges[m + 1]], again[edges[m]:edges[m + 1]])
    dy = torch.randn_like(y)
    dx, dw, db = ops.ragged_linear_backward(dy, x, w, y, offsets, **kw)
    (_, _, want), (_, _, mag) = routed.ragged_linear(x, w, None, edges, in_f, out_f, relu, dy, y)
    assert not dx[rows].any() and not dw[1].any()
    n = edges[2] - edges[1]
    assert ((db.double() - want).abs()[1] <= mag[1] * (n / 8 + 64) * 2.0 ** -24).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('format', ['nvfp4', 'mxfp4'])
@pytest.mark.parametrize('relu,biased', [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_linear_in_4_bits(shape, relu, biased, format, dtype):
    x, w, b, edges, in_f, out_f = data(*SHAPES[shape], shape)
    x, b = x.to(dtype), b if biased else None
    offsets = torch.tensor(edges, dtype=torch.int32, device='cuda')
    weight = ops.fp4_quantize(w, format, n_features=in_f)
    y = ops.fp4_linear_forward(x, weight, b, offsets, in_features=in_f, out_features=out_f, relu=relu)
    want = torch.zeros(w.shape[1], device='cuda') if b is None else b[1].clone()
    want[int(out_f[1]):] = 0.0
    want = (want.relu() if relu else want).to(dtype)
    assert torch.equal(y[edges[1]:edges[2]], want.expand(edges[2] - edges[1], -1))
    assert not y[:1].any() and not y[edges[-1]:].any()
    # equal batches
    y = ops.fp4_linear_forward(x[:5].expand(len(in_f), 5, -1), weight, b, in_features=in_f, out_features=out_f, relu=relu)
    assert torch.equal(y[1], want.expand(5, -1))
