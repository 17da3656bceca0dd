"""4-bit linear layers of rows far from 1: scaling x up and w down by powers of two changes nothing."""

import pytest
import torch

from tabpack_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('format', ['nvfp4', 'mxfp4'])
@pytest.mark.parametrize('up,down', [(118, 80), (-80, -100), (60, 60), (100, 60)])
@pytest.mark.parametrize('sizes,K,N', [([1, 5], 1000, 136), ([1], 4096, 520), ([300, 140], 260, 333), ([3000], 520, 1104)])
def test_scaled_operands(sizes, K, N, up, down, format, dtype):
    gen = torch.Generator(device='cuda').manual_seed(N)
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    P, R = len(sizes), sum(sizes)
    x, w = normal(R, K).clamp(-7, 7).to(dtype), normal(P, N, K).clamp(-7, 7)
    edges = torch.tensor([0] + sizes, device='cuda').cumsum(0).int()
    plain = ops.fp4_linear_forward(x, ops.fp4_quantize(w, format), None, edges)
    assert torch.isfinite(plain).all()
    got = ops.fp4_linear_forward(x * 2.0 ** up, ops.fp4_quantize(w * 2.0 ** -down, format), None, edges)
    assert torch.equal(got, plain * 2.0 ** (up - down))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('sizes,K,N', [([1, 5], 1000, 136), ([300, 140], 260, 333), ([3000], 520, 1104)])
def test_sums_of_zero_and_overflows(sizes, K, N, dtype):
    P, R = len(sizes), sum(sizes)
    x, w, b = torch.zeros(R, K, device='cuda'), torch.zeros(P, N, K, device='cuda'), torch.randn(P, N, device='cuda')
    x[:, 0], w[:, :, 1] = 2.0 ** 120, 2.0 ** 120  # 0
    x[:, 2], w[:, 3::4, 2] = 2.0 ** 120, 2.0 ** 117  # beyond the largest number
    x[:, 2] *= torch.where(torch.arange(R, device='cuda') % 2 == 0, 1.0, -1.0)
    edges = torch.tensor([0] + sizes, device='cuda').cumsum(0).int()
    y = ops.fp4_linear_forward(x.to(dtype), ops.fp4_quantize(w), b, edges)
    want = torch.cat([b[m].expand(n, N) for m, n in enumerate(sizes)]).clone()
    want[0::2, 3::4], want[1::2, 3::4] = torch.inf, -torch.inf
    assert torch.equal(y, want.to(dtype))
