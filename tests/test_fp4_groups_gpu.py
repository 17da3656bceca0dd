"""4-bit rows of ragged groups: the same as each group's rows alone, whatever lies between the groups' tiles."""

import ctypes

import pytest
import torch

from tabpack_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def check(x, edges, format, n_features=None):
    offsets = torch.tensor(edges, dtype=torch.int32, device='cuda')
    q = ops.fp4_quantize(x, format, offsets=offsets, n_features=n_features)
    for g, (a, b) in enumerate(zip(edges, edges[1:])):
        if a == b:
            continue
        alone = ops.fp4_quantize(x[a:b], format, n_features=None if n_features is None else n_features[g:g + 1])
        assert torch.equal(q.codes[a:b], alone.codes)
        assert torch.equal(q.row_scale[a:b], alone.row_scale)
        first = a // 128 + g
        assert torch.equal(q.scales[first:first + len(alone.scales)], alone.scales)


# the numbers of columns give a row 32, 64, 128 and 256 threads; groups of 128 and 256 rows leave a tile without rows behind
# each of them
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('format', ['nvfp4', 'mxfp4'])
@pytest.mark.parametrize('vectors', [100, 130, 300, 521, 1024])
@pytest.mark.parametrize('P,rows', [(64, 256), (100, 128)])
def test_tiles_without_rows_between_groups(P, rows, vectors, format, dtype):
    K = vectors * 16 // torch.finfo(dtype).bits * 8 - (3 if vectors % 2 else 0)
    gen = torch.Generator(device='cuda').manual_seed(P + vectors)
    x = torch.randn(P * rows, K, generator=gen, device='cuda')
    x *= torch.exp2(torch.randint(-20, 20, (P * rows, 1), generator=gen, device='cuda').float())  # maxima far apart
    x = x.to(dtype)
    for _ in range(3):
        check(x, [rows * g for g in range(P + 1)], format)


@pytest.mark.parametrize('format', ['nvfp4', 'mxfp4'])
def test_groups_of_any_size(format):
    gen = torch.Generator(device='cuda').manual_seed(1)
    edges = [3, 3, 130, 131, 131, 259, 643, 643, 1000]
    x = torch.randn(1003, 4500, generator=gen, device='cuda').bfloat16()
    n = torch.tensor([1, 4500, 4, 7, 4499, 2048, 5, 1111], dtype=torch.int32, device='cuda')
    check(x, edges, format)
    check(x, edges, format, n_features=n)


def linear_of_codes(q, weight, bias, dtype, shape, offsets=None, in_f=None, out_f=None, relu=False, shared=False):
    """`tp_fp4_linear_forward` over rows that are in 4 bits already."""
    P, N = weight.row_scale.shape
    y = torch.full(shape, 7.0, dtype=dtype, device='cuda')
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = _lib.Fp4LinearArgs(P=P, K=q.columns, N=N, format=_lib.TP_FP4[q.format], dtype=1 if dtype == torch.bfloat16 else 0,
                           x_shared=int(shared), rows=q.row_scale.numel(), offsets=ptr(offsets), in_features=ptr(in_f), out_features=ptr(out_f),
                           x_codes=ptr(q.codes), x_scales=ptr(q.scales), x_row_scale=ptr(q.row_scale), w_codes=ptr(weight.codes),
                           w_scales=ptr(weight.scales), w_row_scale=ptr(weight.row_scale), bias=ptr(bias), relu=int(relu), y=ptr(y))
    _lib.check(_lib.load().tp_fp4_linear_forward(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), 'tp_fp4_linear_forward')
    return y


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('format', ['nvfp4', 'mxfp4'])
@pytest.mark.parametrize('edges,K,N', [([2, 3, 3, 9], 1040, 72), ([0, 130, 131, 700], 300, 200), ([5, 1300, 1300, 2600], 520, 1104)])
def test_linear_of_rows_in_4_bits(edges, K, N, format, dtype):
    gen = torch.Generator(device='cuda').manual_seed(N)
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    P, R = len(edges) - 1, edges[-1] + 4
    x, w, b = normal(R, K).to(dtype), normal(P, N, K), normal(P, N)
    in_f = torch.tensor([K, K - 9, K // 2], dtype=torch.int32, device='cuda')
    out_f = torch.tensor([N - 3, N, N // 2], dtype=torch.int32, device='cuda')
    offsets = torch.tensor(edges, dtype=torch.int32, device='cuda')
    weight = ops.fp4_quantize(w, format, n_features=in_f)
    q = ops.fp4_quantize(x, format, offsets=offsets, n_features=in_f)
    got = linear_of_codes(q, weight, b, dtype, (R, N), offsets, in_f, out_f, relu=True)
    want = ops.fp4_linear_forward(x, weight, b, offsets, in_features=in_f, out_features=out_f, relu=True)
    assert torch.equal(got, want)
    # equal batches, and one that all members read
    some = x[:min(R, 300) // P * P]
    q = ops.fp4_quantize(some.view(P, -1, K), format)
    weight = ops.fp4_quantize(w, format)
    got = linear_of_codes(q, weight, b, dtype, (P, len(some) // P, N))
    assert torch.equal(got, ops.fp4_linear_forward(some.view(P, -1, K), weight, b))
    got = linear_of_codes(ops.fp4_quantize(some, format), weight, None, dtype, (P, len(some), N), shared=True)
    assert torch.equal(got, ops.fp4_linear_forward(some, weight))
