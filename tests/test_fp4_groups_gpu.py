"""4-bit rows of ragged groups: the same as each group's rows alone, whatever lies between the groups' tiles."""

import pytest
import torch

from tabpack_b200 import ops

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
