"""Offsets that decrease, in the ragged linear layers: a member of negative length has no rows, and takes none from the members
behind it.  (Rows in 4 bits are laid out by offsets that do not decrease.)"""

import pytest
import torch

from tabpack_b200 import ops

pytestmark = pytest.mark.gpu

# (offsets, the same without the decrease)
CASES = [([8, 3, 10], [3, 3, 10]), ([9, 0, 9], [0, 0, 9]), ([40000, 0, 40000], [0, 0, 40000]), ([300, 20, 20, 260], [20, 20, 20, 260]),
         ([5000] * 40 + [7, 4000, 5000], [7] * 40 + [7, 4000, 5000])]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('case', range(len(CASES)))
def test_first_members_without_rows(case, dtype):
    offsets, plain = (torch.tensor(o, dtype=torch.int32, device='cuda') for o in CASES[case])
    R, P, K, N = max(CASES[case][0]) + 3, len(offsets) - 1, 72, 264
    gen = torch.Generator(device='cuda').manual_seed(case)
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    x, w, b, dy = normal(R, K).to(dtype), normal(P, N, K).to(dtype), normal(P, N), normal(R, N).to(dtype)
    for _ in range(5):
        assert torch.equal(ops.ragged_linear_forward(x, w, b, offsets), ops.ragged_linear_forward(x, w, b, plain))
        for got, want in zip(ops.ragged_linear_backward(dy, x, w, None, offsets), ops.ragged_linear_backward(dy, x, w, None, plain)):
            assert torch.equal(got, want)
