"""Models of which some layers are in 4 bits, run for selected members with their own maximum width."""

import copy

import pytest
import torch

from tabpack_b200.nn import TabPack, fp4_

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('autocast', [True, False])
@pytest.mark.parametrize('keep', [[], [0], [1], [2], [0, 1], [0, 2], [1, 2], [3], [0, 3]])
def test_kept_layers_with_a_maximum_width(keep, autocast):
    torch.manual_seed(1)
    model = TabPack(n_numerical_features=12, categorical_cardinalities=[], d_out=5, n_blocks=[1, 3, 2, 1],
                    d_block=[64, 40, 33, 24], dropout=0.0, pack_size=4, max_d_block=64).cuda().eval()
    model = copy.deepcopy(model)
    linears = [b.linear for b in model.backbone.blocks] + [model.output]
    fp4_(model, keep=[linears[i] for i in keep])
    x = torch.randn(70, 12, device='cuda')
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16, enabled=autocast):
        whole = model(x, None)
        idx = torch.tensor([3, 1, 2], device='cuda')
        got = model(x, None, idx, max_width=40)
        # the columns that fall away are zeros: only the kept layers' sums may come in another order, and rows near a
        # rounding's middle go either way by one step of 4 bits
        assert got.shape == (3, 70, 5) and torch.isfinite(got).all()
        if not keep:
            assert torch.equal(got, whole[idx])
        else:
            error = (got.float() - whole[idx].float()).norm() / whole[idx].float().norm()
            assert error < 0.05
