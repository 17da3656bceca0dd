"""What a module keeps from call to call (int32 widths, bf16 weights) belongs to one tensor: a member
selection installs tensors of its own, which may lie where the last selection's lay (no GPU)."""

import numpy as np
import pytest
import torch

from tabpack_b200.nn import LayerNormPack, LinearPack, _widths_cached


def test_widths_of_another_buffer_at_the_same_address():
    module = torch.nn.Module()
    memory = np.array([3, 5, 7])
    first = torch.from_numpy(memory)
    assert _widths_cached(module, 'n', first).tolist() == [3, 5, 7]
    address = first.data_ptr()
    del first
    memory[:] = [8, 2, 4]
    second = torch.from_numpy(memory)
    assert second.data_ptr() == address and second._version == 0
    assert _widths_cached(module, 'n', second).tolist() == [8, 2, 4]


@pytest.mark.parametrize('make,name', [
    (lambda n: LayerNormPack(n, max_n_features=64, pack_size=len(n)), 'n_features'),
    (lambda n: LinearPack(4, n, max_out_features=64, pack_size=len(n)), 'out_features')])
@pytest.mark.parametrize('k', [3, 40, 300])
def test_widths_of_selections_in_a_row(make, name, k):
    widths = [1 + (17 * i + i // 64) % 64 for i in range(3000)]
    pack = make(widths).eval()
    for i in range(20):
        idx = torch.arange(k) * 7 + 31 * i
        with pack.temporarily_select(pack_idx=idx):
            got = _widths_cached(pack, 'w', getattr(pack, name))
            assert got.dtype == torch.int32 and got.tolist() == [widths[j] for j in idx]
    assert _widths_cached(pack, 'w', getattr(pack, name)).tolist() == widths


def test_widths_are_kept_until_the_buffer_changes():
    module, buf = torch.nn.Module(), torch.tensor([3, 5])
    first = _widths_cached(module, 'n', buf)
    assert _widths_cached(module, 'n', buf) is first and _widths_cached(module, 'n', None) is None
    buf[0] = 4
    assert _widths_cached(module, 'n', buf).tolist() == [4, 5] and first.tolist() == [3, 5]
    with torch.inference_mode():
        made = torch.tensor([6, 1])
        assert _widths_cached(module, 'n', made).tolist() == [6, 1]
        made[0] = 2
        assert _widths_cached(module, 'n', made).tolist() == [2, 1]
