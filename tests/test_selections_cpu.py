"""What a module keeps from call to call (int32 widths, bf16 weights) belongs to one tensor: a member
selection installs tensors of its own, which may lie where the last selection's lay (no GPU)."""

import copy

import numpy as np
import pytest
import torch

from tabpack_b200 import nn
from tabpack_b200.nn import LayerNormPack, LinearPack, _state, _WeightCache, _widths_cached


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


def test_bf16_copy_of_another_weight_at_the_same_address():
    memory = np.ones((2, 8, 8), np.float32)
    cache, first = _WeightCache(), torch.from_numpy(memory)
    copy = cache.get(first, torch.bfloat16, 8)
    assert (copy == 1).all() and cache.get(first, torch.bfloat16, 8) is copy
    memory[:] = 2
    second = torch.from_numpy(memory)
    assert second.data_ptr() == first.data_ptr() and second._version == first._version
    assert (cache.get(second, torch.bfloat16, 8) == 2).all()
    assert cache.begin_update(first) is None
    second.fill_(3)
    assert (cache.get(second, torch.bfloat16, 8) == 3).all()


def test_bf16_copy_follows_the_widths():
    """A copy made for one set of widths is not taken for another set at the same address."""
    memory, w = np.array([8, 8], np.int32), torch.ones(2, 8, 8)
    cache, a = _WeightCache(), torch.from_numpy(memory)
    copy = cache.get(w, torch.bfloat16, 8, widths=(a, None, None, 0))
    assert cache.get(w, torch.bfloat16, 8, widths=(a, None, None, 0)) is copy
    assert cache.get(w, torch.bfloat16, 8, widths=(torch.from_numpy(memory), None, None, 0)) is not copy


def test_states_of_tensors():
    t = torch.zeros(3)
    assert _state(t) == _state(t) and _state(None) is None and _state(t) != _state(t.view(3))
    before = _state(t)
    t += 1
    assert _state(t) != before
    gone = _state(torch.zeros(3))
    assert gone != gone[:0] + _state(torch.zeros(3)) and not gone[0] == gone[0]


@pytest.mark.parametrize('k', [3, 300])
def test_bf16_copies_of_selections_in_a_row(k):
    linear = LinearPack(8, 8, pack_size=3000).eval()
    with torch.no_grad():
        linear.weight.copy_(torch.arange(3000.0)[:, None, None].bfloat16().expand(3000, 8, 8))
        for i in range(20):
            idx = torch.arange(k) * 7 + 31 * i
            with linear.temporarily_select(pack_idx=idx):
                copy = linear._cache.get(linear.weight, torch.bfloat16, 8)
                assert torch.equal(copy.float(), linear.weight)


def test_layer_norm_widths_are_kept_as_the_kernels_read_them():
    """int32, through construction, replacement and a checkpoint written with other integers."""
    pack = LayerNormPack([3, 5], pack_size=2)
    state = {**pack.state_dict(), 'n_features': torch.tensor([4, 2])}
    pack.load_state_dict(state)
    assert pack.n_features.dtype == torch.int32 and pack.n_features.tolist() == [4, 2]
    pack.replace(pack_idx=torch.tensor([1]), n_features=[5])
    pack.load_state_dict_at(state, pack_idx=torch.tensor([0]), state_dict_idx=torch.tensor([1]))
    assert pack.n_features.dtype == torch.int32 and pack.n_features.tolist() == [2, 5]


def test_copies_recorded_into_a_graph_are_not_kept(monkeypatch):
    """While a graph is captured nothing is computed: what it will write on a replay is no one else's copy, and a
    copy that was there before is taken as it is."""
    monkeypatch.setattr(nn, '_capturing', lambda t: True)
    module, buf = torch.nn.Module(), torch.tensor([3, 5])
    cache, w = _WeightCache(), torch.ones(2, 8, 8)
    backbone = nn.MLPBackbonePack(d_in=4, n_blocks=[1, 2], d_block=[8, 8], dropout=0.0, pack_size=2)
    widths, copy, depths = _widths_cached(module, 'n', buf), cache.get(w, torch.bfloat16, 8), backbone._n_blocks_i32(None)
    assert widths.tolist() == [3, 5] and (copy == 1).all() and depths.tolist() == [1, 2]
    assert cache.key is None and cache.value is None and backbone._nb_cache is None
    monkeypatch.undo()
    kept = _widths_cached(module, 'n', buf), cache.get(w, torch.bfloat16, 8), backbone._n_blocks_i32(None)
    assert kept[0] is not widths and kept[1] is not copy and kept[2] is not depths
    monkeypatch.setattr(nn, '_capturing', lambda t: True)
    assert _widths_cached(module, 'n', buf) is kept[0] and cache.get(w, torch.bfloat16, 8) is kept[1]
    assert backbone._n_blocks_i32(None) is kept[2]


def test_modules_in_use_are_copied_and_saved(tmp_path):
    """A whole module after a call: its copies are made anew where it arrives."""
    linear = LinearPack(8, [4, 8], pack_size=2)
    use = lambda m: m._cache.get(m.weight, torch.bfloat16, 8, widths=(  # noqa: E731
        _widths_cached(m, 'out', m.out_features), None, None, 0))
    first = use(linear)
    torch.save(linear, tmp_path / 'linear.pt')
    for other in (copy.deepcopy(linear), torch.load(tmp_path / 'linear.pt', weights_only=False)):
        with torch.no_grad():
            other.weight.fill_(2)
        assert (use(other) == 2).all() and use(other) is use(other)
    assert use(linear) is first
