"""Member selections in a row, captures and streams: a module's int32 widths and bf16 weights are those
of the tensors that it holds at the call."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')


def norm_pack(P=12, W=40):
    from tabpack_b200.nn import LayerNormPack

    pack = LayerNormPack([1 + (11 * i + 6) % W for i in range(P)], max_n_features=W, pack_size=P).cuda().eval()
    gen = torch.Generator(device='cuda').manual_seed(0)
    with torch.no_grad():
        pack.weight.copy_(torch.rand(P, W, generator=gen, device='cuda'))
        pack.bias.copy_(torch.rand(P, W, generator=gen, device='cuda'))
    return pack, torch.randn(P, 7, W, generator=gen, device='cuda')


SELECTIONS = [[0, 4, 7], [1, 2, 3], [11, 10, 9], [5, 0, 6], [2, 2, 8]]


def test_layer_norm_selections_in_a_row():
    """Equally many members each time, no call on the whole pack between."""
    pack, x = norm_pack()
    with torch.no_grad():
        picks = [torch.tensor(s, device='cuda') for s in SELECTIONS]
        want = [pack(x[i], i) for i in picks]
        for i, t in zip(picks, want):
            with pack.temporarily_select(pack_idx=i):
                assert torch.equal(pack(x[i]), t)


@pytest.mark.parametrize('ragged', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_linear_selections_in_a_row(ragged, dtype):
    from tabpack_b200.nn import LinearPack

    P = 12
    torch.manual_seed(1)
    linear = LinearPack(24, [8 + (5 * i) % 33 for i in range(P)] if ragged else 40, max_out_features=40,
                        pack_size=P).cuda().eval()
    x = torch.randn(P, 9, 24, device='cuda').to(dtype)
    with torch.no_grad():
        picks = [torch.tensor(s, device='cuda') for s in SELECTIONS]
        want = [linear(x[i], i) for i in picks]
        for i, t in zip(picks, want):
            with linear.temporarily_select(pack_idx=i):
                assert torch.equal(linear(x[i]), t)


def test_one_hot_weights_of_another_tensor_at_the_same_address():
    from tabpack_b200.nn import _OneHotWeightCache

    memory = torch.empty(2, 16, 12, device='cuda')
    view = lambda: torch.empty(0, device='cuda').set_(memory.untyped_storage(), 0, memory.shape)  # noqa: E731
    cache, got = _OneHotWeightCache(), []
    for value in (1.0, 2.0):
        memory.fill_(value)
        w = view()
        got.append([t.clone() for t in cache.get(w, None, 4, 16, 8)])
        assert cache.get(w, None, 4, 16, 8)[0] is cache.dense
        del w
    for a, b in zip(*got):
        assert torch.equal(2 * a, b)


def test_layer_norm_captured_first():
    """A graph may hold a pack's first call, and its replays follow the members' widths."""
    pack, x = norm_pack()
    every = torch.arange(12, device='cuda')
    with torch.no_grad():
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pack(x)
        assert torch.equal(pack(x), pack(x, every))
        graph.replay()
        assert torch.equal(y, pack(x))
        pack.replace(pack_idx=torch.tensor([3, 5], device='cuda'), n_features=[40, 2])
        graph.replay()
        assert torch.equal(y, pack(x, every)) and torch.equal(y, pack(x))


def test_linear_captured_first():
    """A layer's first call recorded into a graph: a call outside makes its own copies of widths and weights."""
    from tabpack_b200.nn import LinearPack

    torch.manual_seed(2)
    linear = LinearPack(24, [8 + (5 * i) % 33 for i in range(12)], max_out_features=40, pack_size=12).cuda().eval()
    x = torch.randn(12, 9, 24, device='cuda').bfloat16()
    every = torch.arange(12, device='cuda')
    with torch.no_grad():
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = linear(x)
        assert torch.equal(linear(x), linear(x, every))
        graph.replay()
        assert torch.equal(y, linear(x))
        linear.weight.mul_(2)
        graph.replay()
        assert torch.equal(y, linear(x))
