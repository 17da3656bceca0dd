"""Host-side rules of routing, ragged linear layers and 4-bit rows: refusals without a GPU, and the stored forms' sizes."""

import ctypes

import pytest
import torch

from oracle import routed
from tabpack_b200 import _lib, ops
from tabpack_b200.nn import Fp4LinearPack, LinearPack, RoutedMLPPack

FAKE = 1 << 20  # an aligned address that no call gets far enough to use


def code(name, args):
    return getattr(_lib.load(), name)(ctypes.byref(args), None)


def ragged(**kw):
    base = dict(P=2, max_in=16, max_out=8, dtype=1, rows=10, offsets=FAKE, x=FAKE, x_stride=16, w=FAKE, w_stride=16, y=FAKE)
    return _lib.RaggedLinearArgs(**{**base, **kw})


@pytest.mark.parametrize('bad,want', [
    (dict(P=0), -1), (dict(P=65536), -1), (dict(max_in=0), -1), (dict(max_out=-1), -1), (dict(rows=0), -1), (dict(rows=1 << 31), -1),
    (dict(dtype=2), -1), (dict(offsets=None), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(y=None), -1),
    (dict(x_stride=15), -1), (dict(w_stride=8), -1), (dict(offsets=FAKE + 2), -2), (dict(x=FAKE + 2), -2), (dict(x_stride=20), -2),
    (dict(w=FAKE + 8), -2), (dict(bias=FAKE + 1), -2), (dict(dtype=0), -1)])
def test_ragged_forward_arguments(bad, want):
    # (fp32 without a workspace is the last)
    assert code('tp_ragged_linear_forward', ragged(**bad)) == want
    assert _lib.load().tp_last_error_string()


@pytest.mark.parametrize('bad,want', [
    (dict(dy=None), -1), (dict(relu=1, y=None), -1), (dict(dy_stride=7), -1), (dict(relu=1), -1), (dict(dy=FAKE + 1), -2)])
def test_ragged_backward_arguments(bad, want):
    args = dict(dy=FAKE, dy_stride=8, dx=FAKE, dw=FAKE, dbias=FAKE)
    assert code('tp_ragged_linear_backward', ragged(**{**args, **bad})) == want


def route(**kw):
    base = dict(rows=10, E=4, top_k=2, dtype=0, logits=FAKE, logits_stride=4, weight=FAKE, expert=FAKE, position=FAKE, offsets=FAKE,
                importance=FAKE, dlogits=FAKE)
    return _lib.RouteArgs(**{**base, **kw})


@pytest.mark.parametrize('bad,want', [
    (dict(rows=0), -1), (dict(E=0), -1), (dict(E=1025, top_k=1), -1), (dict(top_k=0), -1), (dict(top_k=5), -1), (dict(rows=1 << 30), -1),
    (dict(E=64, top_k=33, logits_stride=64), -1), (dict(dtype=3), -1), (dict(logits=None), -1), (dict(logits_stride=3), -1), (dict(expert=None), -1),
    (dict(logits=FAKE + 2), -2), (dict(weight=FAKE + 2), -2)])
def test_route_arguments(bad, want):
    assert code('tp_route_forward', route(**bad)) == want
    assert code('tp_route_backward', route(**bad)) == want


@pytest.mark.parametrize('rows,top_k', [((1 << 31) - (1 << 20) + 1, 1), ((1 << 30) - (1 << 19) + 1, 2), (1 << 62, 4)])
def test_route_refuses_more_pairs_than_it_counts(rows, top_k):
    assert code('tp_route_forward', route(rows=rows, top_k=top_k)) == -1
    assert code('tp_route_backward', route(rows=rows, top_k=top_k)) == -1


def test_route_outputs_and_workspace():
    for name in ('position', 'offsets', 'importance'):
        assert code('tp_route_forward', route(**{name: None})) == -1
    assert code('tp_route_backward', route(dlogits=None)) == -1
    size = _lib.load().tp_route_workspace_size
    assert size(100, 4, 2) == 0 and size(100000, 4, 2) > 0
    assert code('tp_route_forward', route(rows=100000)) == -1
    assert code('tp_route_forward', route(rows=100000, workspace=FAKE, workspace_bytes=size(100000, 4, 2) - 1)) == -1


def moves(**kw):
    base = dict(rows=10, k=2, W=8, E=4, dtype=0, position=FAKE, offsets=FAKE, x=FAKE, x_stride=8, out=FAKE, dout=FAKE, dout_stride=8,
                dy=FAKE, dweight=FAKE)
    return _lib.RowsArgs(**{**base, **kw})


@pytest.mark.parametrize('bad,want', [
    (dict(rows=0), -1), (dict(k=0), -1), (dict(k=33), -1), (dict(W=0), -1), (dict(E=0), -1), (dict(rows=1 << 30), -1), (dict(dtype=2), -1),
    (dict(position=None), -1), (dict(offsets=None), -1), (dict(x=FAKE + 2), -2), (dict(position=FAKE + 1), -2)])
def test_row_move_arguments(bad, want):
    for name in ('tp_dispatch_rows', 'tp_combine_rows', 'tp_combine_rows_backward'):
        assert code(name, moves(**bad)) == want
    assert code('tp_dispatch_rows', moves(x=None)) == code('tp_combine_rows', moves(out=None)) == -1
    assert code('tp_combine_rows_backward', moves(dout=None)) == -1
    assert code('tp_combine_rows_backward', moves(dy=None, dweight=None)) == 0


def fp4(**kw):
    base = dict(P=2, K=40, format=0, dtype=0, rows=10, x=FAKE, x_stride=40, codes=FAKE, scales=FAKE, row_scale=FAKE, values=FAKE)
    return _lib.Fp4Args(**{**base, **kw})


@pytest.mark.parametrize('bad,want', [
    (dict(P=0), -1), (dict(P=3), -1), (dict(K=0), -1), (dict(format=2), -1), (dict(rows=0), -1), (dict(codes=None), -1),
    (dict(row_scale=None), -1), (dict(codes=FAKE + 8), -2), (dict(scales=FAKE + 4), -2), (dict(offsets=FAKE + 2), -2)])
def test_fp4_arguments(bad, want):
    assert code('tp_fp4_quantize', fp4(**bad)) == code('tp_fp4_values', fp4(**bad)) == want
    assert code('tp_fp4_quantize', fp4(x=None)) == code('tp_fp4_quantize', fp4(dtype=2)) == -1
    assert code('tp_fp4_quantize', fp4(x_stride=39)) == code('tp_fp4_values', fp4(values=None)) == -1
    assert code('tp_fp4_quantize', fp4(x=FAKE + 2)) == -2


def fp4_linear(**kw):
    base = dict(P=2, K=40, N=8, format=0, dtype=0, rows=10, x_codes=FAKE, x_scales=FAKE, x_row_scale=FAKE, w_codes=FAKE, w_scales=FAKE,
                w_row_scale=FAKE, y=FAKE)
    return _lib.Fp4LinearArgs(**{**base, **kw})


@pytest.mark.parametrize('bad,want', [
    (dict(P=0), -1), (dict(P=3), -1), (dict(N=0), -1), (dict(format=-1), -1), (dict(dtype=2), -1), (dict(x_codes=None), -1),
    (dict(w_scales=None), -1), (dict(y=None), -1), (dict(x_shared=1, offsets=FAKE), -1), (dict(w_codes=FAKE + 8), -2),
    (dict(bias=FAKE + 2), -2), (dict(x=FAKE, x_stride=40), -1), (dict(x=FAKE, x_stride=40, workspace=FAKE, workspace_bytes=10), -1)])
def test_fp4_linear_arguments(bad, want):
    assert code('tp_fp4_linear_forward', fp4_linear(**bad)) == want
    assert _lib.load().tp_fp4_linear_forward(None, None) == -1


@pytest.mark.parametrize('bad,want', [
    (dict(x=None), -1), (dict(out=None), -1), (dict(rows=0), -1), (dict(rows=1 << 31), -1), (dict(cols=0), -1), (dict(stride=4), -1),
    (dict(wide=4), -1), (dict(wide=12), -1), (dict(x=FAKE + 1), -2), (dict(out=FAKE + 8), -2)])
def test_align_rows_arguments(bad, want):
    a = {**dict(x=FAKE, stride=5, rows=3, cols=5, out=FAKE, wide=8), **bad}
    assert _lib.load().tp_align_rows(a['x'], a['stride'], a['rows'], a['cols'], a['out'], a['wide'], None) == want


def test_sizes_of_the_stored_form():
    lib = _lib.load()
    for K in (1, 16, 31, 32, 33, 255, 256, 257, 8192):
        assert lib.tp_fp4_pitch(K) == ops._fp4_pitch(K) == -(-K // 32) * 16
        for name, c in _lib.TP_FP4.items():
            blocks = -(-K // routed.FP4_BLOCK[name])
            tiles = lib.tp_fp4_scale_tiles(K, c)
            assert tiles == ops._fp4_scale_tiles(K, c) and 4 * tiles >= blocks
    # ragged groups begin in scale tiles of their own: as many as each needs, in order
    for edges in ([0, 0, 5, 128, 257, 257, 1000], [3, 130, 131, 132, 300], [127, 255, 384]):
        for g, (a, b) in enumerate(zip(edges, edges[1:])):
            assert b // 128 + g + 1 - (a // 128 + g) >= -(-(b - a) // 128)
        last = len(edges) - 2
        assert edges[last] // 128 + last + -(-(edges[-1] - edges[last]) // 128) <= edges[-1] // 128 + len(edges) - 1


def test_reference_rounding_on_known_numbers():
    x = torch.tensor([[6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -5.1, 0.26, 0.0, 0.24, 4.9, 1.3, -0.8, 2.4]])
    want = [6.0, 4.0, 4.0, 2.0, 2.0, 1.0, 1.0, 0.0, -6.0, 0.5, 0.0, 0.0, 4.0, 1.5, -1.0, 2.0]
    for format in routed.FP4_BLOCK:
        assert routed.fp4_round(x, format)[0][0].tolist() == want


def test_cpu_tensors_are_refused():
    x, o = torch.zeros(4, 16), torch.tensor([0, 2, 4], dtype=torch.int32)
    w = torch.zeros(2, 8, 16)
    plan = torch.zeros(4, 1, dtype=torch.int32), o
    q = ops.Fp4Rows(torch.zeros(2, 8, 16, dtype=torch.uint8), torch.zeros(2, 1, 4, 512, dtype=torch.uint8), torch.zeros(2, 8), 16, 'nvfp4')
    for call in (lambda: ops.route_forward(x, 2), lambda: ops.dispatch_rows(x, *plan), lambda: ops.combine_rows(x, None, *plan),
                 lambda: ops.combine_rows_backward(x, x, None, *plan), lambda: ops.ragged_linear_forward(x, w, None, o),
                 lambda: ops.ragged_linear_backward(torch.zeros(4, 8), x, w, None, o), lambda: ops.fp4_quantize(x),
                 lambda: ops.fp4_values(q), lambda: ops.fp4_linear_forward(x, q), lambda: LinearPack(16, 8, pack_size=2).forward_rows(x, o),
                 lambda: RoutedMLPPack(16, 8, 4, top_k=1, pack_size=2)(x),
                 lambda: Fp4LinearPack.from_linear(LinearPack(16, 8, pack_size=2))):
        with pytest.raises(RuntimeError):
            call()
