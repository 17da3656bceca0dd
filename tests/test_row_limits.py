"""The largest numbers of rows: where 32-bit row numbers would wrap, calls are refused; just below, they work."""

import ctypes

import pytest
import torch

from tabpack_b200 import _lib, ops

FAKE = 1 << 20  # an aligned address that no call gets far enough to use
MOST = (1 << 31) - (1 << 20)


def refused(name, args):
    return getattr(_lib.load(), name)(ctypes.byref(args), None) == -1 and b'2^31 - 2^20' in _lib.load().tp_last_error_string()


@pytest.mark.parametrize('rows,k', [(MOST + 1, 1), ((1 << 31) - 1, 1), (MOST // 2 + 1, 2), (MOST // 32 + 1, 32)])
def test_row_moves_are_refused(rows, k):
    for name in ('tp_dispatch_rows', 'tp_combine_rows', 'tp_combine_rows_backward'):
        assert refused(name, _lib.RowsArgs(rows=rows, k=k, W=1, E=4, dtype=1, position=FAKE, offsets=FAKE, x=FAKE, x_stride=1, out=FAKE,
                                           dout=FAKE, dout_stride=1, dy=FAKE, dweight=FAKE))


@pytest.mark.parametrize('rows', [MOST + 1, (1 << 31) - 257])
def test_ragged_linear_is_refused(rows):
    a = _lib.RaggedLinearArgs(P=2, max_in=8, max_out=8, dtype=1, rows=rows, offsets=FAKE, x=FAKE, x_stride=8, w=FAKE, w_stride=8, y=FAKE,
                              dy=FAKE, dy_stride=8, dx=FAKE, dw=FAKE, dbias=FAKE)
    assert refused('tp_ragged_linear_forward', a) and refused('tp_ragged_linear_backward', a)


@pytest.mark.gpu
def test_row_moves_of_the_most_rows():
    T, dev = MOST, 'cuda'
    position = torch.empty(T, 1, dtype=torch.int32, device=dev)
    torch.arange(T - 1, -1, -1, dtype=torch.int32, device=dev, out=position.view(T))
    offsets = torch.tensor([0, T - 5], dtype=torch.int32, device=dev)  # the first five rows go to no member
    x = torch.empty(T, 1, dtype=torch.bfloat16, device=dev)
    x.view(torch.int16).random_(0, 0x4000)  # (finite numbers)
    out = ops.dispatch_rows(x, position, offsets)
    assert torch.equal(out[:T - 5], x.flip(0)[:T - 5]) and not out[T - 5:].any()
    del out
    y = ops.combine_rows(x, None, position, offsets)
    assert torch.equal(y[5:], x.flip(0)[5:]) and not y[:5].any()
    del y
    dy, dw = ops.combine_rows_backward(x, x, None, position, offsets)
    assert torch.equal(dy[:T - 5], x.flip(0)[:T - 5]) and not dy[T - 5:].any()
    del dy
    for a, e in ((5, 1 << 20), (T - (1 << 20), T)):
        assert torch.equal(dw[a:e], x[a:e].float() * x.flip(0)[a:e].float())
    assert not dw[:5].any()


@pytest.mark.gpu
def test_weight_gradient_of_the_most_rows():
    # the sums over all rows of one member, in parts and pieces; every number is a small power of two, so that they are exact
    R, dev = MOST, 'cuda'
    offsets = torch.tensor([0, R], dtype=torch.int32, device=dev)
    x = torch.zeros(R, 8, dtype=torch.bfloat16, device=dev)
    dy = torch.zeros(R, 8, dtype=torch.bfloat16, device=dev)
    rows = torch.tensor([0, 1, 12345, R // 2, R - 4000, R - 2, R - 1], device=dev)
    x[rows, torch.arange(7, device=dev)] = 2.0
    dy[rows, 7 - torch.arange(7, device=dev)] = 0.25
    w = torch.ones(1, 8, 8, dtype=torch.bfloat16, device=dev)
    _, dw, db = ops.ragged_linear_backward(dy, x, w, None, offsets, need_dx=False)
    want = torch.zeros(1, 8, 8, device=dev)
    want[0, 7 - torch.arange(7), torch.arange(7)] = 0.5
    assert torch.equal(dw, want)
    assert torch.equal(db[0], torch.tensor([0.0] + [0.25] * 7, device=dev))
    del dy, dw
    y = ops.ragged_linear_forward(x, w, None, offsets)
    assert (y[rows] == 2.0).all() and sum(torch.count_nonzero(part).item() for part in y.split(1 << 28)) == 8 * 7
