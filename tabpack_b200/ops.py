"""Torch-facing wrappers of the C ABI.

These functions only validate tensors, allocate outputs with PyTorch's caching
allocator and pass raw pointers plus the current CUDA stream to the library.
All arithmetic happens in the CUDA kernels; CPU tensors are rejected.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from tabpack_b200 import _lib
from tabpack_b200._lib import TP_DTYPE_BF16, TP_DTYPE_F32, check, load


class KernelTimes:
    """Per-family device time of this library's kernel launches (`tp_profile_start` /
    `tp_profile_stop`): `with KernelTimes() as kt: ...` then `kt.ms` and `kt.launches`, dicts
    keyed by family name (`_lib.TP_PROF_KINDS`).  Each launch is bracketed by two CUDA events
    on its stream; the totals are read once the block ends (a synchronisation)."""

    def __init__(self, capacity: int = 1 << 16) -> None:
        self.capacity = capacity
        self.ms: dict[str, float] = {}
        self.launches: dict[str, int] = {}
        self.dropped = 0

    def __enter__(self) -> 'KernelTimes':
        check(load().tp_profile_start(self.capacity), 'tp_profile_start')
        return self

    def __exit__(self, *exc) -> None:
        n = len(_lib.TP_PROF_KINDS)
        ms = (ctypes.c_double * n)()
        cnt = (ctypes.c_int64 * n)()
        dropped = ctypes.c_int32(0)
        check(load().tp_profile_stop(ms, cnt, n, ctypes.byref(dropped)), 'tp_profile_stop')
        self.ms = {k: ms[i] for i, k in enumerate(_lib.TP_PROF_KINDS)}
        self.launches = {k: cnt[i] for i, k in enumerate(_lib.TP_PROF_KINDS)}
        self.dropped = dropped.value


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _dtype_code(dt: torch.dtype) -> int:
    if dt == torch.bfloat16:
        return TP_DTYPE_BF16
    if dt == torch.float32:
        return TP_DTYPE_F32
    raise TypeError(f'unsupported activation dtype {dt} (bf16 or fp32)')


def _cuda(name: str, t: Tensor | None, dtype: torch.dtype | None = None) -> Tensor | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError(f'{name} must be a CUDA tensor (tabpack_b200 has no CPU path)')
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f'{name} must have dtype {dtype}, got {t.dtype}')
    return t.contiguous()


def _i32(name: str, t: Tensor | None) -> Tensor | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError(f'{name} must be a CUDA tensor')
    return t.to(torch.int32).contiguous()


def _linear_args(x, weight, bias, in_features, out_features, n_blocks, block_index, relu,
                 dropout_p, seed, offset, member_base, y, row_index=None) -> _lib.LinearArgs:
    P, max_out, max_in = weight.shape
    shared = x.ndim == 2 and row_index is None
    B = row_index.shape[1] if row_index is not None else x.shape[0] if shared else x.shape[1]
    a = _lib.LinearArgs()
    a.P, a.B, a.max_in, a.max_out = P, B, max_in, max_out
    a.dtype = _dtype_code(x.dtype)
    a.x_shared = 1 if shared else 0
    if row_index is not None:
        a.row_index, a.x_rows = row_index.data_ptr(), x.shape[0]
    a.in_features = _ptr(in_features)
    a.out_features = _ptr(out_features)
    a.n_blocks = _ptr(n_blocks)
    a.block_index = int(block_index)
    a.relu = 1 if relu else 0
    a.dropout_p = _ptr(dropout_p)
    a.seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    a.offset = int(offset) & 0xFFFFFFFF
    a.member_base = int(member_base) & 0xFFFFFFFF
    a.x = _ptr(x)
    a.w = _ptr(weight)
    a.bias = _ptr(bias)
    a.y = _ptr(y)
    return a


def _row_index(row_index: Tensor | None, P: int) -> Tensor | None:
    """(P, B) int32 CUDA row indices of a gathered input, or None."""
    if row_index is None:
        return None
    if row_index.ndim != 2 or row_index.shape[0] != P:
        raise ValueError(f'row_index must be (pack_size={P}, batch), got {tuple(row_index.shape)}')
    if not row_index.is_cuda:
        raise RuntimeError('row_index must be a CUDA tensor (tabpack_b200 has no CPU path)')
    return row_index.to(torch.int32).contiguous()


def linear_forward(
    x: Tensor,
    weight: Tensor,
    bias: Tensor | None,
    *,
    in_features: Tensor | None = None,
    out_features: Tensor | None = None,
    n_blocks: Tensor | None = None,
    block_index: int = 0,
    relu: bool = False,
    dropout_p: Tensor | None = None,
    seed: int = 0,
    offset: int = 0,
    member_base: int = 0,
    row_index: Tensor | None = None,
    y: Tensor | None = None,
) -> Tensor:
    """Packed linear (+ReLU +dropout +depth gating) forward; see `tp_linear_forward`.  With
    `row_index` (P, B), x is a (rows, in) table and member m's input row b is
    x[row_index[m, b]] (gathered by the GEMM's operand loads).  `y`: an output buffer whose
    padding columns already hold zeros (`y_pad_zero`: only the members' column tiles are
    written); by default a new one."""
    weight = _cuda('weight', weight)
    x = _cuda('x', x, weight.dtype)
    row_index = _row_index(row_index, weight.shape[0])
    bias = _cuda('bias', bias, torch.float32)
    dropout_p = _cuda('dropout_p', dropout_p, torch.float32)
    in_features, out_features, n_blocks = (_i32(n, t) for n, t in (
        ('in_features', in_features), ('out_features', out_features), ('n_blocks', n_blocks)))
    P, max_out, _ = weight.shape
    B = x.shape[-2] if row_index is None else row_index.shape[1]
    pad_zero = y is not None
    if y is None:
        y = torch.empty((P, B, max_out), dtype=x.dtype, device=x.device)
    elif tuple(y.shape) != (P, B, max_out) or y.dtype != x.dtype or not y.is_contiguous() or y.device != x.device:
        raise ValueError(f'y must be a contiguous ({P}, {B}, {max_out}) {x.dtype} tensor on {x.device}')
    a = _linear_args(x, weight, bias, in_features, out_features, n_blocks, block_index, relu,
                     dropout_p, seed, offset, member_base, y, row_index)
    a.y_pad_zero = 1 if pad_zero else 0
    check(load().tp_linear_forward(ctypes.byref(a), _stream()), 'tp_linear_forward')
    if pad_zero:
        increment_version([y])
    return y


def linear_backward(
    dy: Tensor,
    x: Tensor,
    weight: Tensor,
    y: Tensor | None,
    *,
    in_features: Tensor | None = None,
    out_features: Tensor | None = None,
    n_blocks: Tensor | None = None,
    block_index: int = 0,
    relu: bool = False,
    dropout_p: Tensor | None = None,
    seed: int = 0,
    offset: int = 0,
    member_base: int = 0,
    need_dx: bool = True,
    need_dw: bool = True,
    need_db: bool = True,
    dw_shape: tuple[int, int] | None = None,
    db_cols: int | None = None,
    dx_cols: int = 0,
    row_index: Tensor | None = None,
    dw_out: Tensor | None = None,
    dw_pad_zero: bool = False,
    dx_out: Tensor | None = None,
) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """Backward of `linear_forward`: returns (dx, dw, db); dw/db are fp32.  With dx_cols > 0
    only dx's first dx_cols columns are computed (the rest are zeros).  With `row_index`, x is
    the forward's table (no dx).  `dw_out`: the weight gradient's buffer (else a new one);
    `dw_pad_zero`: it already holds zeros outside the active members' blocks (`tp_linear_grad_args`).
    `dx_out`: the input gradient's buffer, whose columns beyond each member's input column tiles
    already hold zeros (`dx_pad_zero`); by default a new one."""
    weight = _cuda('weight', weight)
    x = _cuda('x', x, weight.dtype)
    row_index = _row_index(row_index, weight.shape[0])
    if row_index is not None and need_dx:
        raise ValueError('a gathered input (a table) takes no input gradient')
    dy = _cuda('dy', dy, weight.dtype)
    y = _cuda('y', y, weight.dtype)
    dropout_p = _cuda('dropout_p', dropout_p, torch.float32)
    in_features, out_features, n_blocks = (_i32(n, t) for n, t in (
        ('in_features', in_features), ('out_features', out_features), ('n_blocks', n_blocks)))
    P, max_out, max_in = weight.shape
    B = x.shape[-2] if row_index is None else row_index.shape[1]
    need_g = relu or dropout_p is not None or out_features is not None or n_blocks is not None
    g = torch.empty_like(dy) if need_g else None
    dx = None
    if need_dx:
        if dx_out is not None:
            if (tuple(dx_out.shape) != (P, B, max_in) or dx_out.dtype != dy.dtype or not dx_out.is_contiguous()
                    or dx_out.device != dy.device):
                raise ValueError(f'dx_out must be a contiguous ({P}, {B}, {max_in}) {dy.dtype} tensor on {dy.device}')
            dx = dx_out
        else:
            dx = torch.empty((P, B, max_in), dtype=dy.dtype, device=dy.device)
    rows, cols = dw_shape if dw_shape is not None else (max_out, max_in)
    dw = None
    if need_dw:
        if dw_out is not None:
            if (tuple(dw_out.shape) != (P, rows, cols) or dw_out.dtype != torch.float32 or not dw_out.is_contiguous()
                    or dw_out.device != dy.device):
                raise ValueError('dw_out must be a contiguous fp32 (P, rows, cols) tensor on the gradient device')
            dw = dw_out
        else:
            dw = torch.empty((P, rows, cols), dtype=torch.float32, device=dy.device)
    dbc = db_cols if db_cols is not None else max_out
    db = torch.empty((P, dbc), dtype=torch.float32, device=dy.device) if need_db else None
    ga = _lib.LinearGradArgs()
    ga.fwd = _linear_args(x, weight, None, in_features, out_features, n_blocks, block_index, relu,
                          dropout_p, seed, offset, member_base, None, row_index)
    ga.dy, ga.y, ga.g = _ptr(dy), _ptr(y), _ptr(g)
    ga.dbias, ga.dx, ga.dw = _ptr(db), _ptr(dx), _ptr(dw)
    ga.dw_rows, ga.dw_cols, ga.db_cols = rows, cols, dbc
    ga.dx_cols = int(dx_cols)
    ga.dw_pad_zero = 1 if (dw_pad_zero and dw_out is not None) else 0
    ga.dx_pad_zero = 1 if (dx is not None and dx_out is not None) else 0
    check(load().tp_linear_backward(ctypes.byref(ga), _stream()), 'tp_linear_backward')
    if ga.dx_pad_zero:
        increment_version([dx])
    return dx, dw, db


def dropout_mask(*, seed: int, offset: int, member_base: int, p: Tensor, rows: int, cols: int) -> Tensor:
    """(P, rows, cols) uint8 Philox keep mask used by the fused dropout."""
    p = _cuda('p', p, torch.float32)
    P = p.shape[0]
    mask = torch.empty((P, rows, cols), dtype=torch.uint8, device=p.device)
    check(load().tp_dropout_mask(int(seed) & 0xFFFFFFFFFFFFFFFF, int(offset) & 0xFFFFFFFF,
                                 int(member_base) & 0xFFFFFFFF, p.data_ptr(), P, rows, cols,
                                 mask.data_ptr(), _stream()), 'tp_dropout_mask')
    return mask


def _hparam(v) -> _lib.HParam:
    h = _lib.HParam()
    if isinstance(v, Tensor):
        if not v.is_cuda or v.dtype != torch.float32 or v.ndim != 1:
            raise TypeError('per-member hyperparameters must be 1-D fp32 CUDA tensors')
        h.per_member = v.data_ptr()
        h.scalar = 0.0
    else:
        h.per_member = None
        h.scalar = float(v)
    return h


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, steps=None, step: int = 0,
               lr, beta1, beta2, eps, weight_decay) -> None:
    """Grouped AdamW over parameter packs (each (P, ...) fp32, contiguous).

    `steps` (per-tensor (P,) int64 tensors, already incremented) or the scalar
    `step` give the bias-correction step.  Hyperparameters are floats or (P,)
    fp32 CUDA tensors.  Tensors are chunked into launches of at most 32.
    """
    hp = [lr, beta1, beta2, eps, weight_decay]
    hp = [v.contiguous() if isinstance(v, Tensor) else v for v in hp]
    n = len(params)
    for s in range(0, n, _lib.TP_MAX_OPT_TENSORS):
        a = _lib.AdamWArgs()
        chunk = range(s, min(n, s + _lib.TP_MAX_OPT_TENSORS))
        a.n_tensors = len(chunk)
        for j, i in enumerate(chunk):
            p = params[i]
            for name, t in (('param', p), ('grad', grads[i]), ('exp_avg', exp_avgs[i]),
                            ('exp_avg_sq', exp_avg_sqs[i])):
                if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
                    raise TypeError(f'{name} must be a contiguous fp32 CUDA tensor')
            ot = a.t[j]
            ot.p, ot.grad = p.data_ptr(), grads[i].data_ptr()
            ot.exp_avg, ot.exp_avg_sq = exp_avgs[i].data_ptr(), exp_avg_sqs[i].data_ptr()
            ot.step = None if steps is None else steps[i].data_ptr()
            ot.numel = p.numel()
            ot.inner = max(1, p.numel() // p.shape[0])
        a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = (_hparam(v) for v in hp)
        a.step = int(step)
        check(load().tp_adamw_step(ctypes.byref(a), _stream()), 'tp_adamw_step')
    # the kernel updated these in place: bump their version counters as torch's in-place ops do
    # (caches keyed on a parameter's version, e.g. its bf16 copy, see the new values)
    increment_version(list(params) + list(exp_avgs) + list(exp_avg_sqs))


def muon_workspace_size(P: int, max_out: int, max_in: int) -> int:
    """Bytes of scratch one `muon_step` call on a (P, max_out, max_in) pack needs."""
    return int(load().tp_muon_workspace_size(P, max_out, max_in))


def _muon_args(p: Tensor, grad: Tensor, momentum_buffer: Tensor, *, out_features=None, in_features=None, lr,
               momentum, weight_decay, update_scale=None, nesterov: bool = True, mutate_grad: bool = True,
               ns_steps: int = 5, p_bf16: Tensor | None = None, n_blocks: Tensor | None = None,
               block_index: int = 0, gated_momentum_zero: bool = False):
    """`tp_muon_args` of one group (workspace unset), the tensors that must stay alive until
    the launch is queued, and the tensors the step writes."""
    for name, t in (('p', p), ('grad', grad), ('momentum_buffer', momentum_buffer)):
        if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous() or t.ndim != 3:
            raise TypeError(f'{name} must be a contiguous 3-D fp32 CUDA tensor')
    P, mo, mi = p.shape
    a = _lib.MuonArgs()
    a.P, a.max_out, a.max_in = P, mo, mi
    a.p, a.grad, a.momentum_buffer = p.data_ptr(), grad.data_ptr(), momentum_buffer.data_ptr()
    of, inf = _i32('out_features', out_features), _i32('in_features', in_features)
    a.out_features, a.in_features = _ptr(of), _ptr(inf)
    a.lr, a.momentum, a.weight_decay = _hparam(lr), _hparam(momentum), _hparam(weight_decay)
    us = _cuda('update_scale', update_scale, torch.float32)
    a.update_scale = _ptr(us)
    a.nesterov, a.mutate_grad, a.ns_steps = int(nesterov), int(mutate_grad), int(ns_steps)
    if p_bf16 is not None:
        if (not p_bf16.is_cuda or p_bf16.dtype != torch.bfloat16 or not p_bf16.is_contiguous() or p_bf16.ndim != 3
                or p_bf16.shape[0] != P):
            raise TypeError('p_bf16 must be a contiguous (P, rows, cols) bf16 CUDA tensor')
        a.p_bf16, a.p_bf16_rows, a.p_bf16_cols = p_bf16.data_ptr(), p_bf16.shape[1], p_bf16.shape[2]
    nb = _i32('n_blocks', n_blocks)
    if nb is not None:
        if nb.shape != (P,):
            raise ValueError(f'n_blocks must be ({P},), got {tuple(nb.shape)}')
        a.n_blocks, a.block_index = nb.data_ptr(), int(block_index)
        a.gated_momentum_zero = 1 if gated_momentum_zero else 0
    keep = (of, inf, us, nb, lr, momentum, weight_decay)
    written = [p, momentum_buffer] + ([grad] if mutate_grad else []) + ([p_bf16] if p_bf16 is not None else [])
    return a, keep, written


def muon_step(p: Tensor, grad: Tensor, momentum_buffer: Tensor, *, out_features=None, in_features=None, lr,
              momentum, weight_decay, update_scale=None, nesterov: bool = True, mutate_grad: bool = True,
              ns_steps: int = 5, workspace: Tensor | None = None, p_bf16: Tensor | None = None,
              n_blocks: Tensor | None = None, block_index: int = 0, gated_momentum_zero: bool = False) -> None:
    """One Muon group step on a packed (P, max_out, max_in) fp32 weight; see `tp_muon_step`.
    `p_bf16` (P, rows >= max_out, cols >= max_in) bf16, optional, receives bf16 of the updated
    weights of each member's out x in block in the same pass.  `n_blocks` / `block_index`: the
    weight's block is depth-gated for members with n_blocks <= block_index (their gradient is
    exactly zero and is not read); `gated_momentum_zero`: their momentum is zero as well (not
    read either)."""
    a, keep, written = _muon_args(p, grad, momentum_buffer, out_features=out_features, in_features=in_features,
                                  lr=lr, momentum=momentum, weight_decay=weight_decay, update_scale=update_scale,
                                  nesterov=nesterov, mutate_grad=mutate_grad, ns_steps=ns_steps, p_bf16=p_bf16,
                                  n_blocks=n_blocks, block_index=block_index,
                                  gated_momentum_zero=gated_momentum_zero)
    P, mo, mi = p.shape
    need = muon_workspace_size(P, mo, mi)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=p.device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    check(load().tp_muon_step(ctypes.byref(a), _stream()), 'tp_muon_step')
    del keep
    increment_version(written)


def muon_grouped_workspace_size(shapes: list[tuple[int, int, int]]) -> int:
    """Bytes of the workspace of a grouped Muon call over weights of these (P, max_out, max_in)."""
    arr = (_lib.MuonArgs * len(shapes))()
    for a, (P, mo, mi) in zip(arr, shapes):
        a.P, a.max_out, a.max_in = P, mo, mi
    return int(load().tp_muon_grouped_workspace_size(arr, len(shapes)))


def muon_step_grouped(steps: list[dict], *, workspace: Tensor | None = None) -> None:
    """Several Muon groups of one device in one call (`tp_muon_step_grouped`): each entry of
    `steps` holds `muon_step`'s arguments for one group (`p`, `grad`, `momentum_buffer`, ...,
    without `workspace`).  Each group's result equals its own `muon_step` bit for bit; the
    Newton-Schulz GEMMs of all groups share launches."""
    if not steps:
        return
    built = [_muon_args(**kw) for kw in steps]
    arr = (_lib.MuonArgs * len(built))(*[b[0] for b in built])
    need = muon_grouped_workspace_size([tuple(kw['p'].shape) for kw in steps])
    dev = steps[0]['p'].device
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    check(load().tp_muon_step_grouped(arr, len(built), workspace.data_ptr(),
                                      workspace.numel() * workspace.element_size(), _stream()),
          'tp_muon_step_grouped')
    del built
    increment_version([t for kw in steps for t in _muon_written(kw)])


def _muon_written(kw: dict) -> list:
    out = [kw['p'], kw['momentum_buffer']]
    if kw.get('mutate_grad', True):
        out.append(kw['grad'])
    if kw.get('p_bf16') is not None:
        out.append(kw['p_bf16'])
    return out


def metric_pack(metric: str, y_pred: Tensor, y_true: Tensor, classes: int = 1) -> Tensor:
    """(P,) metric values; y_pred (P, N[, classes]); see `tp_metric_pack`."""
    code = _lib.TP_METRIC[metric]
    y_pred = _cuda('y_pred', y_pred)
    y_true = _cuda('y_true', y_true)
    if code == _lib.TP_METRIC['accuracy']:
        y_pred, y_true = y_pred.to(torch.int64), y_true.to(torch.int64)
    elif code in (_lib.TP_METRIC['mse'], _lib.TP_METRIC['mae'], _lib.TP_METRIC['r2']):
        y_pred, y_true = y_pred.to(torch.float32), y_true.to(torch.float32)
    else:
        y_pred, y_true = y_pred.to(torch.float32), y_true.to(torch.int64)
    y_pred, y_true = y_pred.contiguous(), y_true.contiguous()
    P = y_pred.shape[0]
    N = y_true.numel()
    out = torch.empty(P, dtype=torch.float32, device=y_pred.device)
    a = _lib.MetricArgs(metric=code, P=P, N=N, C=classes, y_pred=y_pred.data_ptr(), y_true=y_true.data_ptr(),
                        out=out.data_ptr())
    check(load().tp_metric_pack(ctypes.byref(a), _stream()), 'tp_metric_pack')
    return out


def greedy_ensemble(predictions: Tensor, y_true: Tensor, *, metric: str, maximize: bool, classes: int = 1,
                    init_top_k: int = 1, max_ensemble_size: int | None = None,
                    with_replacement: bool = False) -> tuple[Tensor, Tensor]:
    """Fused greedy selection; returns (counts (n_pred,) int32, status (3,) int32) on the device."""
    code = _lib.TP_METRIC[metric]
    pred = _cuda('predictions', predictions).to(torch.float32).contiguous()
    yt = _cuda('y_true', y_true)
    yt = (yt.to(torch.float32) if metric in ('mse', 'mae') else yt.to(torch.int64)).contiguous()
    n_pred = pred.shape[0]
    N = yt.numel()
    ws = torch.empty(int(load().tp_greedy_workspace_size(n_pred, N, classes)), dtype=torch.uint8, device=pred.device)
    counts = torch.empty(n_pred, dtype=torch.int32, device=pred.device)
    status = torch.zeros(3, dtype=torch.int32, device=pred.device)
    a = _lib.GreedyArgs(metric=code, maximize=int(maximize), n_pred=n_pred, N=N, C=classes,
                        predictions=pred.data_ptr(), y_true=yt.data_ptr(), init_top_k=init_top_k,
                        max_ensemble_size=0 if max_ensemble_size is None else int(max_ensemble_size),
                        with_replacement=int(with_replacement), counts=counts.data_ptr(), workspace=ws.data_ptr(),
                        workspace_bytes=ws.numel(), status=status.data_ptr())
    check(load().tp_greedy_ensemble(ctypes.byref(a), _stream()), 'tp_greedy_ensemble')
    return counts, status


def ensemble_mean(pred: Tensor, idx: Tensor, weights: Tensor | None = None) -> Tensor:
    """(Weighted) mean of pred[idx] over the first dimension; see `tp_ensemble_mean`."""
    pred = _cuda('pred', pred, torch.float32)
    idx = _i32('idx', idx)
    weights = None if weights is None else _cuda('weights', weights).to(torch.float32).contiguous()
    out = torch.empty(pred.shape[1:], dtype=torch.float32, device=pred.device)
    n = out.numel()
    check(load().tp_ensemble_mean(pred.data_ptr(), idx.data_ptr(), _ptr(weights), idx.numel(), n, out.data_ptr(),
                                  _stream()), 'tp_ensemble_mean')
    return out


def softmax_rows(x: Tensor) -> Tensor:
    """Softmax over the last dimension (fp32); see `tp_softmax_rows`."""
    x = _cuda('x', x).to(torch.float32).contiguous()
    out = torch.empty_like(x)
    C = x.shape[-1]
    check(load().tp_softmax_rows(x.data_ptr(), x.numel() // C, C, out.data_ptr(), _stream()), 'tp_softmax_rows')
    return out


def permutation_keys(*, seed: int, epoch: int, member_base: int, P: int, N: int, device) -> Tensor:
    """(P, N) int32 Philox keys whose per-row stable argsort is each member's batch order."""
    keys = torch.empty((P, N), dtype=torch.int32, device=device)
    check(load().tp_permutation_keys(int(seed) & 0xFFFFFFFFFFFFFFFF, int(epoch) & 0xFFFFFFFF,
                                     int(member_base) & 0xFFFFFFFF, P, N, keys.data_ptr(), _stream()),
          'tp_permutation_keys')
    return keys


def _cos_emb_args(x, weight, bias, affine_weight, affine_bias, d_embedding):
    P, F, D = affine_weight.shape
    for name, t in (('weight', weight), ('bias', bias), ('affine_weight', affine_weight),
                    ('affine_bias', affine_bias)):
        if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
            raise TypeError(f'{name} must be a contiguous fp32 CUDA tensor')
    x = _cuda('x', x, torch.float32)
    if x.ndim == 2:
        B, shared = x.shape[0], 1
    else:
        B, shared = x.shape[1], 0
    if x.shape[-1] != F:
        raise ValueError('The number of input features must match the number of features configured for the embeddings')
    d = _i32('d_embedding', d_embedding)
    a = _lib.CosEmbArgs(P=P, B=B, F=F, D=D, x_shared=shared, x=x.data_ptr(), weight=weight.data_ptr(),
                        bias=bias.data_ptr(), affine_weight=affine_weight.data_ptr(),
                        affine_bias=affine_bias.data_ptr(), d_embedding=_ptr(d))
    return a, (x, d)


def cos_emb_forward(x: Tensor, weight: Tensor, bias: Tensor, affine_weight: Tensor, affine_bias: Tensor,
                    d_embedding: Tensor | None = None, *, out: Tensor | None = None,
                    dtype: torch.dtype = torch.float32) -> Tensor:
    """Cosine embeddings of x (P, B, F) or shared (B, F) into the first F * D columns of `out`
    (P, B, >= F * D; allocated (P, B, F * D) of `dtype` when None); see `tp_cos_emb_forward`."""
    a, keep = _cos_emb_args(x, weight, bias, affine_weight, affine_bias, d_embedding)
    if out is None:
        out = torch.empty(a.P, a.B, a.F * a.D, dtype=dtype, device=weight.device)
    if out.stride(-1) != 1 or out.stride(0) != out.shape[1] * out.stride(1) or out.dtype not in (torch.float32,
                                                                                                   torch.bfloat16):
        raise TypeError('out must be a row-major fp32 or bf16 (P, B, width) tensor')
    a.out, a.out_ld = out.data_ptr(), out.stride(1)
    a.out_dtype = TP_DTYPE_BF16 if out.dtype == torch.bfloat16 else TP_DTYPE_F32
    check(load().tp_cos_emb_forward(ctypes.byref(a), _stream()), 'tp_cos_emb_forward')
    del keep
    return out


def cos_emb_backward(x: Tensor, weight: Tensor, bias: Tensor, affine_weight: Tensor, affine_bias: Tensor,
                     d_embedding: Tensor | None, grad_out: Tensor):
    """Parameter gradients (dweight, dbias, daffine_weight, daffine_bias) from the gradient of the
    flattened embedding (its first F * D columns); see `tp_cos_emb_backward`."""
    a, keep = _cos_emb_args(x, weight, bias, affine_weight, affine_bias, d_embedding)
    if grad_out.stride(-1) != 1 or grad_out.stride(0) != grad_out.shape[1] * grad_out.stride(1):
        grad_out = grad_out.contiguous()
    if grad_out.dtype not in (torch.float32, torch.bfloat16):
        grad_out = grad_out.float()
    a.grad_out, a.grad_ld = grad_out.data_ptr(), grad_out.stride(1)
    a.grad_dtype = TP_DTYPE_BF16 if grad_out.dtype == torch.bfloat16 else TP_DTYPE_F32
    dweight, dbias = torch.empty_like(weight), torch.empty_like(bias)
    daw, dab = torch.empty_like(affine_weight), torch.empty_like(affine_bias)
    a.dweight, a.dbias = dweight.data_ptr(), dbias.data_ptr()
    a.daffine_weight, a.daffine_bias = daw.data_ptr(), dab.data_ptr()
    need = int(load().tp_cos_emb_workspace_size(a.P, a.B, a.F, a.D))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=weight.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    check(load().tp_cos_emb_backward(ctypes.byref(a), _stream()), 'tp_cos_emb_backward')
    del keep
    return dweight, dbias, daw, dab


def tabpack_input(x_num: Tensor | None, x_cat: Tensor | None, cat_offsets: Tensor, width: int,
                  dtype: torch.dtype, row_index: Tensor | None = None, *, out: Tensor | None = None,
                  col0: int = 0) -> Tensor:
    """[x_num | one-hot(x_cat)] in `dtype`, zero-padded to `width` columns; leading dimensions
    of the inputs are kept, or with `row_index` (any shape, int64) output row r is built from
    dataset row row_index[r] and the output takes row_index's shape; see `tp_tabpack_input`.
    With `out` (contiguous, last dimension `width`) the columns from `col0` on are written into
    it and the columns before are left as they are."""
    ref = x_num if x_num is not None else x_cat
    ri = None if row_index is None else _cuda('row_index', row_index).to(torch.int64).contiguous()
    lead = ref.shape[:-1] if ri is None else ri.shape
    rows = ref[..., 0].numel() if ri is None else ri.numel()
    xn = None if x_num is None else _cuda('x_num', x_num).to(torch.float32).contiguous()
    xc = None if x_cat is None else _cuda('x_cat', x_cat).to(torch.int64).contiguous()
    if out is None:
        out = torch.empty(*lead, width, dtype=dtype, device=ref.device)
    elif (out.dtype != dtype or out.shape[-1] != width or not out.is_contiguous()
          or out.numel() != rows * width):
        raise ValueError('out must be a contiguous tensor of the rows x width output')
    a = _lib.InputArgs(rows=rows, n_num=0 if xn is None else xn.shape[-1], n_cat=0 if xc is None else xc.shape[-1],
                       x_num=_ptr(xn), x_cat=_ptr(xc), row_index=_ptr(ri), cat_offsets=cat_offsets.data_ptr(),
                       out=out.data_ptr(),
                       out_ld=width, out_dtype=TP_DTYPE_BF16 if dtype == torch.bfloat16 else TP_DTYPE_F32,
                       out_col0=int(col0))
    check(load().tp_tabpack_input(ctypes.byref(a), _stream()), 'tp_tabpack_input')
    return out


def weight_cast(src: Tensor, dst: Tensor, *, out_features: Tensor | None = None, in_features: Tensor | None = None,
                n_blocks: Tensor | None = None, block_index: int = 0, src_cols: int | None = None) -> Tensor:
    """Write bf16(src) into `dst` (P, dst_rows, dst_cols) over each active member's rows
    r < out_features[m], zero beyond in_features[m]; other rows of `dst` keep their contents
    (see `tp_weight_cast`).  `src_cols` takes only the first columns of each source row.
    Returns `dst`."""
    src = _cuda('src', src, torch.float32)
    dst = _cuda('dst', dst, torch.bfloat16)
    if not src.is_contiguous() or not dst.is_contiguous():
        raise ValueError('weight_cast needs contiguous tensors')
    P, R, ld = src.shape
    C = ld if src_cols is None else int(src_cols)
    if dst.shape[0] != P:
        raise ValueError('src and dst differ in their pack size')
    outf, inf, nb = (_i32(n, t) for n, t in (('out_features', out_features), ('in_features', in_features),
                                             ('n_blocks', n_blocks)))
    a = _lib.WeightCastArgs(P=P, src_rows=R, src_cols=C, src_ld=ld, dst_rows=dst.shape[1], dst_cols=dst.shape[2],
                            out_features=_ptr(outf), in_features=_ptr(inf), n_blocks=_ptr(nb),
                            block_index=block_index, src=src.data_ptr(), dst=dst.data_ptr())
    check(load().tp_weight_cast(ctypes.byref(a), _stream()), 'tp_weight_cast')
    increment_version(dst)
    return dst


def weight_cast_transposed(src: Tensor, dst: Tensor, *, col0: int, ncols: int,
                           out_features: Tensor | None = None) -> Tensor:
    """dst[m, j, n] = bf16(src[m, n, col0 + j]) over each member's rows n < out_features[m]
    (zeros up to the next multiple of 8); see `tp_weight_cast_transposed`.  Returns `dst`."""
    src = _cuda('src', src, torch.float32)
    dst = _cuda('dst', dst, torch.bfloat16)
    if not src.is_contiguous() or not dst.is_contiguous():
        raise ValueError('weight_cast_transposed needs contiguous tensors')
    P, R, ld = src.shape
    if tuple(dst.shape[:2]) != (P, ncols):
        raise ValueError('dst must be (P, ncols, dst_ld)')
    outf = _i32('out_features', out_features)
    a = _lib.WeightCastTArgs(P=P, src_rows=R, src_ld=ld, col0=int(col0), ncols=int(ncols), dst_ld=dst.shape[2],
                             out_features=_ptr(outf), src=src.data_ptr(), dst=dst.data_ptr())
    check(load().tp_weight_cast_transposed(ctypes.byref(a), _stream()), 'tp_weight_cast_transposed')
    increment_version(dst)
    return dst


def _round(n: int, k: int) -> int:
    return (n + k - 1) // k * k


def _onehot_args(oh: dict) -> _lib.OneHotArgs:
    a = _lib.OneHotArgs()
    a.n_dense, a.n_cat, a.n_onehot = oh['n_dense'], oh['n_cat'], oh['n_onehot']
    a.cat_offsets = oh['cat_offsets'].data_ptr()
    a.x_cat = oh['x_cat'].data_ptr()
    a.x_cat_member_stride = oh['x_cat_member_stride']
    a.row_index = _ptr(oh.get('row_index'))
    a.row_index_member_stride = oh.get('row_index_member_stride', 0)
    a.w_onehot_t = _ptr(oh.get('w_onehot_t'))
    a.wt_ld = 0 if oh.get('w_onehot_t') is None else oh['w_onehot_t'].shape[-1]
    a.sorted_keys = _ptr(oh.get('sorted_keys'))
    a.addend = _ptr(oh.get('addend'))
    a.addend_ld = 0 if oh.get('addend') is None else oh['addend'].shape[-1]
    return a


def onehot_linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None, *, x_cat: Tensor, cat_offsets: Tensor,
                          n_dense: int, w_onehot_t: Tensor, row_index: Tensor | None = None,
                          out_features: Tensor | None = None, relu: bool = False, dropout_p: Tensor | None = None,
                          seed: int = 0, offset: int = 0, member_base: int = 0,
                          need_sort: bool = True) -> tuple[Tensor, dict]:
    """First layer over [dense | one-hot(x_cat)] with the one-hot columns gathered (bf16);
    see `tp_onehot_linear_forward`.  x: dense input (P or 1, B, max_in) bf16; weight: the bf16
    dense weight copy (P, max_out, max_in); w_onehot_t: (P, n_onehot, >= max_out) bf16.
    x_cat: (B, n_cat) shared, (P, B, n_cat) per member, or dataset rows with row_index (P, B).
    Returns (y, state) where state holds the category sort the backward needs (skipped with
    need_sort=False: a forward that no backward follows)."""
    weight = _cuda('weight', weight, torch.bfloat16)
    x = _cuda('x', x, torch.bfloat16)
    bias = _cuda('bias', bias, torch.float32)
    dropout_p = _cuda('dropout_p', dropout_p, torch.float32)
    outf = _i32('out_features', out_features)
    xc = _cuda('x_cat', x_cat, torch.int64).contiguous()
    P, max_out, _ = weight.shape
    B = x.shape[-2]
    n_cat = xc.shape[-1]
    ri = None
    if row_index is not None:
        ri = _cuda('row_index', row_index, torch.int64).contiguous()
        if ri.shape[-1] != B or (ri.ndim == 2 and ri.shape[0] not in (1, P)):
            raise ValueError('row_index must be (B,) or (P, B)')
        xcs, ris = 0, (B if ri.ndim == 2 and ri.shape[0] == P else 0)
    else:
        if xc.shape[-2] != B:
            raise ValueError('x_cat rows must match the batch')
        xcs, ris = (B if xc.ndim == 3 else 0), 0
    n_onehot = int(w_onehot_t.shape[1])
    dev = x.device
    state = {
        'n_dense': int(n_dense), 'n_cat': n_cat, 'n_onehot': n_onehot, 'cat_offsets': cat_offsets, 'x_cat': xc,
        'x_cat_member_stride': xcs, 'row_index': ri, 'row_index_member_stride': ris, 'w_onehot_t': w_onehot_t,
        'sorted_keys': torch.empty((P, n_cat, B), dtype=torch.int64, device=dev) if need_sort else None,
        'addend': torch.empty((P, B, _round(max_out, 16)), dtype=torch.float32, device=dev),
    }
    y = torch.empty((P, B, max_out), dtype=torch.bfloat16, device=dev)
    a = _linear_args(x, weight, bias, None, outf, None, 0, relu, dropout_p, seed, offset, member_base, y)
    oa = _onehot_args(state)
    check(load().tp_onehot_linear_forward(ctypes.byref(a), ctypes.byref(oa), _stream()), 'tp_onehot_linear_forward')
    state['addend'] = state['w_onehot_t'] = None  # used by the forward only
    return y, state


def onehot_linear_backward(dy: Tensor, x: Tensor, weight: Tensor, y: Tensor, state: dict, *,
                           out_features: Tensor | None = None, relu: bool = False, dropout_p: Tensor | None = None,
                           seed: int = 0, offset: int = 0, member_base: int = 0, need_dx: bool = False,
                           need_db: bool = True, dw_rows: int, db_cols: int) -> tuple[Tensor | None, Tensor, Tensor | None]:
    """Backward of `onehot_linear_forward`: (dx of the dense input or None, dw (P, dw_rows,
    n_dense + n_onehot) fp32, db fp32); see `tp_onehot_linear_backward`."""
    weight = _cuda('weight', weight, torch.bfloat16)
    dy = _cuda('dy', dy, torch.bfloat16)
    dropout_p = _cuda('dropout_p', dropout_p, torch.float32)
    outf = _i32('out_features', out_features)
    P, max_out, max_in = weight.shape
    B = x.shape[-2]
    g = torch.empty_like(dy)
    dx = torch.empty((P, B, max_in), dtype=torch.bfloat16, device=dy.device) if need_dx else None
    cols = state['n_dense'] + state['n_onehot']
    dw = torch.empty((P, dw_rows, cols), dtype=torch.float32, device=dy.device)
    db = torch.empty((P, db_cols), dtype=torch.float32, device=dy.device) if need_db else None
    ga = _lib.LinearGradArgs()
    ga.fwd = _linear_args(x, weight, None, None, outf, None, 0, relu, dropout_p, seed, offset, member_base, None)
    ga.dy, ga.y, ga.g = _ptr(dy), _ptr(y), _ptr(g)
    ga.dbias, ga.dx, ga.dw = _ptr(db), _ptr(dx), _ptr(dw)
    ga.dw_rows, ga.dw_cols, ga.db_cols = dw_rows, cols, db_cols
    oa = _onehot_args(state)
    check(load().tp_onehot_linear_backward(ctypes.byref(ga), ctypes.byref(oa), _stream()), 'tp_onehot_linear_backward')
    return dx, dw, db


def binary_roc_auc(scores: Tensor, labels: Tensor, workspace: Tensor | None = None) -> Tensor:
    """(P,) ROC AUC of each row of `scores` (P, N) fp32/fp64 against int64 labels (N,);
    see `tp_binary_roc_auc`.  The result has the scores' dtype."""
    scores = _cuda('scores', scores).contiguous()
    labels = _cuda('labels', labels, torch.int64).contiguous()
    if scores.dtype not in (torch.float32, torch.float64):
        raise TypeError('scores must be float32 or float64')
    P, N = scores.shape
    dtype = _lib.TP_DTYPE_F64 if scores.dtype == torch.float64 else _lib.TP_DTYPE_F32
    need = int(load().tp_roc_auc_workspace_size(P, N, dtype))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=scores.device)
    out = torch.empty(P, dtype=scores.dtype, device=scores.device)
    check(load().tp_binary_roc_auc(scores.data_ptr(), labels.data_ptr(), P, N, dtype, out.data_ptr(),
                                   workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream()),
          'tp_binary_roc_auc')
    return out


_functions: dict = {}


def _function(name: str):
    """The library's function of that name."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(load(), name)
    return fn


def _call(name: str, args, device: int) -> None:
    """`name(args)` on the current stream of device number `device`, whichever device is current.
    (The raw stream handle: building a `torch.cuda.Stream` takes as long as the launch.)"""
    fn = _functions.get(name) or _function(name)
    if device == torch._C._cuda_getDevice():
        check(fn(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(device)), name)
    else:
        with torch.cuda.device(device):
            check(fn(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(device)), name)


def _device_of(name: str, t: Tensor) -> int:
    i = t.get_device()
    if i < 0:
        raise RuntimeError(f'{name} must be a CUDA tensor (tabpack_b200 has no CPU path)')
    return i


def _operand(name: str, t: Tensor | None, shape: tuple, dtype: torch.dtype, device: int) -> Tensor | None:
    """`t` contiguous, checked against the shape, type and device that it has to have."""
    if t is None:
        return None
    if t.dtype is not dtype:
        raise TypeError(f'{name} must have dtype {dtype}, got {t.dtype}')
    if t.shape != shape:
        raise ValueError(f'{name} must be {shape}, got {tuple(t.shape)}')
    if t.get_device() != device:
        raise ValueError(f'{name} must be on cuda:{device}, got {t.device}')
    return t if t.is_contiguous() else t.contiguous()


def _empty2(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> Tensor:
    """A contiguous (rows, cols) tensor (the strided form is the cheapest of torch's factories)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _empty(shape: tuple, dtype: torch.dtype, device: torch.device) -> Tensor:
    strides, n = [], 1
    for d in reversed(shape):
        strides.append(n)
        n *= d
    return torch.empty_strided(shape, strides[::-1], dtype=dtype, device=device)


def _empty3(a: int, b: int, c: int, dtype: torch.dtype, device: torch.device) -> Tensor:
    return torch.empty_strided((a, b, c), (b * c, c, 1), dtype=dtype, device=device)


def _empty_as(t: Tensor, dtype: torch.dtype) -> Tensor:
    """A contiguous tensor of t's shape."""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else t.new_empty(tuple(t.shape), dtype=dtype)


ADAMW8_BLOCK = 128
"""Elements of a member that share one scale per moment in `adamw8_step`'s states."""


def adamw8_state(p: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Zero moments of `adamw8_step` for a parameter pack (P, ...): (exp_avg, exp_avg_scale,
    exp_avg_sq, exp_avg_sq_scale), uint8 codes of p's shape and fp32 (P, blocks) scales."""
    P = p.shape[0]
    nb = (p.numel() // max(P, 1) + ADAMW8_BLOCK - 1) // ADAMW8_BLOCK
    codes = lambda: torch.zeros(p.shape, dtype=torch.uint8, device=p.device)  # noqa: E731
    scales = lambda: torch.zeros((P, nb), dtype=torch.float32, device=p.device)  # noqa: E731
    return codes(), scales(), codes(), scales()


def _adamw8_state_fits(shape, P: int, nb: int, device: int, m: Tensor, ms: Tensor, v: Tensor, vs: Tensor) -> bool:
    return (m.dtype is torch.uint8 and v.dtype is torch.uint8 and m.shape == shape and v.shape == shape
            and ms.dtype is torch.float32 and vs.dtype is torch.float32 and ms.shape == (P, nb) and vs.shape == (P, nb)
            and m.get_device() == device and v.get_device() == device and ms.get_device() == device
            and vs.get_device() == device and m.is_contiguous() and v.is_contiguous() and ms.is_contiguous()
            and vs.is_contiguous())


def _adamw8_state_error(shape, P: int, nb: int, device: int) -> TypeError:
    return TypeError(f'exp_avg and exp_avg_sq must be contiguous uint8 {tuple(shape)} tensors, exp_avg_scale and '
                     f'exp_avg_sq_scale contiguous fp32 ({P}, {nb}) tensors, on cuda:{device}')


def adamw8_step(params, grads, exp_avgs, exp_avg_scales, exp_avg_sqs, exp_avg_sq_scales, *, steps=None,
                step: int = 0, lr, beta1, beta2, eps, weight_decay, seed: int, member_base: int = 0,
                tensor_base: int = 0) -> None:
    """Grouped AdamW over parameter packs (each (P, ...) fp32, contiguous) with both moments in
    8 bits, in place; see `tp_adamw8_step` and `adamw8_state`.

    `steps` (per-tensor (P,) int64 tensors, already incremented) or the scalar `step` give the
    bias-correction step.  Hyperparameters are floats or (P,) fp32 CUDA tensors.  `seed`, the
    step, the member (`member_base` + position) and the tensor's number (`tensor_base` + position)
    give the random bits of the moments' rounding.  Tensors are chunked into launches of at most 32.
    """
    n = len(params)
    if not n == len(grads) == len(exp_avgs) == len(exp_avg_scales) == len(exp_avg_sqs) == len(exp_avg_sq_scales) or (
            steps is not None and len(steps) != n):
        raise ValueError('one gradient, state and step per parameter is required')
    if steps is None and int(step) <= 0:
        raise ValueError('the step count must be positive')
    if n == 0:
        return
    device = _device_of('param', params[0])
    hp, members = [], None
    for name, v in (('lr', lr), ('beta1', beta1), ('beta2', beta2), ('eps', eps), ('weight_decay', weight_decay)):
        if isinstance(v, Tensor):
            if v.get_device() != device:
                raise ValueError(f'{name} must be on cuda:{device}, got {v.device}')
            if members not in (None, v.numel()):
                raise ValueError('per-member hyperparameters must have one value per member')
            v, members = v.contiguous(), v.numel()
        hp.append(v)
    f32 = torch.float32
    calls, a, used, count, written = [], None, 0, 0, set()
    for i, p in enumerate(params):
        g, m, ms, v, vs = grads[i], exp_avgs[i], exp_avg_scales[i], exp_avg_sqs[i], exp_avg_sq_scales[i]
        shape = p.shape
        if p.dtype is not f32 or p.get_device() != device or not p.is_contiguous() or not shape:
            raise TypeError(f'param must be a contiguous fp32 tensor with a pack dimension on cuda:{device}')
        if g.dtype is not f32 or g.get_device() != device or g.shape != shape or not g.is_contiguous():
            raise TypeError(f'grad must be a contiguous fp32 tensor of the shape of its parameter on cuda:{device}')
        P, numel = shape[0], p.numel()
        inner = numel // P if P else 0
        nb = (inner + ADAMW8_BLOCK - 1) // ADAMW8_BLOCK
        if not _adamw8_state_fits(shape, P, nb, device, m, ms, v, vs):
            raise _adamw8_state_error(shape, P, nb, device)
        if members is not None and members != P:
            raise ValueError('per-member hyperparameters must have one value per member')
        st = None
        if steps is not None:
            st = steps[i]
            if st.dtype is not torch.int64 or st.shape != (P,) or st.get_device() != device or not st.is_contiguous():
                raise TypeError(f'steps must be contiguous int64 ({P},) tensors on cuda:{device}')
            st = st.data_ptr()
        if numel == 0:
            continue
        if used % _lib.TP_MAX_OPT_TENSORS == 0:
            a = _lib.AdamW8Args()
            calls.append(a)
            used = 0
        out = p.data_ptr(), m.data_ptr(), ms.data_ptr(), v.data_ptr(), vs.data_ptr()
        written.update(out)
        a.t[used] = (out[0], g.data_ptr(), *out[1:], st, numel, inner, (tensor_base + i) & 0xFFFFFFFF)
        used += 1
        count += 1
        a.n_tensors = used
    values = [_hparam(v) for v in hp]  # bare pointers: `hp` holds the contiguous copies until the last launch
    if len(written) < 5 * count:
        raise ValueError('a parameter or a state appears twice')
    # every argument is checked before the first launch
    for a in calls:
        a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = values
        a.step, a.seed = int(step), int(seed) & 0xFFFFFFFFFFFFFFFF
        a.member_base = int(member_base) & 0xFFFFFFFF
        _call('tp_adamw8_step', a, device)
    # updated in place: bump the version counters as torch's in-place ops do
    increment_version([*params, *exp_avgs, *exp_avg_scales, *exp_avg_sqs, *exp_avg_sq_scales])


def adamw8_moments(exp_avgs, exp_avg_scales, exp_avg_sqs, exp_avg_sq_scales, *,
                   dtype: torch.dtype = torch.float32) -> tuple[list[Tensor], list[Tensor]]:
    """The moments that `adamw8_step`'s states stand for: lists of exp_avg and exp_avg_sq, of the
    codes' shapes in fp32 or bf16 (a code has at most five significant bits, its square ten: bf16
    rounds the latter); see `tp_adamw8_moments`."""
    n = len(exp_avgs)
    if not n == len(exp_avg_scales) == len(exp_avg_sqs) == len(exp_avg_sq_scales):
        raise ValueError('every state needs its codes and scales')
    code = _dtype_code(dtype)
    if n == 0:
        return [], []
    device = _device_of('exp_avg', exp_avgs[0])
    out_m, out_v = [], []
    calls, a, used = [], None, 0
    for i, m in enumerate(exp_avgs):
        ms, v, vs = exp_avg_scales[i], exp_avg_sqs[i], exp_avg_sq_scales[i]
        shape = m.shape
        if not shape:
            raise TypeError('a state must have a pack dimension')
        P, numel = shape[0], m.numel()
        inner = numel // P if P else 0
        nb = (inner + ADAMW8_BLOCK - 1) // ADAMW8_BLOCK
        if not _adamw8_state_fits(shape, P, nb, device, m, ms, v, vs):
            raise _adamw8_state_error(shape, P, nb, device)
        om, ov = torch.empty_like(m, dtype=dtype), torch.empty_like(m, dtype=dtype)
        out_m.append(om)
        out_v.append(ov)
        if numel == 0:
            continue
        if used % _lib.TP_MAX_OPT_TENSORS == 0:
            a = _lib.AdamW8MomentsArgs(dtype=code)
            calls.append(a)
            used = 0
        a.t[used] = (m.data_ptr(), ms.data_ptr(), v.data_ptr(), vs.data_ptr(), om.data_ptr(), ov.data_ptr(), numel, inner)
        used += 1
        a.n_tensors = used
    for a in calls:
        _call('tp_adamw8_moments', a, device)
    return out_m, out_v


def _norm_rows(name: str, t: Tensor, dtype: torch.dtype, device: int, shape: tuple) -> tuple[Tensor, int, int]:
    """`t` with contiguous columns (copied where they are not), and its member and row strides; a
    (batch, features) tensor is shared by the members (member stride 0)."""
    if t.dtype is not dtype:
        raise TypeError(f'{name} must have dtype {dtype}, got {t.dtype}')
    if t.get_device() != device:
        raise ValueError(f'{name} must be on cuda:{device}, got {t.device}')
    if t.shape != (shape if t.ndim == 3 else shape[1:]):
        raise ValueError(f'{name} must be {shape} or {shape[1:]}, got {tuple(t.shape)}')
    stride = t.stride()
    if stride[-1] != 1 and shape[2] != 1:
        t = t.contiguous()
        stride = t.stride()
    return t, stride[0] if len(stride) == 3 and shape[0] > 1 else 0, stride[-2] if shape[1] > 1 else 0


def layer_norm_forward(x: Tensor, weight: Tensor | None, bias: Tensor | None, *, n_features: Tensor | None = None,
                       eps: float = 1e-5, pack_size: int | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """Layer norm of x (P, B, W), or (B, W) shared by the members, bf16 or fp32, with each member's
    own weight and bias (P, W) fp32 or None; see `tp_layer_norm_forward`.  `n_features` (P,): member
    m's rows are normalised over their first n_features[m] columns, the others are zero in y.
    `pack_size`: P, where a shared x has nothing else that tells it (1 if not given).
    Returns (y (P, B, W), mean (P, B), rstd (P, B)); the backward takes the last two."""
    if not 0.0 <= eps < float('inf'):
        raise ValueError('eps must be finite and not negative')
    if x.ndim not in (2, 3):
        raise ValueError('x must be (pack_size, batch, features) or a shared (batch, features)')
    device, dtype = _device_of('x', x), x.dtype
    code = _dtype_code(dtype)
    if x.ndim == 3:
        P, B, W = x.shape
        if pack_size not in (None, P):
            raise ValueError(f'x has {P} members, not {pack_size}')
    else:
        B, W = x.shape
        if pack_size is not None and pack_size < 0:
            raise ValueError('the pack size must not be negative')
        P = pack_size
        if P is None:
            P = next((t.shape[0] for t in (weight, bias, n_features) if t is not None), 1)
    x, sm, sr = _norm_rows('x', x, dtype, device, (P, B, W))
    weight = _operand('weight', weight, (P, W), torch.float32, device)
    bias = _operand('bias', bias, (P, W), torch.float32, device)
    if n_features is not None:
        n_features = _operand('n_features', n_features if n_features.dtype is torch.int32
                              else n_features.to(torch.int32), (P,), torch.int32, device)
    y = _empty_as(x, dtype) if x.ndim == 3 else x.new_empty((P, B, W))
    mean, rstd = _empty2(P, B, torch.float32, x.device), _empty2(P, B, torch.float32, x.device)
    if P and B and W:
        a = _lib.LayerNormArgs(P, B, W, code, sm, sr, _ptr(n_features), x.data_ptr(), _ptr(weight), _ptr(bias), eps,
                               y.data_ptr(), mean.data_ptr(), rstd.data_ptr())
        _call('tp_layer_norm_forward', a, device)
    return y, mean, rstd


def layer_norm_backward(dy: Tensor, x: Tensor, weight: Tensor | None, mean: Tensor, rstd: Tensor, *,
                        n_features: Tensor | None = None, need_dx: bool = True, need_dw: bool = True,
                        need_db: bool = True) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """Backward of `layer_norm_forward`: (dx of x's shape and type, dw (P, W), db (P, W) fp32); a
    shared x takes the sum over the members.  See `tp_layer_norm_backward`."""
    if dy.ndim != 3 or x.ndim not in (2, 3):
        raise ValueError('dy must be (pack_size, batch, features), and x too or shared (batch, features)')
    device, dtype = _device_of('x', x), x.dtype
    code = _dtype_code(dtype)
    shape = P, B, W = tuple(dy.shape)
    x, sm, sr = _norm_rows('x', x, dtype, device, shape)
    dy, dm, dr = _norm_rows('dy', dy, dtype, device, shape)
    weight = _operand('weight', weight, (P, W), torch.float32, device)
    if n_features is not None:
        n_features = _operand('n_features', n_features if n_features.dtype is torch.int32
                              else n_features.to(torch.int32), (P,), torch.int32, device)
    for name, t in (('mean', mean), ('rstd', rstd)):
        if t.shape != (P, B) or t.dtype is not torch.float32 or t.get_device() != device or not t.is_contiguous():
            raise TypeError(f'{name} must be the contiguous fp32 ({P}, {B}) tensor of the forward')
    dx = dw = db = None
    # the members' terms of a shared input are added up before they are rounded
    terms = 0
    if need_dx:
        dx = _empty2(B, W, dtype, x.device) if x.ndim == 2 else _empty_as(dy, dtype)
        terms = P * B * W if x.ndim == 2 and P > 1 else 0
    if need_dw:
        dw = _empty2(P, W, torch.float32, x.device)
    if need_db:
        db = _empty2(P, W, torch.float32, x.device)
    if P and B and W and (need_dx or need_dw or need_db):
        need = load().tp_layer_norm_workspace_size(P, B, W) if need_dw or need_db else 0
        ws = None
        if need or terms:
            scratch = torch.empty_strided((terms + need // 4,), (1,), dtype=torch.float32, device=x.device)
            ws = scratch.data_ptr()
        a = _lib.LayerNormArgs(P, B, W, code, sm, sr, _ptr(n_features), x.data_ptr(), _ptr(weight), None, 0.0, None,
                               mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), dm, dr, ws if terms else _ptr(dx),
                               TP_DTYPE_F32 if terms else code, dx.data_ptr() if terms else None, _ptr(dw), _ptr(db),
                               ws + 4 * terms if need else None, need)
        _call('tp_layer_norm_backward', a, device)
    else:
        for t in (dx, dw, db):
            if t is not None:
                t.zero_()
    return dx, dw, db


def _logit_rows(logits: Tensor) -> tuple[Tensor, int, int]:
    """logits (..., C) as rows at one stride: (tensor, rows, stride), copied only where the rows
    are not at one stride."""
    shape, strides = logits.shape, logits.stride()
    C = shape[-1]
    if logits.is_contiguous():
        return logits, logits.numel() // C, C
    rows, stride, ok = 1, C, C == 1 or strides[-1] == 1
    for d in range(len(shape) - 2, -1, -1):
        if shape[d] != 1:
            if rows == 1:
                stride = strides[d]
            elif strides[d] != stride * rows:
                ok = False
            rows *= shape[d]
    if not ok or stride < C:
        logits, stride = logits.contiguous(), C
    return logits, rows, stride


def _log_probs_operands(logits: Tensor, labels: Tensor):
    device = _device_of('logits', logits)
    lead = logits.shape[:-1]
    if logits.ndim == 0 or logits.shape[-1] == 0:
        raise ValueError('logits must have at least one class')
    if labels.dtype is not torch.int64:
        raise TypeError('labels must have the int64 data type')
    if labels.shape != lead[len(lead) - labels.ndim:] or labels.ndim > len(lead):
        raise ValueError('The label and logit shapes are incompatible; only missing leading label dimensions '
                         'may be broadcast')
    if labels.get_device() != device:
        raise ValueError(f'labels must be on cuda:{device}, got {labels.device}')
    code = _dtype_code(logits.dtype)
    logits, rows, stride = _logit_rows(logits)
    return device, code, lead, logits, rows, stride, labels if labels.is_contiguous() else labels.contiguous()


def label_log_probs_forward(logits: Tensor, labels: Tensor, *, top_k: int = 0, ignore_index: int = -100
                            ) -> tuple[Tensor, Tensor, Tensor | None, Tensor | None, Tensor | None]:
    """Log probabilities of `labels` under softmax(logits), with entropies and the `top_k` best
    classes; see `tp_label_log_probs_forward`.  logits (..., C) bf16 or fp32; labels int64 of
    the leading shape, or without its first dimensions (labels that the members share).  Returns
    (log_prob, entropy, top_log_prob or None, top_label or None, stats or None): fp32 of the leading
    shape, (..., top_k) fp32 and int64, and what the backward takes."""
    device, code, lead, logits, rows, stride, labels = _log_probs_operands(logits, labels)
    C = logits.shape[-1]
    if not 0 <= top_k <= min(C, _lib.TP_MAX_TOP_K):
        raise ValueError(f'top_k must be between 0 and {min(C, _lib.TP_MAX_TOP_K)}, got {top_k}')
    f32 = torch.float32
    if labels.shape == lead:
        log_prob, entropy = torch.empty_like(labels, dtype=f32), torch.empty_like(labels, dtype=f32)
    else:
        log_prob, entropy = (logits.new_empty(tuple(lead), dtype=f32) for _ in range(2))
    stats = _empty2(rows, 3, f32, logits.device) if C > _lib.TP_LABEL_STATS_CLASSES else None
    top = which = None
    if top_k:
        top = logits.new_empty((*lead, top_k), dtype=f32)
        which = logits.new_empty((*lead, top_k), dtype=torch.int64)
    if rows:
        a = _lib.LabelLogProbsArgs(rows, C, code, logits.data_ptr(), stride, labels.data_ptr(), labels.numel(),
                                   ignore_index, top_k, log_prob.data_ptr(), entropy.data_ptr(), _ptr(top),
                                   _ptr(which), _ptr(stats))
        _call('tp_label_log_probs_forward', a, device)
    return log_prob, entropy, top, which, stats


def _row_gradient(name: str, g: Tensor | None, lead, device: int) -> tuple[Tensor | None, int]:
    """A per-row fp32 gradient and its stride: 0 for one value that was expanded over the rows."""
    if g is None:
        return None, 0
    if g.shape != lead or g.dtype is not torch.float32 or g.get_device() != device:
        raise TypeError(f'{name} must be a {tuple(lead)} fp32 tensor on cuda:{device}')
    if g.is_contiguous():
        return g, 1
    if not any(g.stride()):
        return g, 0
    return g.contiguous(), 1


def label_log_probs_backward(g_log_prob: Tensor | None, g_entropy: Tensor | None, logits: Tensor, labels: Tensor,
                             stats: Tensor | None, *, ignore_index: int = -100) -> Tensor:
    """The gradient of the logits (contiguous, of their shape and type) from the gradients of
    `label_log_probs_forward`'s log_prob and entropy (either may be None);
    see `tp_label_log_probs_backward`."""
    device, code, lead, logits, rows, stride, labels = _log_probs_operands(logits, labels)
    C = logits.shape[-1]
    if C > _lib.TP_LABEL_STATS_CLASSES and (stats is None or stats.shape != (rows, 3) or stats.get_device() != device
                                            or stats.dtype is not torch.float32 or not stats.is_contiguous()):
        raise TypeError('stats must be the tensor that the forward returned')
    g_log_prob, sl = _row_gradient('g_log_prob', g_log_prob, lead, device)
    g_entropy, sh = _row_gradient('g_entropy', g_entropy, lead, device)
    dlogits = _empty_as(logits, logits.dtype)
    if rows:
        a = _lib.LabelLogProbsArgs(rows, C, code, logits.data_ptr(), stride, labels.data_ptr(), labels.numel(),
                                   ignore_index, 0, None, None, None, None, _ptr(stats), _ptr(g_log_prob),
                                   _ptr(g_entropy), sl, sh, dlogits.data_ptr())
        _call('tp_label_log_probs_backward', a, device)
    return dlogits


def _rows2(name: str, t: Tensor, shape: tuple, dtype: torch.dtype, device: int) -> tuple[Tensor, int]:
    """A matrix with contiguous columns and rows that do not overlap (copied where it has none), and its row stride."""
    if t.dtype is not dtype:
        raise TypeError(f'{name} must have dtype {dtype}, got {t.dtype}')
    if t.shape != shape:
        raise ValueError(f'{name} must be {shape}, got {tuple(t.shape)}')
    if t.get_device() != device:
        raise ValueError(f'{name} must be on cuda:{device}, got {t.device}')
    if t.is_contiguous():
        return t, shape[1]
    sr, sc = t.stride()
    if (sc != 1 and shape[1] != 1) or (shape[0] > 1 and sr < shape[1]):
        return t.contiguous(), shape[1]
    return t, sr if shape[0] > 1 else shape[1]


def _members(name: str, t: Tensor | None, n: int, device: int) -> Tensor | None:
    """Whole numbers of the members as int32, or None."""
    if t is None:
        return None
    if t.is_floating_point() or t.is_complex() or t.dtype is torch.bool:
        raise TypeError(f'{name} must hold whole numbers, got {t.dtype}')
    return _operand(name, t if t.dtype is torch.int32 else t.to(torch.int32), (n,), torch.int32, device)


def route_forward(logits: Tensor, top_k: int, *, renormalize: bool = True
                  ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Routing of rows to members by scores (T, E), bf16 or fp32; see `tp_route_forward`.  Returns
    (weight (T, top_k) fp32, expert (T, top_k) int32, position (T, top_k) int32, offsets (E + 1,)
    int32, importance (E,) fp32)."""
    if logits.ndim != 2:
        raise ValueError('logits must be (rows, members)')
    device = _device_of('logits', logits)
    code = _dtype_code(logits.dtype)
    T, E = logits.shape
    if not 1 <= E <= _lib.TP_ROUTE_MAX_EXPERTS:
        raise ValueError(f'logits must have 1 to {_lib.TP_ROUTE_MAX_EXPERTS} members, got {E}')
    if not 1 <= top_k <= min(E, _lib.TP_ROUTE_MAX_K):
        raise ValueError(f'top_k must be between 1 and {min(E, _lib.TP_ROUTE_MAX_K)}, got {top_k}')
    logits, stride = _rows2('logits', logits, (T, E), logits.dtype, device)
    dev, i32, f32 = logits.device, torch.int32, torch.float32
    weight, expert, position = _empty2(T, top_k, f32, dev), _empty2(T, top_k, i32, dev), _empty2(T, top_k, i32, dev)
    if not T:
        return weight, expert, position, torch.zeros(E + 1, dtype=i32, device=dev), torch.zeros(E, device=dev)
    offsets = torch.empty_strided((E + 1,), (1,), dtype=i32, device=dev)
    importance = torch.empty_strided((E,), (1,), dtype=f32, device=dev)
    need = _function('tp_route_workspace_size')(T, E, top_k)
    ws = torch.empty_strided((need // 4,), (1,), dtype=i32, device=dev) if need else None
    a = _lib.RouteArgs(T, E, top_k, code, int(renormalize), logits.data_ptr(), stride, weight.data_ptr(),
                       expert.data_ptr(), position.data_ptr(), offsets.data_ptr(), importance.data_ptr(), _ptr(ws),
                       need)
    _call('tp_route_forward', a, device)
    return weight, expert, position, offsets, importance


def route_backward(g_weight: Tensor | None, g_importance: Tensor | None, logits: Tensor, weight: Tensor, expert: Tensor,
                   *, renormalize: bool = True) -> Tensor:
    """The scores' gradient (contiguous, of their shape and type) from those of `route_forward`'s
    weight and importance (either may be None); see `tp_route_backward`."""
    if logits.ndim != 2 or weight.ndim != 2:
        raise ValueError('logits must be (rows, members), weight (rows, top_k)')
    device = _device_of('logits', logits)
    code = _dtype_code(logits.dtype)
    T, E = logits.shape
    k = weight.shape[1]
    if not 1 <= E <= _lib.TP_ROUTE_MAX_EXPERTS or not 1 <= k <= min(E, _lib.TP_ROUTE_MAX_K):
        raise ValueError(f'{k} of {E} members cannot be routed to')
    logits, stride = _rows2('logits', logits, (T, E), logits.dtype, device)
    weight = _operand('weight', weight, (T, k), torch.float32, device)
    expert = _operand('expert', expert, (T, k), torch.int32, device)
    g_weight = _operand('g_weight', g_weight, (T, k), torch.float32, device)
    g_importance = _operand('g_importance', g_importance, (E,), torch.float32, device)
    dlogits = _empty2(T, E, logits.dtype, logits.device)
    if T:
        a = _lib.RouteArgs(T, E, k, code, int(renormalize), logits.data_ptr(), stride, weight.data_ptr(),
                           expert.data_ptr(), None, None, None, None, 0, _ptr(g_weight), _ptr(g_importance),
                           dlogits.data_ptr())
        _call('tp_route_backward', a, device)
    return dlogits


def _plan(position: Tensor, offsets: Tensor, device: int) -> tuple[Tensor, Tensor, int, int, int]:
    if position.ndim != 2 or offsets.ndim != 1 or offsets.shape[0] < 2:
        raise ValueError('position must be (rows, k), offsets (members + 1,)')
    T, k = position.shape
    if not 1 <= k <= _lib.TP_ROUTE_MAX_K:
        raise ValueError(f'a row goes to 1 to {_lib.TP_ROUTE_MAX_K} members, got {k}')
    E = offsets.shape[0] - 1
    return (_operand('position', position, (T, k), torch.int32, device),
            _operand('offsets', offsets, (E + 1,), torch.int32, device), T, k, E)


def dispatch_rows(x: Tensor, position: Tensor, offsets: Tensor) -> Tensor:
    """(T k, W): row t of x (T, W) at each of its places, zero rows behind the last member's; see
    `tp_dispatch_rows`.  `position` and `offsets` are `route_forward`'s."""
    if x.ndim != 2:
        raise ValueError('x must be (rows, features)')
    device = _device_of('x', x)
    code = _dtype_code(x.dtype)
    position, offsets, T, k, E = _plan(position, offsets, device)
    W = x.shape[1]
    x, stride = _rows2('x', x, (T, W), x.dtype, device)
    out = _empty2(T * k, W, x.dtype, x.device)
    if T and W:
        a = _lib.RowsArgs(T, k, W, E, code, position.data_ptr(), offsets.data_ptr(), None, x.data_ptr(), stride,
                          out.data_ptr())
        _call('tp_dispatch_rows', a, device)
    return out


def combine_rows(y: Tensor, weight: Tensor | None, position: Tensor, offsets: Tensor) -> Tensor:
    """(T, W): the sum of a row's k rows of y (T k, W), times weight (T, k) fp32 if given; see
    `tp_combine_rows`.  Without a weight it is also the backward of `dispatch_rows`."""
    if y.ndim != 2:
        raise ValueError('y must be (rows k, features)')
    device = _device_of('y', y)
    code = _dtype_code(y.dtype)
    position, offsets, T, k, E = _plan(position, offsets, device)
    W = y.shape[1]
    y, stride = _rows2('y', y, (T * k, W), y.dtype, device)
    weight = _operand('weight', weight, (T, k), torch.float32, device)
    out = _empty2(T, W, y.dtype, y.device)
    if T and W:
        a = _lib.RowsArgs(T, k, W, E, code, position.data_ptr(), offsets.data_ptr(), _ptr(weight), y.data_ptr(), stride,
                          out.data_ptr())
        _call('tp_combine_rows', a, device)
    return out


def combine_rows_backward(dout: Tensor, y: Tensor, weight: Tensor | None, position: Tensor, offsets: Tensor, *,
                          need_dy: bool = True, need_dweight: bool = True) -> tuple[Tensor | None, Tensor | None]:
    """Backward of `combine_rows`: (dy (T k, W), zero rows behind the last member's; dweight (T, k));
    see `tp_combine_rows_backward`."""
    if dout.ndim != 2 or y.ndim != 2:
        raise ValueError('dout must be (rows, features), y (rows k, features)')
    device = _device_of('y', y)
    code = _dtype_code(y.dtype)
    position, offsets, T, k, E = _plan(position, offsets, device)
    W = y.shape[1]
    y, stride = _rows2('y', y, (T * k, W), y.dtype, device)
    dout, dstride = _rows2('dout', dout, (T, W), y.dtype, device)
    weight = _operand('weight', weight, (T, k), torch.float32, device)
    dy = _empty2(T * k, W, y.dtype, y.device) if need_dy else None
    dw = _empty2(T, k, torch.float32, y.device) if need_dweight else None
    if T and W and (need_dy or need_dweight):
        a = _lib.RowsArgs(T, k, W, E, code, position.data_ptr(), offsets.data_ptr(), _ptr(weight), y.data_ptr(), stride,
                          None, dout.data_ptr(), dstride, _ptr(dy), _ptr(dw))
        _call('tp_combine_rows_backward', a, device)
    elif dw is not None:
        dw.zero_()
    return dy, dw


def _align_rows(t: Tensor, stride: int, rows: int, cols: int, device: int) -> tuple[Tensor, int]:
    """`rows` bf16 rows of t, `stride` elements apart, as rows on 16-byte boundaries; see `tp_align_rows`."""
    wide = _round(cols, 8)
    out = _empty2(rows, wide, t.dtype, t.device)
    if rows:
        args = t.data_ptr(), stride, rows, cols, out.data_ptr(), wide, torch._C._cuda_getCurrentRawStream(device)
        if device == torch._C._cuda_getDevice():
            check(_function('tp_align_rows')(*args), 'tp_align_rows')
        else:
            with torch.cuda.device(device):
                check(_function('tp_align_rows')(*args), 'tp_align_rows')
    return out, wide


def _vector_rows(name: str, t: Tensor, shape: tuple, device: int) -> tuple[Tensor, int]:
    """A matrix as an operand of the ragged products: bf16 rows on 16-byte boundaries (copied to such where not)."""
    t, stride = _rows2(name, t, shape, t.dtype, device)
    if t.dtype is torch.bfloat16 and (stride % 8 or t.data_ptr() % 16):
        return _align_rows(t, stride, shape[0], shape[1], device)
    return t, stride


def _ragged_weight(weight: Tensor, device: int) -> tuple[Tensor, int]:
    P, N, K = weight.shape
    if weight.is_contiguous() and (weight.dtype is torch.float32 or (K % 8 == 0 and weight.data_ptr() % 16 == 0)):
        return weight, K
    s = weight.stride()
    if s[2] == 1 and s[1] >= K and s[0] == N * s[1] and (weight.dtype is torch.float32 or (
            s[1] % 8 == 0 and weight.data_ptr() % 16 == 0)):
        return weight, s[1]
    if weight.dtype is torch.float32:
        return weight.contiguous(), K
    wide, cols = _align_rows(weight.contiguous(), K, P * N, K, device)
    return wide.view(P, N, cols), cols


def _ragged_operands(x, weight, offsets, in_features, out_features):
    if x.ndim != 2 or weight.ndim != 3:
        raise ValueError('x must be (rows, features), weight (pack_size, out, in)')
    device, dtype = _device_of('x', x), x.dtype
    code = _dtype_code(dtype)
    P, N, K = weight.shape
    if not P or not N or not K:
        raise ValueError('weight must not be empty')
    if weight.dtype is not dtype:
        raise TypeError(f'weight must have dtype {dtype}, got {weight.dtype}')
    if weight.get_device() != device:
        raise ValueError(f'weight must be on cuda:{device}, got {weight.device}')
    if x.shape[1] != K:
        raise ValueError(f'x must have {K} features, got {x.shape[1]}')
    offsets = _members('offsets', offsets, P + 1, device)
    return (device, code, offsets, _members('in_features', in_features, P, device),
            _members('out_features', out_features, P, device))


def ragged_linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None, offsets: Tensor, *,
                          in_features: Tensor | None = None, out_features: Tensor | None = None,
                          relu: bool = False) -> Tensor:
    """Linear layer (+ReLU) of a pack over ragged groups of rows: member m's rows are
    x[offsets[m] : offsets[m + 1]] of x (R, in), bf16 or fp32 like weight (P, out, in); bias (P, out)
    fp32 or None; offsets (P + 1,) on the device, not decreasing, within 0 .. R.  Returns y (R, out), zero
    in the rows of no member and beyond a member's out_features; see `tp_ragged_linear_forward`."""
    device, code, offsets, inf, outf = _ragged_operands(x, weight, offsets, in_features, out_features)
    P, N, K = weight.shape
    R = x.shape[0]
    bias = _operand('bias', bias, (P, N), torch.float32, device)
    y = _empty2(R, N, x.dtype, x.device)
    if R:
        x, xs = _vector_rows('x', x, (R, K), device)
        w, ws = _ragged_weight(weight, device)
        a = _lib.RaggedLinearArgs(P, K, N, code, R, offsets.data_ptr(), _ptr(inf), _ptr(outf), int(relu), x.data_ptr(),
                                  xs, w.data_ptr(), ws, _ptr(bias), y.data_ptr())
        if code == TP_DTYPE_F32:
            a.workspace_bytes = need = _function('tp_ragged_linear_workspace_size')(ctypes.byref(a))
            scratch = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=x.device)
            a.workspace = scratch.data_ptr()
        _call('tp_ragged_linear_forward', a, device)
    return y


def ragged_linear_backward(dy: Tensor, x: Tensor, weight: Tensor, y: Tensor | None, offsets: Tensor, *,
                           in_features: Tensor | None = None, out_features: Tensor | None = None, relu: bool = False,
                           need_dx: bool = True, need_dw: bool = True, need_db: bool = True
                           ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """Backward of `ragged_linear_forward`: (dx (R, in) of x's type, dw (P, out, in), db (P, out) fp32);
    `y` is the forward's output, needed with relu.  See `tp_ragged_linear_backward`."""
    device, code, offsets, inf, outf = _ragged_operands(x, weight, offsets, in_features, out_features)
    P, N, K = weight.shape
    R = x.shape[0]
    dev, f32 = x.device, torch.float32
    dy, ds = _rows2('dy', dy, (R, N), x.dtype, device)
    if relu:
        if y is None:
            raise ValueError("the forward's output is needed with relu")
        y = _operand('y', y, (R, N), x.dtype, device)
    dx = _empty2(R, K, x.dtype, dev) if need_dx else None
    dw = torch.empty_strided((P, N, K), (N * K, K, 1), dtype=f32, device=dev) if need_dw else None
    db = _empty2(P, N, f32, dev) if need_db else None
    if not (need_dx or need_dw or need_db):
        return None, None, None
    if not R:
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_()
    x, xs = _vector_rows('x', x, (R, K), device)
    w, ws = _ragged_weight(weight, device)
    a = _lib.RaggedLinearArgs(P, K, N, code, R, offsets.data_ptr(), _ptr(inf), _ptr(outf), int(relu), x.data_ptr(), xs,
                              w.data_ptr(), ws, None, _ptr(y) if relu else None, dy.data_ptr(), ds, _ptr(dx), _ptr(dw),
                              _ptr(db))
    need = _function('tp_ragged_linear_workspace_size')(ctypes.byref(a))
    if need:
        scratch = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = scratch.data_ptr(), need
    _call('tp_ragged_linear_backward', a, device)
    return dx, dw, db


class Fp4Rows(NamedTuple):
    """Rows in 4-bit floating point, as `fp4_quantize` returns them and `fp4_linear_forward` takes a
    layer's weights; the layout is described at `tp_fp4_args`."""

    codes: Tensor  # (..., rows, 16 ceil(columns / 32)) uint8: two a byte
    scales: Tensor  # (..., row tiles, column tiles, 512) uint8: a byte per block of columns
    row_scale: Tensor  # (..., rows) fp32
    columns: int
    format: str  # 'nvfp4' or 'mxfp4'


def _fp4_format(format: str) -> int:
    code = _lib.TP_FP4.get(format)
    if code is None:
        raise ValueError(f"format must be 'nvfp4' or 'mxfp4', got {format!r}")
    return code


def _fp4_pitch(K: int) -> int:
    return (K + 31) // 32 * 16


def _fp4_scale_tiles(K: int, code: int) -> int:
    return (K + 255) // 256 * (4 if code == 0 else 2)


def fp4_quantize(x: Tensor, format: str = 'nvfp4', *, offsets: Tensor | None = None,
                 n_features: Tensor | None = None) -> Fp4Rows:
    """x (R, K) or (P, R, K), bf16 or fp32, in 4-bit floating point with a scale per block of columns;
    see `tp_fp4_quantize`.  `n_features` (P,): only the first columns of a member's rows count (the others
    are zero).  `offsets` (P + 1,): x is (R, K), member m's rows are x[offsets[m] : offsets[m + 1]] (those
    of no member stay unwritten), and the scales lie as `tp_fp4_linear_forward` takes rows in 4 bits over these groups
    (`fp4_linear_forward` quantises its rows itself, `fp4_values` takes rows without offsets)."""
    code = _fp4_format(format)
    if x.ndim not in (2, 3) or (offsets is not None and x.ndim != 2):
        raise ValueError('x must be (rows, columns) or (pack_size, rows, columns)')
    device = _device_of('x', x)
    dtype = _dtype_code(x.dtype)
    K = x.shape[-1]
    if not K:
        raise ValueError('x must have columns')
    lead = tuple(x.shape[:-1])
    rows = x.numel() // K
    if offsets is not None:
        if offsets.ndim != 1 or offsets.shape[0] < 2:
            raise ValueError('offsets must be (pack_size + 1,)')
        P = offsets.shape[0] - 1
        offsets = _members('offsets', offsets, P + 1, device)
        tiles = (rows // 128 + P,)
    else:
        P = x.shape[0] if x.ndim == 3 else 1
        tiles = (*lead[:-1], (lead[-1] + 127) // 128)
    n_features = _members('n_features', n_features, P, device)
    x, stride = _rows2('x', x if x.ndim == 2 else x.reshape(rows, K), (rows, K), x.dtype, device)
    u8, dev = torch.uint8, x.device
    codes = _empty((*lead, _fp4_pitch(K)), u8, dev)
    scales = _empty((*tiles, _fp4_scale_tiles(K, code), 512), u8, dev)
    row_scale = _empty(lead, torch.float32, dev)
    if rows:
        a = _lib.Fp4Args(P, K, code, dtype, rows, _ptr(offsets), _ptr(n_features), x.data_ptr(), stride,
                         codes.data_ptr(), scales.data_ptr(), row_scale.data_ptr())
        _call('tp_fp4_quantize', a, device)
    return Fp4Rows(codes, scales, row_scale, K, format)


def _fp4_checked(name: str, q: Fp4Rows, device: int, tiles: tuple) -> Fp4Rows:
    """Codes and scales of the shapes that their columns and format ask for, contiguous."""
    lead, code = tuple(q.row_scale.shape), _fp4_format(q.format)
    codes = _operand(f'{name}.codes', q.codes, (*lead, _fp4_pitch(q.columns)), torch.uint8, device)
    scales = _operand(f'{name}.scales', q.scales, (*tiles, _fp4_scale_tiles(q.columns, code), 512), torch.uint8, device)
    row_scale = _operand(f'{name}.row_scale', q.row_scale, lead, torch.float32, device)
    if codes.data_ptr() % 16 or scales.data_ptr() % 16:
        codes, scales = codes.clone(), scales.clone()
    return Fp4Rows(codes, scales, row_scale, q.columns, q.format)


def fp4_values(q: Fp4Rows) -> Tensor:
    """The values that `fp4_quantize`'s rows (without offsets) stand for, bf16 (which holds them exactly)."""
    device = _device_of('codes', q.codes)
    lead = tuple(q.row_scale.shape)
    if len(lead) not in (1, 2) or q.columns < 1:
        raise ValueError('the rows must be (rows, columns) or (pack_size, rows, columns)')
    q = _fp4_checked('q', q, device, (*lead[:-1], (lead[-1] + 127) // 128))
    out = _empty((*lead, q.columns), torch.bfloat16, q.codes.device)
    if out.numel():
        a = _lib.Fp4Args(lead[0] if len(lead) == 2 else 1, q.columns, _fp4_format(q.format), 0, q.row_scale.numel(), None,
                         None, None, 0, q.codes.data_ptr(), q.scales.data_ptr(), q.row_scale.data_ptr(), out.data_ptr())
        _call('tp_fp4_values', a, device)
    return out


def fp4_linear_forward(x: Tensor, weight: Fp4Rows, bias: Tensor | None = None, offsets: Tensor | None = None, *,
                       in_features: Tensor | None = None, out_features: Tensor | None = None,
                       relu: bool = False) -> Tensor:
    """Linear layer (+ReLU) of a pack with both operands in 4 bits; see `tp_fp4_linear_forward`.  `weight`:
    `fp4_quantize` of (P, out, in) (its columns beyond a member's in_features zero); x, bf16 or fp32, is
    quantised in the weight's format: (P, B, in) or (B, in) shared by the members, giving (P, B, out), or with
    `offsets` (P + 1,) ragged groups of rows (R, in), giving (R, out).  Bias (P, out) fp32 or None.  The
    result has x's type."""
    device = _device_of('x', x)
    dtype = _dtype_code(x.dtype)
    if weight.row_scale.ndim != 2:
        raise ValueError('weight must be (pack_size, out, in) in 4 bits')
    P, N = weight.row_scale.shape
    K = weight.columns
    if not P or not N or K < 1:
        raise ValueError('weight must not be empty')
    if weight.codes.get_device() != device:
        raise ValueError(f'weight must be on cuda:{device}, got {weight.codes.device}')
    weight = _fp4_checked('weight', weight, device, (P, (N + 127) // 128))
    if x.shape[-1] != K:
        raise ValueError(f'x must have {K} features, got {x.shape[-1]}')
    bias = _operand('bias', bias, (P, N), torch.float32, device)
    inf, outf = _members('in_features', in_features, P, device), _members('out_features', out_features, P, device)
    shared = offsets is None and x.ndim == 2
    if offsets is not None:
        offsets = _members('offsets', offsets, P + 1, device)
        if x.ndim != 2:
            raise ValueError('x must be (rows, features) with offsets')
    elif x.ndim == 3 and x.shape[0] != P:
        raise ValueError(f'x must have {P} members, got {x.shape[0]}')
    elif x.ndim not in (2, 3):
        raise ValueError('x must be (pack_size, batch, features) or a shared (batch, features)')
    if shared and inf is not None and P > 1:
        # members of different widths see different rows, and have scales of their own
        x, shared = x.expand(P, *x.shape), False
    lead = x.shape
    rows = lead[0] if len(lead) == 2 else lead[0] * lead[1]
    y = (_empty2(rows, N, x.dtype, x.device) if offsets is not None
         else _empty3(P, lead[-2], N, x.dtype, x.device))
    if not rows:
        return y
    x, stride = _rows2('x', x if len(lead) == 2 else x.reshape(rows, K), (rows, K), x.dtype, device)
    a = _lib.Fp4LinearArgs(P, K, N, _lib.TP_FP4[weight.format], dtype, int(shared), rows, _ptr(offsets), _ptr(inf),
                           _ptr(outf), None, None, None, weight.codes.data_ptr(), weight.scales.data_ptr(),
                           weight.row_scale.data_ptr(), _ptr(bias), int(relu), y.data_ptr(), x.data_ptr(), stride)
    a.workspace_bytes = need = _function('tp_fp4_linear_workspace_size')(ctypes.byref(a))
    scratch = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=x.device)
    a.workspace = scratch.data_ptr()
    _call('tp_fp4_linear_forward', a, device)
    return y


def device_error() -> int:
    """Read and clear the device-side error flag (0 or TP_ETIMEOUT)."""
    return load().tp_device_error()
