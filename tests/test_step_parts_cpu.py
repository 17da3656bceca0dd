"""Host-side rules of the layer norm, the label log probabilities and AdamW with 8-bit moments: what
the C entry points and the Python wrappers refuse before anything runs, and optimizer states."""

import ctypes

import pytest
import torch

from tabpack_b200 import _lib, ops
from tabpack_b200.nn import LayerNormPack, ParameterPack, label_log_probs
from tabpack_b200.optim import AdamWPack, MuonAdamWPack

FAKE = 1 << 20  # a non-null, aligned address that no refused call touches


def refused(name, args, text=''):
    rc = getattr(_lib.load(), name)(None if args is None else ctypes.byref(args), None)
    assert rc in (-1, -2), rc
    assert text in _lib.load().tp_last_error_string().decode()


def norm_args(**kw):
    base = dict(P=2, B=3, W=8, dtype=1, dx_dtype=1, x_member_stride=24, x_row_stride=8, x=FAKE, y=FAKE, mean=FAKE,
                rstd=FAKE, dy=FAKE, dx=FAKE, eps=1e-5)
    return _lib.LayerNormArgs(**{**base, **kw})


@pytest.mark.parametrize('bad', [dict(P=0), dict(B=0), dict(W=-1), dict(dtype=2), dict(x=None), dict(mean=None),
                                 dict(rstd=None), dict(P=1 << 20, B=1 << 20), dict(B=(1 << 30) + 1, P=1),
                                 dict(W=(1 << 30) + 8)])
def test_layer_norm_refusals(bad):
    refused('tp_layer_norm_forward', norm_args(**bad))
    refused('tp_layer_norm_backward', norm_args(**bad))


def test_layer_norm_direction_refusals():
    refused('tp_layer_norm_forward', None)
    refused('tp_layer_norm_forward', norm_args(y=None), 'null layer norm output')
    refused('tp_layer_norm_backward', norm_args(dy=None), 'null layer norm gradient')
    refused('tp_layer_norm_backward', norm_args(dx_dtype=2), 'bad dx dtype')
    P, B, W = 1, 4096, 512
    need = _lib.load().tp_layer_norm_workspace_size(P, B, W)
    assert need > 0
    for ws in (dict(), dict(workspace=FAKE, workspace_bytes=need - 1), dict(workspace=FAKE + 1, workspace_bytes=need)):
        refused('tp_layer_norm_backward', norm_args(P=P, B=B, W=W, dweight=FAKE, **ws), 'workspace')


@pytest.mark.parametrize('bad', [dict(dx=None), dict(dx_dtype=1)])
def test_layer_norm_member_sums_need_terms_in_fp32(bad):
    refused('tp_layer_norm_backward', norm_args(dx_sum=FAKE, **{'dx_dtype': 0, **bad}), 'sum over the members')


def test_layer_norm_workspace_sizes():
    size = _lib.load().tp_layer_norm_workspace_size
    assert size(0, 4, 4) == size(4, 0, 4) == size(4, 4, -1) == 0
    assert size(4, 1, 64) == 0  # one row: nothing to split
    for P, B, W in ((1, 10**6, 8192), (512, 1024, 512), (3, 77, 20000), (100000, 2, 16)):
        splits = size(P, B, W) / (8 * P * W)
        assert splits == int(splits) and splits != 1 and splits <= max(1, B)


def labels_args(**kw):
    base = dict(rows=4, C=300, dtype=1, logits=FAKE, logits_stride=300, labels=FAKE, label_rows=4, log_prob=FAKE,
                entropy=FAKE, stats=FAKE, dlogits=FAKE)
    return _lib.LabelLogProbsArgs(**{**base, **kw})


@pytest.mark.parametrize('bad', [dict(rows=0), dict(rows=1 << 31), dict(C=0), dict(C=(1 << 30) + 1), dict(dtype=2),
                                 dict(logits=None), dict(labels=None), dict(stats=None), dict(label_rows=0),
                                 dict(label_rows=3), dict(logits_stride=299), dict(logits=FAKE + 1)])
def test_label_refusals(bad):
    refused('tp_label_log_probs_forward', labels_args(**bad))
    refused('tp_label_log_probs_backward', labels_args(**bad))


@pytest.mark.parametrize('bad', [dict(log_prob=None), dict(entropy=None), dict(top_k=-1), dict(top_k=33),
                                 dict(top_k=3), dict(top_k=6, C=5, top_log_prob=FAKE, top_label=FAKE)])
def test_label_forward_refusals(bad):
    refused('tp_label_log_probs_forward', labels_args(**bad))


@pytest.mark.parametrize('bad', [dict(dlogits=None), dict(dlogits=FAKE + 1), dict(g_log_prob_stride=2),
                                 dict(g_entropy_stride=-1)])
def test_label_backward_refusals(bad):
    refused('tp_label_log_probs_backward', labels_args(**bad))


def adamw_args(n=1, tensor=None, **kw):
    a = _lib.AdamW8Args(n_tensors=n, step=1, **kw)
    t = dict(p=FAKE, grad=FAKE, exp_avg=FAKE, exp_avg_scale=FAKE, exp_avg_sq=FAKE, exp_avg_sq_scale=FAKE, numel=256,
             inner=128)
    a.t[0] = _lib.Opt8Tensor(**{**t, **(tensor or {})})
    return a


def moments_args(**kw):
    a = _lib.AdamW8MomentsArgs(n_tensors=1, dtype=1)
    t = dict(exp_avg=FAKE, exp_avg_scale=FAKE, exp_avg_sq=FAKE, exp_avg_sq_scale=FAKE, m=FAKE, v=FAKE, numel=256,
             inner=128)
    a.t[0] = _lib.Opt8Values(**{**t, **kw})
    return a


@pytest.mark.parametrize('bad', [dict(p=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_scale=None),
                                 dict(exp_avg_sq=None), dict(exp_avg_sq_scale=None), dict(numel=0), dict(inner=0),
                                 dict(numel=200), dict(inner=(1 << 33) + 1, numel=(1 << 33) + 1), dict(p=FAKE + 2),
                                 dict(exp_avg_scale=FAKE + 1), dict(numel=1 << 62, inner=1)])
def test_adamw8_refusals(bad):
    refused('tp_adamw8_step', adamw_args(tensor=bad))


def test_adamw8_argument_refusals():
    refused('tp_adamw8_step', None)
    refused('tp_adamw8_step', adamw_args(n=0))
    refused('tp_adamw8_step', adamw_args(n=33))
    a = adamw_args()
    a.step = 0
    refused('tp_adamw8_step', a, 'step count')
    m = _lib.AdamW8MomentsArgs(n_tensors=1, dtype=2)
    refused('tp_adamw8_moments', m, 'dtype')
    refused('tp_adamw8_moments', _lib.AdamW8MomentsArgs(n_tensors=1, dtype=0), 'null')


@pytest.mark.parametrize('call,args', [
    ('tp_layer_norm_forward', lambda: norm_args(x=FAKE + 1)), ('tp_layer_norm_forward', lambda: norm_args(y=FAKE + 1)),
    ('tp_layer_norm_forward', lambda: norm_args(weight=FAKE + 2)),
    ('tp_layer_norm_backward', lambda: norm_args(dx_dtype=0, dx=FAKE + 2)),
    ('tp_layer_norm_backward', lambda: norm_args(dtype=0, dx_dtype=0, dx_sum=FAKE + 2)),
    ('tp_layer_norm_backward', lambda: norm_args(rstd=FAKE + 2)),
    ('tp_label_log_probs_forward', lambda: labels_args(labels=FAKE + 4)),
    ('tp_label_log_probs_forward', lambda: labels_args(top_k=1, top_log_prob=FAKE, top_label=FAKE + 4)),
    ('tp_label_log_probs_forward', lambda: labels_args(log_prob=FAKE + 2)),
    ('tp_label_log_probs_backward', lambda: labels_args(g_entropy=FAKE + 2)),
    ('tp_adamw8_step', lambda: adamw_args(tensor=dict(step=FAKE + 4))),
    ('tp_adamw8_moments', lambda: moments_args(m=FAKE + 1)),
    ('tp_adamw8_moments', lambda: moments_args(exp_avg_sq_scale=FAKE + 2))])
def test_misaligned_data_is_refused(call, args):
    refused(call, args(), 'aligned')


def test_cpu_tensors_are_refused():
    x, w = torch.randn(2, 3, 8), torch.ones(2, 8)
    with pytest.raises(RuntimeError):
        ops.layer_norm_forward(x, w, w)
    with pytest.raises(RuntimeError):
        LayerNormPack(8, pack_size=2)(x)
    with pytest.raises(RuntimeError):
        label_log_probs(x, torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        ops.adamw8_step([w], [w], *([t] for t in ops.adamw8_state(w)), step=1, lr=1.0, beta1=0.9, beta2=0.9, eps=1e-8,
                        weight_decay=0.0, seed=0)


def test_layer_norm_pack_arguments():
    for bad in (dict(pack_size=0), dict(eps=0.0), dict(eps=float('inf')), dict(n_features=0), dict(n_features=[4, 9]),
                dict(n_features=[4]), dict(n_features=[4, 0])):
        with pytest.raises(ValueError):
            LayerNormPack(**{**dict(n_features=8, max_n_features=8, pack_size=2), **bad})
    pack = LayerNormPack([3, 5], pack_size=2)
    assert pack.weight.shape == (2, 5) and set(pack.state_dict()) == {'weight', 'bias', 'n_features'}
    with pytest.raises(ValueError):
        pack.replace(pack_idx=torch.tensor([0]), n_features=[6])
    with pytest.raises(RuntimeError):
        LayerNormPack(4, pack_size=2).replace(pack_idx=torch.tensor([0]), n_features=[3])
    other = LayerNormPack([5, 2], pack_size=2)
    with torch.no_grad():
        other.weight.fill_(7.0)
    pack.load_state_dict_at(other.state_dict(), pack_idx=torch.tensor([1]), state_dict_idx=torch.tensor([0]))
    assert pack.n_features.tolist() == [3, 5] and (pack.weight[1] == 7).all() and (pack.weight[0] == 1).all()
    plain = LayerNormPack(4, elementwise_affine=False, pack_size=2)
    assert plain.try_get_pack_size() is None and list(plain.parameters()) == []


def _opt(cls=AdamWPack, **kw):
    p = ParameterPack(torch.zeros(2, 200))
    base = dict(lr=1e-3, weight_decay=0.0) if cls is AdamWPack else dict(
        adamw_lr=1e-3, muon_lr=1e-2, weight_decay=0.0, allow_inplace_grad_mutation=False)
    return p, cls([p], pack_size=2, **{**base, **kw})


def test_state_bits_are_checked():
    with pytest.raises(ValueError):
        _opt(state_bits=16)
    with pytest.raises(ValueError):
        _opt(MuonAdamWPack, adamw_state_bits=4)


def test_32_bit_optimizers_draw_no_seed():
    """Without 8-bit states nothing is taken from torch's generator and no key is added."""
    torch.manual_seed(0)
    want = torch.rand(1)
    torch.manual_seed(0)
    _, opt = _opt()
    assert torch.equal(torch.rand(1), want)
    assert set(opt.state_dict()) == {'state', 'param_groups'}


def test_state_round_trip():
    """torch casts the states of fp32 parameters to fp32 on loading: codes come back as uint8."""
    p, opt = _opt(state_bits=8, state_seed=12, support_replacement=True)
    m, ms, v, vs = ops.adamw8_state(p.data)
    m.copy_(torch.arange(400).view(2, 200) % 256)
    v.copy_(255 - m)
    ms.fill_(0.25)
    opt.state[p] = {'step': torch.tensor([3, 5]), 'exp_avg': m, 'exp_avg_scale': ms, 'exp_avg_sq': v,
                    'exp_avg_sq_scale': vs}
    q, other = _opt(state_bits=8, support_replacement=True)
    other.load_state_dict(opt.state_dict())
    assert other.state_seed == 12
    for k, t in opt.state[p].items():
        assert other.state[q][k].dtype == t.dtype and torch.equal(other.state[q][k], t)
    with pytest.raises(ValueError):
        _opt()[1].load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        opt.moments(ParameterPack(torch.zeros(2, 3)))


def test_zero_state():
    m, ms, v, vs = ops.adamw8_state(torch.zeros(3, 5, 60))
    assert m.shape == v.shape == (3, 5, 60) and ms.shape == vs.shape == (3, 3)
    assert m.dtype == v.dtype == torch.uint8 and ms.dtype == vs.dtype == torch.float32
    assert all((t == 0).all() for t in (m, ms, v, vs))


def test_oracle_codes_round_to_neighbours():
    """Every stored value is one of its two neighbours in the code's grid, and the grid's own values
    are kept whatever the random bits."""
    import numpy as np

    from oracle import adamw8 as o8

    rng = np.random.default_rng(0)
    x = (rng.standard_normal((3, 300)) * np.exp(2 * rng.standard_normal((3, 300)))).astype(np.float32)
    for store, load, sign in ((o8.store_first, o8.load_first, True), (o8.store_root, o8.load_root, False)):
        y = x if sign else np.abs(x)
        lo, hi = (load(*store(y, np.full(y.shape, r))) for r in (0, 65535))
        scale = np.repeat(store(y, np.zeros(y.shape, int))[1], 128, 1)[:, :300]
        slack = 4 * 2.0**-24 * np.abs(y)
        small = np.abs(y) < scale * 2.0**-14
        assert ((np.abs(lo) <= np.abs(y) + slack) | small).all() and ((np.abs(hi) >= np.abs(y) - slack) | small).all()
        codes, s = store(y, rng.integers(0, 65536, y.shape))
        again, s2 = store(load(codes, s), rng.integers(0, 65536, y.shape))
        kept = np.abs(load(again, s2) - load(codes, s)) <= 4 * 2.0**-24 * np.abs(load(codes, s))
        assert kept.mean() >= 0.99  # a value an ulp below its code is rounded down by 1 in 2^16


def test_layer_norm_takes_no_weight_decay():
    from tabpack_b200.nn import LinearPack
    from tabpack_b200.optim import split_weight_decay

    model = torch.nn.Sequential(LinearPack(4, 8, pack_size=2), LayerNormPack(8, pack_size=2),
                                LayerNormPack(8, bias=False, pack_size=2), LinearPack(8, 3, pack_size=2))
    decay, no_decay = split_weight_decay(model)
    assert [id(p) for p in decay] == [id(model[0].weight), id(model[3].weight)]
    assert len(no_decay) == len(list(model.parameters())) - 2


@pytest.mark.parametrize('cls,kw', [(AdamWPack, {}), (AdamWPack, dict(state_bits=8)), (MuonAdamWPack, {}),
                                    (MuonAdamWPack, dict(adamw_state_bits=8))])
def test_loaded_step_counts_go_to_their_parameter(cls, kw):
    """A checkpoint read to the host: torch moves the moments, and leaves what is called 'step'."""
    p, opt = _opt(cls, support_replacement=True, **kw)
    state = {'step': torch.tensor([3, 5]), 'exp_avg': torch.ones(2, 200), 'exp_avg_sq': torch.ones(2, 200)}
    if kw:
        state = dict(zip(('exp_avg', 'exp_avg_scale', 'exp_avg_sq', 'exp_avg_sq_scale'), ops.adamw8_state(p.data)),
                     step=state['step'])
    opt.state[p] = state
    q = ParameterPack(torch.zeros(2, 200, device='meta'))
    base = dict(lr=1e-3, weight_decay=0.0) if cls is AdamWPack else dict(
        adamw_lr=1e-3, muon_lr=1e-2, weight_decay=0.0, allow_inplace_grad_mutation=False)
    other = cls([q], pack_size=2, support_replacement=True, **base, **kw)
    other.load_state_dict(opt.state_dict())
    assert set(other.state[q]) == set(state)
    for k, t in other.state[q].items():
        assert t.device.type == 'meta' and t.dtype == state[k].dtype, k


def test_loaded_8_bit_states_are_copies_as_a_whole():
    """Codes without their scales are worth nothing: what another optimizer goes on to do to the loaded tensors
    changes neither."""
    p, opt = _opt(state_bits=8, support_replacement=True)
    names = ('exp_avg', 'exp_avg_scale', 'exp_avg_sq', 'exp_avg_sq_scale')
    opt.state[p] = {**dict(zip(names, ops.adamw8_state(p.data))), 'step': torch.tensor([3, 5])}
    q, other = _opt(state_bits=8, support_replacement=True)
    other.load_state_dict(opt.state_dict())
    before = {k: t.clone() for k, t in other.state[q].items()}
    for t in opt.state[p].values():
        t.add_(1)
    assert all(torch.equal(t, before[k]) for k, t in other.state[q].items())


def test_moments_of_an_unknown_parameter_leave_the_optimizer_alone():
    p, opt = _opt(state_bits=8)
    for stranger in (p, ParameterPack(torch.zeros(2, 3))):
        with pytest.raises(ValueError):
            opt.moments(stranger)
    assert len(opt.state) == 0 and opt.state_dict()['state'] == {}


@pytest.mark.parametrize('name', ['lr', 'beta1', 'beta2', 'eps', 'weight_decay'])
def test_misaligned_hyperparameters_are_refused(name):
    a = adamw_args()
    getattr(a, name).per_member = FAKE + 2
    refused('tp_adamw8_step', a, 'aligned')
