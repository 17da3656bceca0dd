"""AdamW with 8-bit moments on the GPU.

Codes and scales agree bit for bit with the fp32 restatement in `oracle/adamw8.py` (one rounding
per operation on both sides).  Parameters agree with the 64-bit definition: with u = 2^-24 the
decayed parameter is off by 3 u relative (1 - lr wd, the product, the final sum), the update by 64 u
relative (the moments' roundings, the bias corrections' exponential and logarithm at 2 ulp each,
the approximate reciprocal, division and root at 2 ulp).
"""

import numpy as np
import pytest
import torch

from oracle import adamw8 as o8

pytestmark = pytest.mark.gpu

U = 2.0**-24
KEYS = ('exp_avg', 'exp_avg_scale', 'exp_avg_sq', 'exp_avg_sq_scale')


@pytest.fixture(scope='module', autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')


def make(shapes, *, seed=0, fresh=False):
    """Parameters, gradients of widely spread sizes and states, as numpy arrays (P, inner)."""
    rng = np.random.default_rng(seed)
    out = []
    for shape in shapes:
        P, inner = shape[0], int(np.prod(shape[1:], dtype=np.int64))
        p = rng.standard_normal((P, inner)).astype(np.float32) * np.float32(0.1)
        size = np.exp(2.5 * rng.standard_normal((P, inner))) * 1e-3
        g = (rng.standard_normal((P, inner)) * size).astype(np.float32)
        r = rng.integers(0, 1 << 16, (2, P, inner))
        m = (0.3 * rng.standard_normal((P, inner)) * size * (not fresh)).astype(np.float32)
        v = (size * rng.uniform(0.5, 1.5, (P, inner)) * (not fresh)).astype(np.float32)
        mc, ms = o8.store_first(m, r[0])
        vc, vs = o8.store_root(v, r[1])
        out.append(dict(shape=shape, p=p, g=g, exp_avg=mc, exp_avg_scale=ms, exp_avg_sq=vc, exp_avg_sq_scale=vs))
    return out


def on_gpu(ts):
    p = [torch.from_numpy(t['p'].reshape(t['shape'])).cuda() for t in ts]
    g = [torch.from_numpy(t['g'].reshape(t['shape'])).cuda() for t in ts]
    st = [[torch.from_numpy(np.ascontiguousarray(t[k])).cuda().view(t['shape'] if k in ('exp_avg', 'exp_avg_sq')
                                                                    else t[k].shape) for t in ts] for k in KEYS]
    return p, g, st


def col(v):
    return v.reshape(-1, 1) if isinstance(v, np.ndarray) else v


def expect(t, i, hp, step, seed, member_base=0):
    """New (p64, update size, codes and scales) of tensor i."""
    P, inner = t['p'].shape
    b1, b2 = col(hp['beta1']), col(hp['beta2'])
    f32 = np.float32
    one = lambda b: f32(1) - b if isinstance(b, np.ndarray) else f32(1 - b)  # noqa: E731
    m0, u0 = o8.load_first(t['exp_avg'], t['exp_avg_scale']), o8.load_root(t['exp_avg_sq'], t['exp_avg_sq_scale'])
    as32 = lambda b: b if isinstance(b, np.ndarray) else f32(b)  # noqa: E731
    m, u = o8.moments32(m0, u0, t['g'], as32(b1), as32(b2), one(b1), one(b2))
    steps = step if isinstance(step, np.ndarray) else np.full(P, step)
    words = o8.bits(P, inner, tensor=i, step=steps, seed=seed, member_base=member_base)
    mc, ms = o8.store_first(m, words & 0xFFFF)
    vc, vs = o8.store_root(u, words >> 16)
    f64 = lambda v: col(v).astype(np.float64) if isinstance(v, np.ndarray) else v  # noqa: E731
    p64, size = o8.step64(t['p'], t['g'], m0, u0, lr=f64(hp['lr']), b1=f64(hp['beta1']), b2=f64(hp['beta2']),
                          eps=f64(hp['eps']), wd=f64(hp['weight_decay']), t=steps.reshape(-1, 1).astype(np.float64))
    return p64, size, dict(exp_avg=mc, exp_avg_scale=ms, exp_avg_sq=vc, exp_avg_sq_scale=vs)


def step_gpu(p, g, st, hp, step, seed, **kw):
    from tabpack_b200 import ops

    hp = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in hp.items()}
    when = dict(steps=[torch.from_numpy(step).cuda()] * len(p)) if isinstance(step, np.ndarray) else dict(step=step)
    ops.adamw8_step(p, g, *st, seed=seed, **when, **hp, **kw)


def check(ts, p, st, hp, step, seed, **kw):
    for i, t in enumerate(ts):
        p64, size, want = expect(t, i + kw.get('tensor_base', 0), hp, step, seed, kw.get('member_base', 0))
        for k, got in zip(KEYS, st):
            np.testing.assert_array_equal(got[i].cpu().numpy().reshape(want[k].shape), want[k], err_msg=f'{k} {i}')
        got = p[i].cpu().numpy().reshape(p64.shape)
        bound = U * (3 * np.abs(t['p']) + 64 * size) + 2.0**-126
        assert (np.abs(got - p64) <= bound).all(), (i, (np.abs(got - p64) - bound).max())


SCALAR = dict(lr=2e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)


def per_member(P, seed=0):
    rng = np.random.default_rng(seed)
    f = lambda lo, hi: rng.uniform(lo, hi, P).astype(np.float32)  # noqa: E731
    return dict(lr=f(1e-4, 5e-3), beta1=f(0.8, 0.97), beta2=f(0.95, 0.9999), eps=f(1e-9, 1e-6),
                weight_decay=f(0, 0.1))


SHAPES = [(1, 1), (1, 3), (2, 4), (3, 127), (3, 128), (3, 129), (2, 130), (4, 512), (2, 1000), (1, 5000), (3, 4099),
          (2, 37, 53), (5, 64, 32), (1, 300, 401), (70, 6)]


@pytest.mark.parametrize('fresh', [False, True])
@pytest.mark.parametrize('shape', SHAPES)
def test_one_tensor(shape, fresh):
    ts = make([shape], seed=sum(shape), fresh=fresh)
    p, g, st = on_gpu(ts)
    step_gpu(p, g, st, SCALAR, 1 if fresh else 7, 123)
    check(ts, p, st, SCALAR, 1 if fresh else 7, 123)


@pytest.mark.parametrize('which', [('lr',), ('beta1',), ('beta2',), ('eps', 'weight_decay'),
                                   ('lr', 'beta1', 'beta2', 'eps', 'weight_decay')])
@pytest.mark.parametrize('step', ['scalar', 'members'])
def test_member_hyperparameters(which, step):
    P = 5
    ts = make([(P, 33, 20), (P, 33), (P, 256)], seed=3)
    hp = {**SCALAR, **{k: v for k, v in per_member(P).items() if k in which}}
    when = np.array([1, 2, 50, 4000, 1 << 33]) if step == 'members' else 3
    p, g, st = on_gpu(ts)
    step_gpu(p, g, st, hp, when, 99)
    check(ts, p, st, hp, when, 99)


def test_many_tensors():
    """More than one launch's worth, with empty ones between."""
    ts = make([(2, 5 * i) for i in range(45)], seed=4)
    p, g, st = on_gpu(ts)
    step_gpu(p, g, st, SCALAR, 9, 5, tensor_base=7)
    check(ts, p, st, SCALAR, 9, 5, tensor_base=7)


def test_unaligned_storage():
    ts = make([(2, 256), (1, 512)], seed=5)
    p, g, st = on_gpu(ts)

    def shift(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device='cuda')[1:].view(t.shape)
        return flat.copy_(t)

    p, g = [shift(t) for t in p], [shift(t) for t in g]
    st = [[shift(t) for t in ts_] for ts_ in st]
    step_gpu(p, g, st, SCALAR, 9, 5)
    check(ts, p, st, SCALAR, 9, 5)


def test_several_steps():
    """Fifty steps: every step's states stay equal to the oracle's (parameters are checked from the
    kernel's own, so that roundings do not add up)."""
    ts = make([(3, 300), (3, 16, 9)], seed=6, fresh=True)
    p, g, st = on_gpu(ts)
    rng = np.random.default_rng(0)
    for step in range(1, 51):
        for t, gi in zip(ts, g):
            t['g'] = (rng.standard_normal(t['g'].shape) * 1e-2).astype(np.float32)
            gi.copy_(torch.from_numpy(t['g'].reshape(t['shape'])))
        step_gpu(p, g, st, SCALAR, step, 77)
        check(ts, p, st, SCALAR, step, 77)
        for i, t in enumerate(ts):
            t['p'] = p[i].cpu().numpy().reshape(t['p'].shape)
            for k, s in zip(KEYS, st):
                t[k] = s[i].cpu().numpy().reshape(t[k].shape)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_moments(dtype):
    from tabpack_b200 import ops

    ts = make([(2, 300), (1, 128), (3, 7, 11), (2, 512)] * 9, seed=7)
    _, _, st = on_gpu(ts)
    m, v = ops.adamw8_moments(*st, dtype=dtype)
    for i, t in enumerate(ts):
        first, root = o8.load_first(t['exp_avg'], t['exp_avg_scale']), o8.load_root(t['exp_avg_sq'], t['exp_avg_sq_scale'])
        for got, want in ((m[i], first), (v[i], root * root)):
            assert got.dtype == dtype and got.shape == t['shape']
            assert torch.equal(got.cpu(), torch.from_numpy(want.reshape(t['shape'])).to(dtype))


def test_every_code():
    """All 256 codes of both kinds read back as their formulas say (NaN for the two unused e4m3 codes)."""
    from tabpack_b200 import ops

    codes = torch.arange(256, dtype=torch.uint8, device='cuda').view(1, 256)
    scale = torch.tensor([[1.0, 0.5]], device='cuda')
    m, v = ops.adamw8_moments([codes], [scale], [codes], [scale])
    c = codes.cpu().numpy()
    used = (c & 127) != 127
    np.testing.assert_array_equal(m[0].cpu().numpy()[used], o8.load_first(c, scale.cpu().numpy())[used])
    np.testing.assert_array_equal(v[0].cpu().numpy(), o8.load_root(c, scale.cpu().numpy()) ** 2)


def test_rounding_is_unbiased():
    """Over 400 seeds the stored first moments average to the true ones: a code step of relative
    width 2^-3 rounds with a deviation of at most half a step, so the mean is within 5 deviations,
    5 x 2^-4 / sqrt(400) relative to the value's power of two (plus 2^-16 steps of bias)."""
    from tabpack_b200 import ops

    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.uniform(0.02, 1.0, (1, 128)).astype(np.float32)).cuda()
    x[0, 0] = 1.0
    total = [torch.zeros(1, 128, dtype=torch.float64, device='cuda') for _ in range(2)]
    for seed in range(400):
        p = torch.zeros(1, 128, device='cuda')
        st = [[t] for t in ops.adamw8_state(p)]
        ops.adamw8_step([p], [x], *st, step=1, lr=0.0, beta1=0.0, beta2=0.0, eps=1e-8, weight_decay=0.0, seed=seed)
        m, v = ops.adamw8_moments(*st)
        total[0] += m[0].double()
        total[1] += v[0].double().sqrt()
    power = 2.0 ** torch.floor(torch.log2(x.double()))
    for t, step in zip(total, (2.0**-3, 2.0**-4)):
        # the scale 1 / 448 (1 / 1.9375) is not a power of two: a code's binade reaches twice the value's
        assert ((t / 400 - x).abs() <= 2 * power * step * (2.5 / 20 + 2.0**-15)).all()


def test_small_blocks_and_nonfinite_gradients():
    """A block next to nothing is stored as zeros; one with an infinity or a NaN reads as NaN, and
    the parameters of its other elements take their ordinary step."""
    from tabpack_b200 import ops

    ts = make([(1, 512)], seed=8, fresh=True)
    g = ts[0]['g']
    g[0, :128] = 1e-35
    g[0, 128:256] = 0.0
    g[0, 300], g[0, 400] = np.nan, np.inf
    p, gt, st = on_gpu(ts)
    step_gpu(p, gt, st, SCALAR, 1, 11)
    m, v = ops.adamw8_moments(*st)
    assert (m[0][0, :256] == 0).all() and (v[0][0, :256] == 0).all()
    assert torch.isnan(m[0][0, 256:]).all() and torch.isnan(v[0][0, 256:]).all()
    fine = np.ones(512, bool)
    fine[[300, 400]] = False
    with np.errstate(invalid='ignore'):
        p64, size, _ = expect(ts[0], 0, SCALAR, 1, 11)
    # 1e-35^2 leaves the fp32 range: those elements' root is 0 in fp32, and their update m / eps
    fine[:128] = False
    got = p[0].cpu().numpy()[0]
    assert (np.abs(got - p64[0])[fine] <= (U * (3 * np.abs(ts[0]['p']) + 64 * size))[0][fine] + 2.0**-126).all()
    assert np.isfinite(got[:128]).all() and np.isnan(got[300])


def test_shards_and_launches_agree():
    """A member's result depends on neither its shard nor the launch it is in."""
    ts = make([(6, 200), (6, 11, 13)], seed=9)
    hp = per_member(6, seed=2)
    step = np.arange(5, 11)
    whole = on_gpu(ts)
    step_gpu(*whole, hp, step, 31, member_base=100)
    for lo, hi in ((0, 2), (2, 6)):
        part = [dict(shape=(hi - lo, *t['shape'][1:]), **{k: t[k][lo:hi] for k in ('p', 'g', *KEYS)}) for t in ts]
        got = on_gpu(part)
        sub = {k: v[lo:hi].copy() for k, v in hp.items()}
        step_gpu(*[[x] if not isinstance(x, list) else x for x in got], sub, step[lo:hi].copy(), 31,
                 member_base=100 + lo)
        for i in range(2):
            assert torch.equal(got[0][i], whole[0][i][lo:hi])
            for a, b in zip(got[2], whole[2]):
                assert torch.equal(a[i], b[i][lo:hi])


def test_other_stream_and_graph():
    ts = make([(2, 600), (2, 31)], seed=10)
    want = on_gpu(ts)
    step_gpu(*want, SCALAR, 4, 1)
    for side in ('stream', 'graph'):
        got = on_gpu(ts)
        if side == 'stream':
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step_gpu(*got, SCALAR, 4, 1)
            torch.cuda.current_stream().wait_stream(s)
        else:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step_gpu(*got, SCALAR, 4, 1)
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([*got[0], *sum(got[2], [])], [*want[0], *sum(want[2], [])]):
            assert torch.equal(a, b)


def test_a_state_given_twice_is_refused():
    """Two parameters on one state, or both moments in one tensor, would be updated by two threads."""
    from tabpack_b200 import ops

    p, g, st = on_gpu(make([(2, 300), (2, 300)], seed=12))
    before = [t.clone() for t in p]
    for j in range(4):
        bad = [list(t) for t in st]
        bad[j][1] = bad[j][0]
        with pytest.raises(ValueError, match='twice'):
            ops.adamw8_step(p, g, *bad, **SCALAR, seed=1, step=1)
    with pytest.raises(ValueError, match='twice'):
        ops.adamw8_step(p, g, st[0], st[1], st[0], st[3], **SCALAR, seed=1, step=1)
    assert all(torch.equal(a, b) for a, b in zip(p, before))


def test_refusals():
    from tabpack_b200 import ops

    ts = make([(2, 300)], seed=11)
    p, g, st = on_gpu(ts)
    before = p[0].clone()
    call = lambda *a, **kw: ops.adamw8_step(*a, **{**SCALAR, 'seed': 1, 'step': 1, **kw})  # noqa: E731
    with pytest.raises(ValueError):
        call(p, g, *st, step=0)
    with pytest.raises(ValueError):
        call(p, [], *st)
    with pytest.raises(ValueError):
        call(p * 2, g * 2, *(t * 2 for t in st))
    with pytest.raises(TypeError):
        call([p[0].double()], g, *st)
    with pytest.raises(TypeError):
        call([p[0].t()], g, *st)
    with pytest.raises(TypeError):
        call(p, [g[0].bfloat16()], *st)
    with pytest.raises(TypeError):
        call(p, [g[0][:, :200]], *st)
    for j in range(4):
        bad = list(st)
        bad[j] = [st[j][0][:1]]
        with pytest.raises(TypeError):
            call(p, g, *bad)
        bad[j] = [st[j][0].double()]
        with pytest.raises(TypeError):
            call(p, g, *bad)
    with pytest.raises(TypeError):
        call(p, g, *st, steps=[torch.ones(3, dtype=torch.int64, device='cuda')])
    with pytest.raises(TypeError):
        call(p, g, *st, steps=[torch.ones(2, dtype=torch.int32, device='cuda')])
    with pytest.raises(ValueError):
        call(p, g, *st, lr=torch.ones(3, device='cuda'))
    with pytest.raises(TypeError):
        call(p, g, *st, lr=torch.ones(2, device='cuda', dtype=torch.float64))
    with pytest.raises(ValueError):
        call(p, g, *st, lr=torch.ones(2))
    with pytest.raises(TypeError):
        ops.adamw8_moments(*st, dtype=torch.float16)
    assert torch.equal(p[0], before)


def test_square_root_is_correctly_rounded():
    """Every mantissa at an even and an odd exponent (the iteration is the same in every binade), and all
    numbers at both ends of the range, against CUDA's square root bit for bit."""
    from tabpack_b200 import _lib

    differ = torch.zeros(1, dtype=torch.int64, device='cuda')
    stream = torch.cuda.current_stream().cuda_stream
    binade = 1 << 23
    for exponent in (33, 34, 126, 127, 200, 252, 253):  # 2^-94, 2^-93, 1/2, 1, 2^73, 2^125, 2^126
        _lib.check(_lib.load().tp_root_check(exponent * binade, binade, differ.data_ptr(), stream), 'tp_root_check')
    assert differ.item() == 0


# ------------------------------------------------------------------ the optimizer packs


def _packs(P=3, seed=0):
    from tabpack_b200.nn import ParameterPack

    gen = torch.Generator(device='cuda').manual_seed(seed)
    return [ParameterPack(torch.randn(P, *s, generator=gen, device='cuda')) for s in ((40, 20), (40,), (2, 40), (2,))]


def _grads(params, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device='cuda') * 0.01


def test_optimizer_is_the_op():
    """`AdamWPack(state_bits=8)` over two groups, one parameter without a gradient."""
    from tabpack_b200 import ops
    from tabpack_b200.optim import AdamWPack

    params = _packs()
    opt = AdamWPack([{'params': params[:2], 'weight_decay': 0.0}, {'params': params[2:]}], lr=[1e-3, 2e-3, 3e-3],
                    weight_decay=0.01, pack_size=3, state_bits=8, state_seed=55)
    ref = [p.detach().clone() for p in params]
    st = [ops.adamw8_state(p) for p in ref]
    lr = torch.tensor([1e-3, 2e-3, 3e-3], device='cuda')
    for step in range(1, 4):
        _grads(params, step)
        params[2].grad = None
        opt.step()
        for i in (0, 1, 3):
            ops.adamw8_step([ref[i]], [params[i].grad], *([t] for t in st[i]), step=step, lr=lr, beta1=0.9,
                            beta2=0.999, eps=1e-8, weight_decay=0.01 if i > 1 else 0.0, seed=55, tensor_base=i)
    for i, p in enumerate(params):
        assert torch.equal(p.detach(), ref[i])
        if i != 2:
            assert set(opt.state[p]) == {'step', *KEYS}
            for k, t in zip(KEYS, st[i]):
                assert torch.equal(opt.state[p][k], t)
    m, v = opt.moments(params[0])
    assert m.shape == v.shape == params[0].shape and m.dtype == torch.float32 and (v >= 0).all()


def test_optimizer_checkpoint():
    """A saved and loaded optimizer continues bit for bit."""
    import copy

    from tabpack_b200.optim import AdamWPack

    kw = dict(lr=1e-3, weight_decay=0.01, pack_size=3, support_replacement=True)
    a = _packs()
    oa = AdamWPack(a, state_bits=8, **kw)
    for step in range(3):
        _grads(a, step)
        oa.step()
    saved = copy.deepcopy(oa.state_dict())
    b = _packs()
    for p, q in zip(b, a):
        p.data.copy_(q.data)
    ob = AdamWPack(b, state_bits=8, state_seed=1, **kw)
    ob.load_state_dict(saved)
    for step in range(3, 6):
        for params, opt in ((a, oa), (b, ob)):
            _grads(params, step)
            opt.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k in ('step', *KEYS):
            assert oa.state[p][k].dtype == ob.state[q][k].dtype and torch.equal(oa.state[p][k], ob.state[q][k])
    with pytest.raises(ValueError):
        AdamWPack(_packs(), **kw).load_state_dict(saved)
    full = AdamWPack(a, **kw)
    _grads(a, 9)
    full.step()
    with pytest.raises(ValueError):
        ob.load_state_dict(full.state_dict())


def test_optimizer_replace_and_remove():
    from tabpack_b200.optim import AdamWPack, optimizer_pack_remove

    params = _packs(4)
    opt = AdamWPack(params, lr=[1e-3] * 4, weight_decay=0.0, pack_size=4, state_bits=8, support_replacement=True)
    _grads(params, 1)
    opt.step()
    before = {k: opt.state[params[0]][k].clone() for k in ('step', *KEYS)}
    opt.replace(pack_idx=torch.tensor([1], device='cuda'), lr=[5e-3])
    keep = [0, 2, 3]
    for k, t in before.items():
        now = opt.state[params[0]][k]
        assert (now[1] == 0).all() and torch.equal(now[keep], t[keep])
    from tabpack_b200.nn import ParameterPack

    mapping = {p: ParameterPack(p.data[keep]) for p in params}
    optimizer_pack_remove(opt, pack_idx=torch.tensor([1], device='cuda'), old_to_new_parameters=mapping)
    new = opt.param_groups[0]['params']
    for k, t in before.items():
        assert torch.equal(opt.state[new[0]][k], t[keep])
    _grads(new, 2)
    opt.step()
    assert all(torch.isfinite(p).all() for p in new)


def test_muon_pack_with_8_bit_rest():
    from tabpack_b200.nn import LinearPack
    from tabpack_b200.optim import MuonAdamWPack

    lin = LinearPack([16, 32], [32, 24], max_in_features=32, max_out_features=32, pack_size=2).cuda()
    out = []
    for bits in (32, 8):
        torch.manual_seed(0)
        lin.reset_parameters()
        opt = MuonAdamWPack([MuonAdamWPack.make_muon_parameter_group(lin), {'params': [lin.bias]}], adamw_lr=1e-3,
                            muon_lr=1e-2, weight_decay=0.0, pack_size=2, allow_inplace_grad_mutation=False,
                            adamw_state_bits=bits)
        _grads(list(lin.parameters()), 3)
        opt.step()
        out.append([p.detach().clone() for p in lin.parameters()])
        assert ('exp_avg_scale' in opt.state[lin.bias]) == (bits == 8)
        assert set(opt.state[lin.weight]) == {'muon_momentum_buffer'}
    # the first step takes the same unrounded moments
    assert torch.equal(out[0][0], out[1][0])
    assert torch.allclose(out[0][1], out[1][1], rtol=0, atol=1e-3 * 64 * U + 3 * U)


def test_strided_member_hyperparameters(monkeypatch):
    """A column of a table of hyperparameters: its copy lives until the launch, whatever is allocated before."""
    from tabpack_b200 import ops

    P = 5
    ts = make([(P, 33, 20), (P, 256)], seed=13)
    hp = per_member(P, seed=4)
    call, taken = ops._call, []

    def busy(*args):
        taken.extend(torch.full((P,), float('nan'), device='cuda') for _ in range(64))
        call(*args)

    monkeypatch.setattr(ops, '_call', busy)
    p, g, st = on_gpu(ts)
    table = torch.stack([torch.from_numpy(v) for v in hp.values()], 1).cuda()
    ops.adamw8_step(p, g, *st, step=3, seed=17, **{k: table[:, i] for i, k in enumerate(hp)})
    check(ts, p, st, hp, 3, 17)
    assert len(taken) == 64


def test_square_root_check_of_all_numbers_ends():
    """The largest count: 2^32 - 1 patterns from 2^-94 on, past the end of the finite numbers and round again."""
    from tabpack_b200 import _lib

    differ = torch.zeros(1, dtype=torch.int64, device='cuda')
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.load().tp_root_check(33 << 23, 0xFFFFFFFF, differ.data_ptr(), stream), 'tp_root_check')
    assert differ.item() > 0  # zeros, subnormals and negative numbers are outside its range


@pytest.mark.parametrize('bits', [8, 32])
def test_checkpoint_through_a_file_read_to_the_host(bits, tmp_path):
    """Saved, read with map_location='cpu' and loaded: training continues bit for bit."""
    from tabpack_b200.optim import AdamWPack

    kw = dict(lr=1e-3, weight_decay=0.01, pack_size=3, support_replacement=True, state_bits=bits)
    a, b = _packs(), _packs()
    oa, ob = AdamWPack(a, **kw), AdamWPack(b, **kw)
    for step in range(3):
        _grads(a, step)
        oa.step()
    torch.save({'opt': oa.state_dict(), 'params': [p.data for p in a]}, tmp_path / 'checkpoint.pt')
    saved = torch.load(tmp_path / 'checkpoint.pt', map_location='cpu', weights_only=True)
    for p, t in zip(b, saved['params']):
        p.data.copy_(t)
    ob.load_state_dict(saved['opt'])
    for p in b:
        assert all(t.device == p.device for t in ob.state[p].values())
    for step in range(3, 6):
        for params, opt in ((a, oa), (b, ob)):
            _grads(params, step)
            opt.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k, t in oa.state[p].items():
            assert torch.equal(t, ob.state[q][k])


# A launch of 1184 tiles or more gives a warp a run of 16 blocks of a member (64 a tile), a smaller one 8,
# 4, 2 or 1; a member's last tile and last block are partial in all of these.
RUNS = [[(1184, 2100)], [(1184, 2101)], [(600, 8200)], [(600, 8197)], [(600, 4100)], [(600, 4103)], [(300, 8188)],
        [(300, 8191)], [(150, 8064)], [(150, 8063)], [(700, 2052), (500, 1023)], [(1, 1300000)]]


@pytest.mark.parametrize('shapes', RUNS, ids=str)
def test_runs_of_blocks(shapes):
    """Codes and scales bit for bit where a warp takes many blocks, with vectors and without, and the moments
    of the same states in both types.

    The parameters' bound at the head of this file counts roundings of the update itself.  Among millions of
    elements some have b1 m and (1 - b1) g that all but cancel: two products and the constant 1 - b1 are each
    off by u of these terms, not of their sum (rounded to fp32 with the rest in 64 bits, the first moment alone
    leaves that bound by 4e-13 at |p| = 7e-7).  So 3 u of what the two terms, added up, would move p by."""
    from tabpack_b200 import ops

    ts = make(shapes, seed=sum(map(sum, shapes)))
    ts[0]['g'][:, 130:400:7] = 0.0
    ts[0]['exp_avg'][0, :256] = ts[0]['exp_avg_sq'][0, :256] = 0
    p, g, st = on_gpu(ts)
    for dtype in (torch.float32, torch.bfloat16):
        m, v = ops.adamw8_moments(*st, dtype=dtype)
        for i, t in enumerate(ts):
            first = o8.load_first(t['exp_avg'], t['exp_avg_scale'])
            root = o8.load_root(t['exp_avg_sq'], t['exp_avg_sq_scale'])
            for got, want in ((m[i], first), (v[i], root * root)):
                assert torch.equal(got.cpu(), torch.from_numpy(want.reshape(t['shape'])).to(dtype))
    step_gpu(p, g, st, SCALAR, 5, 21, tensor_base=2)
    lr, b1, b2 = SCALAR['lr'], SCALAR['beta1'], SCALAR['beta2']
    for i, t in enumerate(ts):
        p64, size, want = expect(t, i + 2, SCALAR, 5, 21)
        for k, got in zip(KEYS, st):
            np.testing.assert_array_equal(got[i].cpu().numpy().reshape(want[k].shape), want[k], err_msg=f'{k} {i}')
        m0, u0 = o8.load_first(t['exp_avg'], t['exp_avg_scale']), o8.load_root(t['exp_avg_sq'], t['exp_avg_sq_scale'])
        m0, u0, g64 = (x.astype(np.float64) for x in (m0, u0, t['g']))
        root = np.sqrt((b2 * u0**2 + (1 - b2) * g64**2) / (1 - b2**5)) + SCALAR['eps']
        terms = lr / (1 - b1**5) * (np.abs(b1 * m0) + np.abs((1 - b1) * g64)) / root
        bound = U * (3 * np.abs(t['p']) + 64 * size + 3 * terms) + 2.0**-126
        assert (np.abs(p[i].cpu().numpy().reshape(p64.shape) - p64) <= bound).all()


@pytest.mark.parametrize('inner', [1_100_000_004, 1_100_000_003])
def test_elements_beyond_32_bits(inner):
    """The last blocks of two members of 1.1 billion elements, in a fresh state (22 GB)."""
    from oracle.philox import philox4x32_10
    from tabpack_b200 import ops

    p, g = (torch.zeros(2, inner, device='cuda') for _ in range(2))
    st = [[t] for t in ops.adamw8_state(p)]
    lo = (inner - 300) // 128 * 128
    gen = torch.Generator(device='cuda').manual_seed(inner % 7)
    g[:, lo:] = torch.randn(2, inner - lo, generator=gen, device='cuda') * 1e-2
    hp = {**SCALAR, 'weight_decay': 0.0}
    ops.adamw8_step([p], [g], *st, step=1, seed=41, member_base=5, tensor_base=3, **hp)
    n, tail = inner - lo, g[:, lo:].cpu().numpy()
    f32, zero = np.float32, np.zeros((2, inner - lo), np.float32)
    m, u = o8.moments32(zero, zero, tail, f32(0.9), f32(0.999), f32(1 - 0.9), f32(1 - 0.999))
    group = np.arange(lo // 4, (inner + 3) // 4, dtype=np.uint32)[None]
    member = np.array([[5], [6]], np.uint32)
    words = philox4x32_10(*np.broadcast_arrays(group, np.uint32(3), member, np.uint32(1)), np.uint32(41), np.uint32(0))
    words = np.stack(words, -1).reshape(2, -1)[:, :n]
    want = (*o8.store_first(m, words & 0xFFFF), *o8.store_root(u, words >> 16))
    for (t,), w in zip(st, want):
        np.testing.assert_array_equal(t[:, t.shape[1] - w.shape[1]:].cpu().numpy(), w)
    p64, size = o8.step64(zero, tail, zero, zero, lr=hp['lr'], b1=0.9, b2=0.999, eps=1e-8, wd=0.0, t=1.0)
    assert (np.abs(p[:, lo:].cpu().numpy() - p64) <= U * 64 * size).all()
    assert not p[:, 128:lo].any() and not st[0][0][:, :lo].any()
    first, root = ops.adamw8_moments(*st, dtype=torch.bfloat16)
    for got, (codes, scales), load, power in ((first[0], want[:2], o8.load_first, 1), (root[0], want[2:], o8.load_root, 2)):
        value = torch.from_numpy(load(codes, scales) ** power).bfloat16()
        assert torch.equal(got[:, lo:].cpu(), value)
    del p, g, st, first, root, got
    torch.cuda.empty_cache()
