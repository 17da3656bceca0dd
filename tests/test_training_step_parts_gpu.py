"""The layer norm, the label log probabilities and AdamW with 8-bit moments together, as a training
step uses them: linear -> layer norm -> ReLU -> linear -> loss with an entropy bonus -> step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.fixture(scope='module', autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')


WIDTHS = [24, 40, 33]
CLASSES = 5


def build():
    from tabpack_b200 import nn as tnn

    torch.manual_seed(0)
    a = tnn.LinearPack(12, WIDTHS, max_out_features=40, pack_size=3).cuda()
    norm = tnn.LayerNormPack(WIDTHS, max_n_features=40, pack_size=3).cuda()
    head = tnn.LinearPack(WIDTHS, CLASSES, max_in_features=40, pack_size=3).cuda()
    return a, norm, head


def forward(parts, x, y, weight):
    from tabpack_b200 import nn as tnn

    a, norm, head = parts
    out = tnn.label_log_probs(head(torch.relu(norm(a(x)))), y)
    return -(out.log_prob + weight * out.entropy).mean(1)


def plain(parts, x, y, weight):
    """The same step in 64 bits, member by member, with autograd: (losses, gradients)."""
    a, norm, head = parts
    losses, grads = [], {p: torch.zeros_like(p, dtype=torch.float64) for m in parts for p in m.parameters()}
    for m, n in enumerate(WIDTHS):
        cut = [(a.weight, (slice(n), slice(None))), (a.bias, (slice(n),)), (norm.weight, (slice(n),)),
               (norm.bias, (slice(n),)), (head.weight, (slice(None), slice(n))), (head.bias, (slice(None),))]
        aw, ab, nw, nb, hw, hb = leaves = [p.detach()[(m, *at)].double().requires_grad_() for p, at in cut]
        h = x[m].double() @ aw.T + ab
        mean, var = h.mean(1, keepdim=True), h.var(1, keepdim=True, correction=0)
        h = torch.relu((h - mean) / torch.sqrt(var + norm.eps) * nw + nb)
        lp = torch.log_softmax(h @ hw.T + hb, 1)
        loss = -(lp.gather(1, y[m][:, None])[:, 0] - weight * (lp.exp() * lp).sum(1)).mean()
        loss.backward()
        losses.append(loss.detach())
        for (p, at), leaf in zip(cut, leaves):
            grads[p][(m, *at)] = leaf.grad
    return torch.stack(losses), grads


def batch(seed=1, B=64):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(3, B, 12, generator=gen, device='cuda')
    return x, torch.randint(0, CLASSES, (3, B), generator=gen, device='cuda')


def test_loss_and_gradients():
    """Each layer adds relative errors of at most its longest chain (12, 40 + 16, 40, 64 rows, 5
    classes) times u to values that the normalisation keeps near 1; together below 400 u of the
    largest value of each gradient (1 / sqrt(var) is below 4 on this batch)."""
    parts = build()
    x, y = batch()
    losses = forward(parts, x, y, 0.1)
    losses.sum().backward()
    want, grads = plain(parts, x, y, 0.1)
    assert ((losses.double() - want).abs() <= 400 * U * (1 + want.abs())).all()
    for p, g in grads.items():
        assert ((p.grad.double() - g).abs() <= 4 * 400 * U * g.abs().max()).all()


def test_steps_with_8_bit_moments():
    """Six steps: every parameter moves as the optimizer op moves it from the same gradients, the
    padding beyond each member's width stays as it was initialised."""
    from tabpack_b200 import ops
    from tabpack_b200.optim import AdamWPack

    parts = build()
    params = [p for m in parts for p in m.parameters()]
    opt = AdamWPack(params, lr=[1e-3, 3e-3, 1e-2], weight_decay=0.0, pack_size=3, state_bits=8, state_seed=9)
    ref = [p.detach().clone() for p in params]
    start = [p.clone() for p in ref]
    states = [ops.adamw8_state(p) for p in ref]
    lr = torch.tensor([1e-3, 3e-3, 1e-2], device='cuda')
    for step in range(1, 7):
        x, y = batch(step)
        opt.zero_grad()
        forward(parts, x, y, 0.05).sum().backward()
        for p, r in zip(params, ref):
            assert torch.equal(p.detach(), r)
        ops.adamw8_step(ref, [p.grad for p in params], *(list(t) for t in zip(*states)), step=step, lr=lr, beta1=0.9,
                        beta2=0.999, eps=1e-8, weight_decay=0.0, seed=9)
        opt.step()
    for p, r, s in zip(params, ref, start):
        assert torch.equal(p.detach(), r) and torch.isfinite(r).all() and not torch.equal(r, s)
    a, norm, head = parts
    for m, n in enumerate(WIDTHS):
        assert torch.equal(a.weight[m, n:], start[0][m, n:]) and torch.equal(norm.weight[m, n:], start[2][m, n:])
        assert torch.equal(head.weight[m, :, n:], start[4][m, :, n:])


def test_captured_step():
    """Forward, backward and step in one graph: replays equal the eager steps bit for bit."""
    from tabpack_b200 import nn as tnn
    from tabpack_b200 import ops

    a, norm, head = build()
    x, y = batch()
    h = a(x).detach()
    w = norm.weight.detach().clone()
    state = [[t] for t in ops.adamw8_state(w)]
    step = torch.zeros(3, dtype=torch.int64, device='cuda')
    hp = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, seed=4)
    n = norm.n_features.to(torch.int32)

    def run():
        out, mean, rstd = ops.layer_norm_forward(h, w, None, n_features=n)
        lp, H, _, _, stats = ops.label_log_probs_forward(out, y)
        g = torch.full_like(lp, -1.0 / lp.numel())
        dz = ops.label_log_probs_backward(g, None, out, y, stats)
        _, dw, _ = ops.layer_norm_backward(dz, h, w, mean, rstd, n_features=n, need_dx=False, need_db=False)
        step.add_(1)
        ops.adamw8_step([w], [dw], *state, steps=[step], **hp)

    def reset():
        w.copy_(norm.weight.detach())
        step.zero_()
        for (t,) in state:
            t.zero_()

    for _ in range(4):
        run()
    want = [w.clone(), *(t[0].clone() for t in state)]
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    reset()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    for t, u in zip([w, *(t[0] for t in state)], want):
        assert torch.equal(t, u)
    del tnn


def test_two_streams_at_once():
    """The same calls on two streams with their own tensors, nothing shared between them."""
    from tabpack_b200 import ops

    def work(seed):
        gen = torch.Generator(device='cuda').manual_seed(seed)
        x = torch.randn(4, 600, 256, generator=gen, device='cuda')
        y = torch.randint(0, 256, (4, 600), generator=gen, device='cuda')
        w = torch.ones(4, 256, device='cuda')
        state = [[t] for t in ops.adamw8_state(w)]
        torch.cuda.synchronize()

        def run():
            for s in range(1, 6):
                out, mean, rstd = ops.layer_norm_forward(x, w, None)
                lp, H, top, which, stats = ops.label_log_probs_forward(out, y, top_k=3)
                dz = ops.label_log_probs_backward(torch.ones_like(lp), H, out, y, stats)
                _, dw, _ = ops.layer_norm_backward(dz, x, w, mean, rstd, need_dx=False, need_db=False)
                ops.adamw8_step([w], [dw], *state, step=s, lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0,
                                seed=seed)
            return [w, top, which]

        return run

    want = [[t.clone() for t in work(s)()] for s in (1, 2)]
    runs = [work(s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in runs]
    got = []
    for run, s in zip(runs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for g, t in zip(got, want):
        for a, b in zip(g, t):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ the trainer


def _trainer(**kw):
    from tabpack_b200.training import PackTrainer

    P = kw.pop('P', 4)
    optimizer = kw.pop('optimizer', {'type': 'adamw', 'lr': 2e-3, 'weight_decay': 0.01, 'state_bits': 8})
    return PackTrainer(n_members=P, model=dict(n_numerical_features=10, categorical_cardinalities=[], d_out=4,
                                               max_d_block=48),
                       per_member_model=[dict(n_blocks=1 + m % 2, d_block=16 + 16 * (m % 3), dropout=0.1)
                                         for m in range(P)],
                       optimizer=optimizer, loss='ce', seed=3, device='cuda', **kw)


def _data(n=300):
    gen = torch.Generator(device='cuda').manual_seed(5)
    return {'x_num': torch.randn(n, 10, generator=gen, device='cuda'),
            'y': torch.randint(0, 4, (n,), generator=gen, device='cuda')}


@pytest.mark.parametrize('optimizer', [
    {'type': 'adamw', 'lr': 2e-3, 'weight_decay': 0.01, 'state_bits': 8},
    {'type': 'muon', 'adamw_lr': 2e-3, 'muon_lr': 1e-2, 'weight_decay': 0.01, 'adamw_state_bits': 8}])
def test_trainer_with_8_bit_moments_and_entropy(optimizer):
    t = _trainer(optimizer=optimizer, entropy_weight=0.05)
    before = [p.detach().clone() for p in t.model.parameters()]
    loss = t.fit_epoch(_data(), batch_size=64, epoch=0)
    assert loss.shape == (4,) and torch.isfinite(loss).all()
    assert any(not torch.equal(p, b) for p, b in zip(t.model.parameters(), before))
    assert all(torch.isfinite(p).all() for p in t.model.parameters())
    assert any('exp_avg_scale' in st for st in t.opt.state.values())


def test_trainer_is_reproducible_over_shards():
    """A shard of two members trains them as the whole pack does (8-bit states included)."""
    data = _data()
    whole = _trainer()
    whole.fit_epoch(data, batch_size=64, epoch=0)
    part = _trainer(member_range=(2, 4))
    part.fit_epoch(data, batch_size=64, epoch=0)
    for p, q in zip(whole.model.parameters(), part.model.parameters()):
        assert torch.equal(p[2:4], q)


def test_member_loss_with_entropy():
    from tabpack_b200.training import member_loss

    gen = torch.Generator(device='cuda').manual_seed(6)
    z = torch.randn(2, 30, 4, generator=gen, device='cuda', requires_grad=True)
    y = torch.randint(0, 4, (2, 30), generator=gen, device='cuda')
    loss = member_loss('ce', z, y, entropy_weight=0.3)
    lp = torch.log_softmax(z.detach().double(), -1)
    want = -(lp.gather(-1, y[..., None])[..., 0] - 0.3 * (lp.exp() * lp).sum(-1)).mean(1)
    # 30 additions and the logarithms: below 128 u
    assert ((loss.double() - want).abs() <= 128 * U * (1 + want.abs())).all()
    with pytest.raises(ValueError):
        member_loss('mse', z, y, entropy_weight=0.3)
    with pytest.raises(ValueError):
        _trainer(entropy_weight=float('nan'))
