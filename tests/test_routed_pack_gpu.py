"""A routed pack: routing, row moves and ragged layers together, in training and in 4 bits."""

import pytest
import torch

from oracle import routed
from tabpack_b200 import ops
from tabpack_b200.nn import Fp4LinearPack, RoutedMLPPack, fp4_, label_log_probs
from tabpack_b200.optim import AdamWPack, split_weight_decay

pytestmark = pytest.mark.gpu


def pack(seed=0, P=6, top_k=2, d_in=20, widths=(24, 64, 40, 17, 33, 64), d_out=7):
    torch.manual_seed(seed)
    return RoutedMLPPack(d_in, list(widths), d_out, top_k=top_k, max_d_block=64, pack_size=P).cuda()


def dense(model, x):
    """The same mixture in 64 bits over every member, with autograd's gradients."""
    p = {n: t.detach().double().requires_grad_() for n, t in model.named_parameters()}
    x = x.detach().double().requires_grad_()
    w, expert, _, offsets, importance = routed.route(x @ p['router'].T, model.top_k, model.renormalize)
    gate = torch.zeros(len(x), model.pack_size + 1, dtype=torch.float64, device=x.device)
    gate = gate.scatter(1, torch.where(expert < 0, model.pack_size, expert), w)[:, :-1]
    keep = torch.arange(64, device=x.device) < model.hidden.out_features[:, None]
    wh = torch.where(keep[..., None], p['hidden.weight'], 0.0)
    bh = torch.where(keep, p['hidden.bias'], 0.0)
    wo = torch.where(keep[:, None], p['output.weight'], 0.0)
    h = torch.relu(x @ wh.mT + bh[:, None])
    out = torch.einsum('bm,mbo->bo', gate, h @ wo.mT + p['output.bias'][:, None])
    counts = torch.diff(offsets).double()
    balance = model.pack_size * (counts / counts.sum() * importance).sum() / len(x)
    return out, balance, p, x


@pytest.mark.parametrize('B', [1, 50, 700])
@pytest.mark.parametrize('renormalize', [True, False])
def test_forward_and_gradients(B, renormalize):
    model = pack(seed=B)
    model.renormalize = renormalize
    x = torch.randn(B, 20, device='cuda', requires_grad=True)
    out, routing = model(x)
    want, balance, p, x64 = dense(model, x)
    torch.testing.assert_close(out.double(), want, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(routing.balance_loss().double(), balance, rtol=1e-5, atol=1e-6)
    c = torch.randn_like(out)
    ((out * c).sum() + routing.balance_loss()).backward()
    grads = torch.autograd.grad((want * c.double()).sum() + balance, [x64, *p.values()])
    for name, got, g in zip(['x', *p], [x.grad, *(t.grad for t in model.parameters())], grads):
        scale = g.abs().max().item() + 1e-3
        assert (got.double() - g).abs().max().item() < 2e-5 * scale * B ** 0.5, name


def test_under_autocast():
    model = pack(seed=1)
    x = torch.randn(300, 20, device='cuda')
    with torch.autocast('cuda', dtype=torch.bfloat16):
        out, _ = model(x)
    assert out.dtype == torch.bfloat16
    want, *_ = dense(model, x)
    # x, w, h and y are rounded to bf16 in each of two layers: a few 2^-8 of the sums' sizes
    assert ((out.double() - want).norm() / want.norm()).item() < 8 * 2.0 ** -8


def test_training_in_a_graph():
    """Routing, loss and optimizer as they are used together, recorded once and replayed."""
    model, loose = pack(seed=2), pack(seed=2)
    opts = []
    for m in (model, loose):
        decay, no_decay = split_weight_decay(m)
        opts.append(AdamWPack([{'params': decay}, {'params': no_decay, 'weight_decay': 0.0}], lr=1e-2,
                              weight_decay=1e-2, pack_size=6))
    x = torch.randn(256, 20, device='cuda')
    y = torch.randint(0, 7, (256,), device='cuda')

    def loss_of(m):
        out, routing = m(x)
        return -label_log_probs(out, y).log_prob.mean() + 0.01 * routing.balance_loss()

    losses = []
    for _ in range(3):
        loss = loss_of(loose)
        opts[1].zero_grad(set_to_none=True)
        loss.backward()
        opts[1].step()
        losses.append(loss.item())
    assert all(torch.isfinite(p).all() for p in loose.parameters())
    # the same gradients from a graph of forward and backward
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        grads = torch.autograd.grad(loss_of(model), list(model.parameters()))
        del grads
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = loss_of(model)
        grads = torch.autograd.grad(loss, list(model.parameters()))
    for step in range(3):
        graph.replay()
        assert abs(loss.item() - losses[step]) < 1e-5
        for p, g in zip(model.parameters(), grads):
            p.grad = g.clone()
        opts[0].step()


def test_members_are_replaced_selected_and_removed():
    model = pack(seed=3)
    before = model.hidden.weight.detach().clone()
    model.replace(pack_idx=torch.tensor([1, 4], device='cuda'), d_block=[8, 50])
    assert model.hidden.out_features.tolist() == [24, 8, 40, 17, 50, 64] == model.output.in_features.tolist()
    assert torch.equal(model.hidden.weight[0], before[0]) and not torch.equal(model.hidden.weight[1], before[1])
    x = torch.randn(40, 20, device='cuda')
    model.eval()
    with torch.no_grad(), model.temporarily_select(pack_idx=torch.tensor([0, 2, 5], device='cuda')):
        out, routing = model(x)
        assert routing.offsets.shape == (4,) and out.shape == (40, 7)
    model.remove(pack_idx=torch.tensor([3], device='cuda'))
    assert model.pack_size == 5 and model(x)[1].offsets.shape == (6,)


@pytest.mark.parametrize('format', ['nvfp4', 'mxfp4'])
@pytest.mark.parametrize('B', [1, 3, 600])
def test_served_in_4_bits(B, format):
    model = pack(seed=4).eval()
    x = torch.randn(B, 20, device='cuda')
    hidden, output = model.hidden, model.output
    with torch.no_grad():
        fp4_(model, format)
        assert isinstance(model.hidden, Fp4LinearPack)
        out, r = model(x)
        rows = ops.dispatch_rows(x, r.position, r.offsets)
        qh = ops.fp4_quantize(hidden.weight, format, n_features=hidden.in_features)
        qo = ops.fp4_quantize(output.weight, format, n_features=output.in_features)
        h = ops.fp4_linear_forward(rows, qh, hidden.bias, r.offsets, out_features=hidden.out_features, relu=True)
        y = ops.fp4_linear_forward(h, qo, output.bias, r.offsets, in_features=output.in_features)
        assert torch.equal(out, ops.combine_rows(y, r.weight, r.position, r.offsets))


def test_refusals():
    with pytest.raises(ValueError):
        RoutedMLPPack(4, 8, 2, top_k=3, pack_size=2)
    with pytest.raises(ValueError):
        RoutedMLPPack(4, 8, 2, top_k=0, pack_size=2)
    model = pack()
    with pytest.raises(ValueError):
        model(torch.zeros(3, 21, device='cuda'))
    with pytest.raises(RuntimeError):
        model(torch.zeros(3, 20))
