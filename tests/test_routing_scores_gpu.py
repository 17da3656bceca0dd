"""Routing by scores of any finite size: rows masked with the type's lowest number, large offsets, both ends at once."""

import pytest
import torch

from oracle import routed
from tabpack_b200 import nn as pnn
from tabpack_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]
# 4, 8, 16 and 32 lanes a row; 160 members take 32 lanes forward and 16 backward
MEMBERS = [(2, 2), (24, 2), (64, 8), (128, 16), (160, 3), (257, 6), (1024, 32)]
KINDS = 10


def scores(T, E, dtype, seed):
    """Row r of kind r % KINDS."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    z = 2.0 * torch.randn(T, E, generator=gen, device='cuda')
    some = torch.rand(T, E, generator=gen, device='cuda') < 0.5
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z[0::KINDS] = low
    z[1::KINDS] = 1e10
    z[2::KINDS] = -1e10
    z[3::KINDS] = 1e30
    z[4::KINDS] = torch.where(some, 4.3e9, 0.0)[4::KINDS]
    z[5::KINDS] = torch.where(some, z, low)[5::KINDS]
    z[6::KINDS] = torch.where(some, high, low)[6::KINDS]
    z[7::KINDS] += 1e6
    z[8::KINDS] = torch.where(some, -1e30, z)[8::KINDS]
    return z.to(dtype)


def tolerance(E):
    """exp(z - max) as 2^((z - max) log2(e)): difference and product are off by 2^-24 each and the constant by 2^-26, of at most
    105 (what is further down is below fp32's smallest number), ex2.approx by 2^-22; a weight has such a term above and their
    sum below, and the sum of E terms over 32 lanes and 5 exchanges rounds (E / 32 + 5) times by 2^-24."""
    return 2 * (2.0 ** -22 + 105 * (2.0 ** -23 + 2.0 ** -26)) + (E / 32 + 8) * 2.0 ** -24


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('E,k', MEMBERS)
@pytest.mark.parametrize('T,renormalize', [(3, True), (30, False), (3001, True), (3001, False)])
def test_weights_and_importance(T, E, k, renormalize, dtype):
    z = scores(T, E, dtype, T + E)
    weight, expert, position, offsets, importance = ops.route_forward(z, k, renormalize=renormalize)
    w, e, p, o, i = routed.route(z, k, renormalize)
    assert torch.equal(expert.long(), e) and torch.equal(position.long(), p) and torch.equal(offsets.long(), o)
    torch.testing.assert_close(weight.double(), w, rtol=tolerance(E), atol=1e-37)
    torch.testing.assert_close(importance.double(), i, rtol=tolerance(E) + (T / 64 + 64) * 2.0 ** -24, atol=1e-30)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('E,k', MEMBERS)
@pytest.mark.parametrize('renormalize', [True, False])
def test_gradient(E, k, renormalize, dtype):
    T = 301
    z = scores(T, E, dtype, E + k)
    gen = torch.Generator(device='cuda').manual_seed(1)
    gw, gi = torch.randn(T, k, generator=gen, device='cuda'), torch.randn(E, generator=gen, device='cuda')
    weight, expert, *_ = ops.route_forward(z, k, renormalize=renormalize)
    got = ops.route_backward(gw, gi, z, weight, expert, renormalize=renormalize)
    z64 = z.double().requires_grad_()
    w, _, _, _, importance = routed.route(z64, k, renormalize)
    want = torch.autograd.grad((w * gw.double()).sum() + (importance * gi.double()).sum(), z64)[0]
    # terms w (g - sum w g) and p (h - sum p h), each off by the weights' tolerance; then one rounding to the scores' type
    size = max(gw.abs().max().item(), gi.abs().max().item())
    torch.testing.assert_close(got.double(), want, rtol=torch.finfo(dtype).eps, atol=4 * size * (tolerance(E) + k * 2.0 ** -23))


@pytest.mark.parametrize('dtype', DTYPES)
def test_rows_masked_as_a_whole_leave_a_training_step_whole(dtype):
    z = torch.randn(40, 24, device='cuda').to(dtype)
    z[7] = torch.finfo(dtype).min
    z.requires_grad_()
    routing = pnn.route(z, 2)
    loss = routing.balance_loss() + (routing.weight ** 2).sum()
    loss.backward()
    assert torch.isfinite(loss) and torch.isfinite(z.grad).all()
    assert routing.expert[7].tolist() == [0, 1] and routing.weight[7].tolist() == [0.5, 0.5]
