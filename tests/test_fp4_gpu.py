"""Rows in 4-bit floating point and products of them, against 64 bits."""

import math

import pytest
import torch

from oracle import routed
from tabpack_b200 import ops
from tabpack_b200.nn import Fp4LinearPack, LinearPack, MLPBackbonePack, TabPack, fp4_
from tabpack_b200.training import PackPredictor, PackTrainer

pytestmark = pytest.mark.gpu

FORMATS = ['nvfp4', 'mxfp4']
DTYPES = [torch.bfloat16, torch.float32]
U24 = 2.0 ** -24


def rows(R, K, dtype, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(R, K, generator=gen, device='cuda') * torch.exp(2 * torch.randn(R, 1, generator=gen, device='cuda'))
    return (x * torch.exp(torch.randn(K, generator=gen, device='cuda'))).to(dtype)


def same(got, want):
    """bf16 holds a value's six significant bits: equal, NaN in the same places.  (Of a row whose largest is next to fp32's
    own, 2^128 (1 - 2^-24), the scale rounds 341 up to 352, and 6 * 352 * 2^117 = 1.03 * 2^128 is infinite in bf16.)"""
    assert torch.equal(got.isnan(), want.isnan())
    want = want.nan_to_num(posinf=math.inf, neginf=-math.inf)
    rounded = want.to(got.dtype)
    assert torch.equal(got.nan_to_num(posinf=math.inf, neginf=-math.inf), rounded)
    assert ((rounded.double() == want) | (want.abs() > 2.0 ** 128)).all()


@pytest.mark.parametrize('format', FORMATS)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('R,K', [(1, 1), (1, 16), (3, 33), (5, 31), (128, 64), (129, 300), (33, 1003), (200, 4096), (1, 8192),
                                 (1300, 40), (2, 20000), (1025, 257)])
def test_values(R, K, dtype, format):
    x = rows(R, K, dtype, seed=R + K)
    q = ops.fp4_quantize(x, format)
    want, _, row = routed.fp4_round(x, format)
    same(ops.fp4_values(q), want)
    same(q.row_scale, row)
    # the stored form, padding included
    values = routed.fp4_unpack(q.codes, q.scales, q.row_scale, K, format)
    assert torch.equal(values, want.cpu())
    assert q.codes.shape == (R, (K + 31) // 32 * 16) and q.scales.shape[0] == (R + 127) // 128
    assert not (q.codes[:, (K + 1) // 2:]).any()
    byte = q.scales.cpu()
    flat = byte.view(byte.shape[0], byte.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(byte.shape[0] * 128, -1)
    blocks = (K + routed.FP4_BLOCK[format] - 1) // routed.FP4_BLOCK[format]
    assert not flat[R:].any() and not flat[:, blocks:].any()


@pytest.mark.parametrize('format', FORMATS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_values_next_to_every_border(dtype, format):
    """Multiples of 1/8 of a scale and the numbers beside them: ties go to the even code."""
    base = torch.arange(-64, 65, device='cuda') / 8.0
    x = torch.stack([base, base * (1 + 2.0 ** -8), base * (1 - 2.0 ** -8), base * 1.0625, base * 0.4375])
    x = torch.nn.functional.pad(x, (0, 160 - x.shape[1]))
    # a block with a largest value of its own each, so that scales with every significand come up
    x = x.view(5, 10, 16) * torch.linspace(1, 2, 10, device='cuda').bfloat16().float()[:, None]
    x = torch.cat([x.flatten(1) * 2.0 ** p for p in (-60, -9, 0, 7, 60)]).to(dtype)
    want, _, _ = routed.fp4_round(x, format)
    same(ops.fp4_values(ops.fp4_quantize(x, format)), want)


@pytest.mark.parametrize('format', FORMATS)
def test_values_of_special_rows(format):
    x = torch.randn(12, 96, device='cuda')
    x[0] = 0
    x[1] = 1e-38
    x[2, 5] = math.nan
    x[3, 90] = math.inf
    x[4, 0] = -math.inf
    x[5] *= 1e30
    x[6] = torch.finfo(torch.float32).max
    x[7, 1:] = 0
    x[8] = 2.0 ** torch.arange(96, device='cuda') * 2.0 ** -60  # a wide range in a row
    x[9] = -0.0
    x[10] = torch.tensor([448.0 * 6, 1.0] * 48, device='cuda')
    x[11] = torch.tensor([448.0 * 6.0001, 1e-3] * 48, device='cuda')
    want, _, _ = routed.fp4_round(x, format)
    q = ops.fp4_quantize(x, format)
    same(ops.fp4_values(q), want)
    assert torch.equal(q.row_scale.isnan(), torch.tensor([i in (2, 3, 4) for i in range(12)], device='cuda'))


@pytest.mark.parametrize('format', FORMATS)
def test_values_of_members_with_widths(format):
    x = rows(6 * 150, 200, torch.float32, seed=1).view(6, 150, 200)
    n = torch.tensor([200, 1, 16, 17, 130, 0], device='cuda')
    for m in range(6):
        x[m, :, int(n[m]):] = math.nan
    got = ops.fp4_values(ops.fp4_quantize(x, format, n_features=n))
    for m in range(6):
        same(got[m], routed.fp4_round(x[m], format, n=int(n[m]))[0])


@pytest.mark.parametrize('format', FORMATS)
def test_strided_rows(format):
    wide = rows(40, 300, torch.bfloat16, seed=2)
    for x in (wide[:, :64], wide[:, 1:65], wide[:, 8:72], wide[::2], wide[:, ::3], wide.T[:64]):
        same(ops.fp4_values(ops.fp4_quantize(x, format)), routed.fp4_round(x, format)[0])
    assert ops.fp4_values(ops.fp4_quantize(wide[:0], format)).shape == (0, 300)


def linear_bound(mag, K):
    """Products of two 4-bit values and their scales are exact; a step of 64 of them is added with less than two units in
    the last place of 24 bits, and the row scales and the bias round once each."""
    return mag * (K / 64 + 4) * 2 * U24


def check_linear(x, w, b, format, edges=None, in_f=None, out_f=None, relu=False):
    """x: (P, B, K), shared (B, K), or (R, K) with edges."""
    P, N, K = w.shape
    weight = ops.fp4_quantize(w, format, n_features=in_f)
    wv = ops.fp4_values(weight)
    offsets = None if edges is None else torch.tensor(edges, device='cuda')
    y = ops.fp4_linear_forward(x, weight, b, offsets, in_features=in_f, out_features=out_f, relu=relu)
    assert y.dtype == x.dtype
    full = x.expand(P, *x.shape) if x.ndim == 2 and edges is None else x
    got = y if edges is not None else y.flatten(0, 1)
    if edges is None:
        B = full.shape[1]
        edges = [B * m for m in range(P + 1)]
        full = full.flatten(0, 1)
    values = torch.zeros(full.shape, dtype=torch.float64, device='cuda')
    for m in range(P):
        i = K if in_f is None else int(in_f[m])
        values[edges[m]: edges[m + 1]] = routed.fp4_round(full[edges[m]: edges[m + 1]], format, n=i)[0]
    (want,), (mag,) = routed.ragged_linear(values, wv.double(), b, edges, in_f, out_f, relu)
    assert torch.equal(got.isnan(), want.isnan())
    want, mag = want.nan_to_num(), mag.nan_to_num()
    error = (got.double().nan_to_num() - want).abs()
    assert (error <= want.abs() * torch.finfo(x.dtype).eps / 2 * 1.01 + linear_bound(mag, K)).all()
    return y


SHAPES = [
    # sizes of the members' batches, features in, features out
    ([1], 16, 8), ([0, 1], 33, 5),
    ([100, 0, 0, 5, 33, 1], 300, 260),               # few rows a member, pieces at every place of a scale tile
    ([1], 8192, 1000),                               # one row, the K loop over a cluster
    ([64, 65, 1, 0], 2100, 130),
    ([500, 128, 1, 0, 257, 129, 127], 1000, 777),    # tiles of 128 rows, partial ones
    ([1] * 300, 64, 33),                             # more members than a warp holds
    ([130] * 30, 96, 64),                            # narrow tiles
    ([3000, 2500], 520, 2300),                       # CTA pairs
]


@pytest.mark.parametrize('format', FORMATS)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('widths', [False, True])
@pytest.mark.parametrize('shape', range(len(SHAPES)))
def test_ragged_linear(shape, widths, dtype, format):
    sizes, K, N = SHAPES[shape]
    P, head, tail = len(sizes), 3, 5
    edges = [head]
    for s in sizes:
        edges.append(edges[-1] + s)
    gen = torch.Generator(device='cuda').manual_seed(shape)
    x = rows(edges[-1] + tail, K, dtype, seed=shape)
    w = torch.randn(P, N, K, generator=gen, device='cuda') * K ** -0.5
    b = torch.randn(P, N, generator=gen, device='cuda')
    in_f = out_f = None
    x[:head] = math.nan
    x[edges[-1]:] = math.inf
    if widths:
        in_f = torch.randint(1, K + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
        out_f = torch.randint(1, N + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
        for m in range(P):
            x[edges[m]: edges[m + 1], int(in_f[m]):] = w[m, :, int(in_f[m]):] = math.nan
            b[m, int(out_f[m]):] = math.nan
    check_linear(x, w, b, format, edges, in_f, out_f, relu=shape % 2 == 0)


@pytest.mark.parametrize('format', FORMATS)
@pytest.mark.parametrize('B', [1, 31, 32, 33, 300])
@pytest.mark.parametrize('shared', [False, True])
def test_linear_of_equal_batches(B, shared, format):
    P, K, N = 3, 130, 200
    x = rows(B if shared else P * B, K, torch.float32, seed=B)
    w, b = torch.randn(P, N, K, device='cuda'), torch.randn(P, N, device='cuda')
    x = x if shared else x.view(P, B, K)
    check_linear(x, w, b, format)
    check_linear(x, w, None, format, relu=True)
    in_f = torch.tensor([130, 7, 64], dtype=torch.int32, device='cuda')
    check_linear(x, w, b, format, in_f=in_f, out_f=torch.tensor([200, 3, 128], device='cuda'))
    assert ops.fp4_linear_forward(x[..., :0, :], ops.fp4_quantize(w, format)).shape == (P, 0, N)


@pytest.mark.parametrize('B', [2, 200])
def test_rows_that_are_not_finite_stay_with_themselves(B):
    x = rows(B, 64, torch.bfloat16, seed=3)[None].repeat(2, 1, 1)
    w = torch.randn(2, 40, 64, device='cuda')
    weight = ops.fp4_quantize(w)
    plain = ops.fp4_linear_forward(x, weight)
    x[0, 1, 5] = math.nan
    got = ops.fp4_linear_forward(x, weight)
    assert got[0, 1].isnan().all()
    got[0, 1] = plain[0, 1]
    assert torch.equal(got, plain)
    w[1, 7, 3] = math.inf
    got = ops.fp4_linear_forward(x[1:], ops.fp4_quantize(w[1:]))
    assert got[..., 7].isnan().all() and not got[..., :7].isnan().any()


def test_a_row_does_not_depend_on_its_batch():
    x, w = rows(2000, 256, torch.bfloat16, seed=4), torch.randn(1, 300, 256, device='cuda')
    weight = ops.fp4_quantize(w)
    every = ops.fp4_linear_forward(x.float()[None], weight)
    for n in (1, 40, 300):
        part = ops.fp4_linear_forward(x.float()[None, :n], weight)
        # (the order of the sums differs with the tiles)
        torch.testing.assert_close(part, every[:, :n], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize('format', FORMATS)
def test_in_graphs_and_on_streams(format):
    sizes = [0, 300, 301, 900]
    offsets = torch.tensor(sizes, dtype=torch.int32, device='cuda')
    x = rows(900, 160, torch.bfloat16, seed=5)
    w = ops.fp4_quantize(torch.randn(3, 72, 160, device='cuda'), format)

    def step():
        q = ops.fp4_quantize(x, format)
        return [ops.fp4_values(q), ops.fp4_linear_forward(x, w, None, offsets),
                ops.fp4_linear_forward(x.view(3, 300, 160)[:, :20], w)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(rows(900, 160, torch.bfloat16, seed=6))
    offsets.copy_(torch.tensor([0, 5, 5, 899], dtype=torch.int32))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    for a, b in zip(other, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize('format', FORMATS)
def test_layer(format):
    torch.manual_seed(7)
    linear = LinearPack([20, 64, 33], [72, 5, 40], max_in_features=64, max_out_features=72, pack_size=3).cuda()
    layer = Fp4LinearPack.from_linear(linear, format)
    assert (layer.max_in_features, layer.max_out_features, layer.pack_size) == (64, 72, 3)
    want = torch.stack([routed.fp4_round(linear.weight[m].detach(), format, n=int(linear.in_features[m]))[0] for m in range(3)])
    same(layer.dequantize(), want)
    x = torch.randn(3, 50, 64, device='cuda')
    for m in range(3):
        x[m, :, int(linear.in_features[m]):] = 0
    with torch.no_grad():
        with torch.autocast('cuda', dtype=torch.bfloat16):
            y = layer(x)
        assert y.dtype == torch.bfloat16
        q = ops.fp4_quantize(linear.weight, format, n_features=linear.in_features)
        kw = dict(in_features=linear.in_features, out_features=linear.out_features)
        assert torch.equal(y, ops.fp4_linear_forward(x.bfloat16(), q, linear.bias, **kw))
        # members by selection, rows of their own, shared rows
        idx = torch.tensor([2, 0], device='cuda')
        picked = layer(x[idx], idx)
        assert torch.equal(picked, layer(x)[idx])
        offsets = torch.tensor([0, 50, 100, 150], device='cuda')
        torch.testing.assert_close(layer.forward_rows(x.flatten(0, 1), offsets).view(3, 50, 72), layer(x), rtol=1e-5, atol=1e-5)
        assert torch.equal(layer(x[:1].expand(3, 50, 64)), layer(x[:1].repeat(3, 1, 1)))
        with layer.eval().temporarily_select(pack_idx=idx):
            assert torch.equal(layer(x[idx]), picked)
    # it is saved and loaded with the other modules
    other = Fp4LinearPack.from_linear(LinearPack([20, 64, 33], [72, 5, 40], max_in_features=64, max_out_features=72,
                                                 pack_size=3).cuda(), format)
    other.load_state_dict(layer.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), layer(x))
    layer.remove(pack_idx=torch.tensor([1], device='cuda'))
    assert layer.pack_size == 2
    with pytest.raises(RuntimeError):
        layer(x[:2].requires_grad_())


@pytest.mark.parametrize('format', FORMATS)
def test_model_in_4_bits(format):
    torch.manual_seed(8)
    model = TabPack(n_numerical_features=12, categorical_cardinalities=[3, 4], d_out=5, n_blocks=[1, 3, 2],
                    d_block=[64, 40, 56], dropout=0.0, pack_size=3, max_d_block=64).cuda().eval()
    xn, xc = torch.randn(70, 12, device='cuda'), torch.randint(0, 3, (70, 2), device='cuda')
    linears = [b.linear for b in model.backbone.blocks] + [model.output]
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        plain = model(xn, xc)
        # block by block from the same layers
        x = ops.tabpack_input(xn, xc, model._cat_offsets, 24, torch.bfloat16)[:, :19].contiguous()
        nb = model.backbone.n_blocks
        for i, layer in enumerate(linears):
            q = ops.fp4_quantize(layer.weight, format, n_features=layer.in_features)
            y = ops.fp4_linear_forward(x, q, layer.bias, in_features=layer.in_features, out_features=layer.out_features,
                                       relu=layer is not model.output)
            x = torch.where((nb > i).view(-1, 1, 1), y, x) if 0 < i < 3 else y
        fp4_(model, format)
        got = model(xn, xc)
        assert not any(isinstance(m, LinearPack) for m in model.modules())
        assert torch.equal(got, x)
        # 4 bits are coarse: the outputs follow the bf16 model's, no more is asked here
        assert torch.corrcoef(torch.stack([got.flatten().float(), plain.flatten().float()]))[0, 1] > 0.9
        idx = torch.tensor([2, 0], device='cuda')
        assert torch.equal(model(xn, xc, idx), got[idx])
        assert torch.equal(model(xn, xc, idx, max_width=64), got[idx])
    with pytest.raises(RuntimeError):
        model.train()
        with torch.autocast('cuda', dtype=torch.bfloat16):
            model(xn.expand(3, 70, 12), xc.expand(3, 70, 2))


def test_kept_layers_and_depth():
    torch.manual_seed(9)
    backbone = MLPBackbonePack(d_in=16, n_blocks=[1, 2], d_block=[32, 24], max_d_block=32, dropout=0.0, pack_size=2).cuda()
    first = backbone.blocks[0].linear
    fp4_(backbone, keep=[first])
    assert backbone.blocks[0].linear is first and isinstance(backbone.blocks[1].linear, Fp4LinearPack)
    x = torch.randn(2, 9, 16, device='cuda')
    with torch.no_grad():
        y = backbone(x)
        h = torch.relu(first(x))
        assert torch.equal(y[0], h[0]) and not torch.equal(y[1], h[1])
    with pytest.raises(TypeError):
        fp4_(first)


def test_predictor_in_4_bits():
    model = dict(n_numerical_features=10, categorical_cardinalities=[], d_out=3, max_n_blocks=2, max_d_block=64)
    members = [dict(n_blocks=2, d_block=w, dropout=0.0) for w in (32, 64, 48, 24)]
    trainer = PackTrainer(n_members=4, model=model, per_member_model=members,
                          optimizer=dict(type='adamw', lr=1e-2, weight_decay=0.0), loss='ce', seed=0, device='cuda')
    x = torch.randn(90, 10, device='cuda')
    heads = {'all': torch.arange(4)}
    before = [p.detach().clone() for p in trainer.model.parameters()]
    predictor = PackPredictor(trainer, heads, weight_format='nvfp4')
    probs, mean = predictor(x, None)
    chunked, _ = predictor(x, None, member_chunk=2)
    plain, _ = PackPredictor(trainer, heads)(x, None)
    assert probs.shape == plain.shape == (4, 90, 3)
    torch.testing.assert_close(probs.sum(-1), torch.ones(4, 90, device='cuda'))
    torch.testing.assert_close(chunked, probs, rtol=2e-2, atol=2e-2)
    assert not torch.equal(probs, plain) and (probs - plain).abs().max() < 0.3
    torch.testing.assert_close(mean['all'], probs.mean(0))
    # the trainer's own model is untouched, the copy holds no fp32 weights and keeps what it was made of
    assert all(torch.equal(a, b) for a, b in zip(before, trainer.model.parameters()))
    assert not any(p.numel() for p in predictor.model.parameters())
    with torch.no_grad():
        for p in trainer.model.parameters():
            p.zero_()
    assert torch.equal(predictor(x, None)[0], probs)


def test_refusals():
    x, w = torch.zeros(4, 32, device='cuda'), torch.randn(2, 8, 32, device='cuda')
    q = ops.fp4_quantize(w)
    with pytest.raises(ValueError):
        ops.fp4_quantize(x, 'fp4')
    with pytest.raises(TypeError):
        ops.fp4_quantize(x.half())
    with pytest.raises(ValueError):
        ops.fp4_quantize(x[0])
    with pytest.raises(ValueError):
        ops.fp4_quantize(x[:, :0])
    with pytest.raises(ValueError):
        ops.fp4_quantize(w, offsets=torch.tensor([0, 4], device='cuda'))
    with pytest.raises(ValueError):
        ops.fp4_quantize(w, n_features=torch.tensor([1, 2, 3], device='cuda'))
    with pytest.raises(ValueError):
        ops.fp4_linear_forward(x[:, :16], q)
    with pytest.raises(ValueError):
        ops.fp4_linear_forward(torch.zeros(3, 4, 32, device='cuda'), q)
    with pytest.raises(ValueError):
        ops.fp4_linear_forward(x, ops.fp4_quantize(w[0]))
    with pytest.raises(ValueError):
        ops.fp4_linear_forward(x, q, torch.zeros(2, 9, device='cuda'))
    with pytest.raises(ValueError):
        ops.fp4_linear_forward(x, q, None, torch.tensor([0, 4], device='cuda'))
    with pytest.raises(ValueError):
        ops.fp4_linear_forward(x, q._replace(scales=q.scales[:, :, :2]))
    with pytest.raises(TypeError):
        ops.fp4_linear_forward(x, q._replace(codes=q.codes.int()))
    with pytest.raises(ValueError):
        ops.fp4_linear_forward(x, q._replace(format='mxfp4'))
    with pytest.raises(RuntimeError):
        ops.fp4_linear_forward(x.cpu(), q)


@pytest.mark.parametrize('K', [32768, 32767])
def test_more_elements_than_31_bits(K):
    x = torch.randn(66000, 32768, device='cuda', dtype=torch.bfloat16)[:, :K]
    for format in ('nvfp4', 'mxfp4'):
        values = ops.fp4_values(ops.fp4_quantize(x, format))
        alone = ops.fp4_values(ops.fp4_quantize(x[-130:].contiguous(), format))
        assert torch.equal(values[-130:], alone)
