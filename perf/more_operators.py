"""Cases of routed packs: routing, moving rows, products over ragged groups of rows, 4-bit rows and products.

Each case is one pass through an operator, in its plain form (elementary torch operations, `own` false)
or through this package's kernels (`own` true).

route, per row of logits z over E members:
    p = softmax(z),  S = the k best finite z (ties: lowest member),  w_j = p_j / sum_S p  or  p_j
    (row, slot) pairs sorted by member, stably; pairs without a member come last;  importance = sum_rows p
    dz_e = w_e (g_e - sum_S w g) [e in S] + p_e (h_e - sum p h)   with w's and importance's gradients g and h
rows:
    xs[position[t, j]] = x[t],  out[t] = sum_j w[t, j] y[position[t, j]]
    dy[position[t, j]] = w[t, j] dout[t],  dw[t, j] = <dout[t], y[position[t, j]]>,  dx[t] = sum_j dxs[position[t, j]]
ragged linear, member m over its own rows (in_m of the columns, out_m of the outputs, zero beyond):
    y = relu(x w_m^T + b_m),  g = dy [y > 0],  dx = g w_m,  dw_m = g^T x,  db_m = sum g
4-bit rows: e2m1 values times a scale per block of a row's columns
    nvfp4: blocks of 16, scale s 2^r; 2^r the row's power of two with max|row| <= 2688 2^r < 2 max|row|, s = e4m3(max|block| / (6 2^r))
    mxfp4: blocks of 32, scale 2^(floor(log2 max|block|) - 2)
4-bit linear: y = relu(q(x) q(w_m)^T + b_m), both operands in 4 bits, sums in 32
"""

import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}
BLOCK = {'nvfp4': 16, 'mxfp4': 32}


def listed():
    return [
        # serving: a handful of rows over the members of a pack
        dict(name='route few rows', op='route', T=4, E=64, k=4, dtype='bf16', renorm=True, masked=False, train=False),
        # a training batch over a pack with members that some rows may not use, odd sizes
        dict(name='route batch train', op='route', T=65521, E=257, k=6, dtype='fp32', renorm=False, masked=True,
             train=True),
        # odd sizes in fp32, slots without a member
        dict(name='rows odd train', op='rows', T=1003, k=3, E=24, W=771, dtype='fp32', masked=True, train=True),
        # a training batch's activations to two members each and back
        dict(name='rows batch train', op='rows', T=32768, k=2, E=64, W=4096, dtype='bf16', masked=False, train=True),
        # serving: sixteen rows spread over 64 members
        dict(name='ragged few rows', op='ragged', P=64, R=16, K=1024, N=4096, dtype='bf16', widths=False, relu=True,
             train=False),
        # a pack of members of different widths and batches, one of them without rows; rows after the last one's
        dict(name='ragged odd train', op='ragged', P=7, R=2571, K=200, N=531, dtype='bf16', widths=True, relu=True,
             train=True),
        # the same without autocast
        dict(name='ragged fp32 train', op='ragged', P=12, R=4099, K=100, N=512, dtype='fp32', widths=False, relu=False,
             train=True),
        # a large routed layer's training step
        dict(name='ragged batch train', op='ragged', P=8, R=32768, K=4096, N=4096, dtype='bf16', widths=False,
             relu=False, train=True),
        # activations of a few rows of an odd width
        dict(name='fp4 few rows', op='quantize', R=33, K=1003, dtype='bf16', format='nvfp4'),
        # a large batch's activations, or a large layer's weights
        dict(name='fp4 batch', op='quantize', R=16384, K=8192, dtype='fp32', format='mxfp4'),
        # serving: one row through a large layer
        dict(name='fp4 linear one row', op='fp4', P=1, R=1, K=8192, N=8192, dtype='bf16', format='nvfp4', ragged=False,
             relu=True),
        # prediction: a routed batch over large members
        dict(name='fp4 linear batch', op='fp4', P=4, R=16384, K=8192, N=8192, dtype='bf16', format='nvfp4', ragged=True,
             relu=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['route', 'rows', 'ragged', 'ragged', 'quantize', 'fp4', 'fp4'])
    some = rng.choice(['bf16', 'bf16', 'fp32'])
    if op == 'route':
        E = _log(rng, 2, 1024)
        T = _log(rng, 1, min(65536, 2 ** 24 // E))
        return dict(op=op, T=T, E=E, k=rng.randint(1, min(E, 8)), dtype=some, renorm=rng.random() < 0.5,
                    masked=rng.random() < 0.4, train=rng.random() < 0.6)
    if op == 'rows':
        W, k = _log(rng, 8, 8192), rng.randint(1, 8)
        T = _log(rng, 1, max(1, min(32768, 2 ** 27 // (W * k))))
        return dict(op=op, T=T, k=k, E=k * _log(rng, 1, 32), W=W, dtype=some, masked=rng.random() < 0.4,
                    train=rng.random() < 0.6)
    if op == 'quantize':
        K = _log(rng, 16, 16384)
        return dict(op=op, R=_log(rng, 1, min(16384, 2 ** 26 // K)), K=K, dtype=some,
                    format=rng.choice(['nvfp4', 'mxfp4']))
    P, K, N = _log(rng, 1, 64), _log(rng, 16, 8192), _log(rng, 8, 8192)
    while P * K * N > 2 ** 28:
        P = max(1, P // 2)
        K, N = max(16, K * 4 // 5), max(8, N * 4 // 5)
    most = 2 ** 38 if op == 'fp4' or some == 'bf16' else 2 ** 35
    R = _log(rng, 1, max(1, min(32768, most // (K * N), 2 ** 27 // max(K, N))))
    if op == 'ragged':
        return dict(op=op, P=P, R=R, K=K, N=N, dtype=some, widths=rng.random() < 0.4, relu=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    ragged = rng.random() < 0.6
    return dict(op=op, P=P, R=R if ragged else max(1, R // P), K=K, N=N, dtype=some,
                format=rng.choice(['nvfp4', 'nvfp4', 'mxfp4']), ragged=ragged, relu=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs


def _group_sizes(case, seed):
    """Rows per member: shares that differ by a factor of a few, one member of a pack without rows, and a few
    rows that belong to none."""
    P, R = case['P'], case['R']
    gen = torch.Generator().manual_seed(seed)
    if R < 4 * P:
        return torch.bincount(torch.randint(0, P, (R,), generator=gen), minlength=P)
    share = 0.5 + torch.rand(P, generator=gen)
    if P > 4:
        share[torch.randint(0, P, (1,), generator=gen)] = 0
    left = R - min(R // 50, 100)
    edges = torch.round(torch.cumsum(share, 0) / share.sum() * left).long()
    return torch.diff(edges, prepend=torch.zeros(1, dtype=torch.long))


def _widths(P, most, gen):
    return torch.randint((most + 1) // 2, most + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=gen, device='cuda')  # noqa: E731
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    state = {'case': case}
    dt = DTYPES[case['dtype']]
    if case['op'] == 'route':
        T, E, k = case['T'], case['E'], case['k']
        # scores of a linear layer, some members preferred
        logits = (1.5 * normal(T, E) + 0.7 * normal(E)).to(dt)
        if case['masked']:
            # members that a row may not use; some rows have none left
            logits.masked_fill_((rand(T, E) < 0.3) | (rand(T, 1) < 0.02), -math.inf)
        state['logits'] = logits
        if case['train']:
            state['g_weight'], state['g_importance'] = normal(T, k) / T, 0.01 * normal(E) / T
        return state
    if case['op'] == 'rows':
        T, k, E, W = case['T'], case['k'], case['E'], case['W']
        expert = rand(T, E).argsort(1)[:, :k]
        if case['masked']:
            expert = torch.where(rand(T, k) < 0.1, E, expert)
        state['position'], state['offsets'] = _plan(expert, E)
        state['weight'] = torch.where(expert < E, rand(T, k), 0.0)
        state['x'], state['y'] = normal(T, W).to(dt), normal(T * k, W).to(dt)
        # nobody writes the rows of slots without a member
        state['y'][torch.arange(T * k, device='cuda') >= state['offsets'][E]] = math.nan
        if case['train']:
            state['dout'], state['dxs'] = (normal(T, W) / T).to(dt), (normal(T * k, W) / T).to(dt)
        return state
    if case['op'] == 'quantize':
        # activations whose size differs from row to row and a little from column to column
        state['x'] = (normal(case['R'], case['K']) * torch.exp(normal(case['R'], 1)) * torch.exp(0.5 * normal(case['K']))).to(dt)
        return state
    P, R, K, N = case['P'], case['R'], case['K'], case['N']
    ragged = case['op'] == 'ragged' or case['ragged']
    if ragged:
        sizes = _group_sizes(case, seed)
        ends = torch.cumsum(sizes, 0)
        state['most'] = int(sizes.max())
        state['offsets'] = torch.nn.functional.pad(ends, (1, 0)).to('cuda', torch.int32)
    state['x'] = normal(*((R, K) if ragged else (P, R, K))).to(dt)
    w, state['b'] = normal(P, N, K) * K ** -0.5, 0.2 * normal(P, N)
    if case['op'] == 'ragged':
        state['w'] = w.to(dt)
        state['in_f'], state['out_f'] = (_widths(P, K, gen), _widths(P, N, gen)) if case['widths'] else (None, None)
        if case['train']:
            state['dy'] = (normal(R, N) / R).to(dt)
            # the activations that the forward of this step left for its backward
            state['saved'] = torch.relu(normal(R, N)).to(dt)
        return state
    # a layer's weights as they are kept for prediction
    state['codes'], state['scales'], state['row_scale'] = _pack(*_encode(w, case['format']), case['format'])
    return state


# ------------------------------------------------------------------ plain forms


def _plan(expert, E):
    """(row, slot) pairs sorted by member: each pair's place, and where the members' rows begin."""
    flat = expert.flatten()
    order = torch.sort(flat, stable=True)[1]
    position = torch.empty_like(order)
    position[order] = torch.arange(len(flat), device=flat.device)
    offsets = torch.searchsorted(flat[order], torch.arange(E + 1, device=flat.device))
    return position.view(expert.shape).int(), offsets.int()


def _route_plain(s):
    case = s['case']
    E, k = case['E'], case['k']
    z, expert = torch.sort(s['logits'].float(), dim=1, descending=True, stable=True)
    z, expert = z[:, :k], expert[:, :k]
    there = z > -math.inf
    expert = torch.where(there, expert, -1)
    best = torch.where(there[:, :1], z[:, :1], 0.0)
    e = torch.exp(s['logits'].float() - best)
    total = e.sum(1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    w = torch.exp(z - best)
    total = w.sum(1, keepdim=True) if case['renorm'] else total
    w = w / torch.where(total > 0, total, 1.0)
    position, offsets = _plan(torch.where(there, expert, E), E)
    out = [w, expert.int(), position, offsets, p.double().sum(0).float()]
    if case['train']:
        g, h = s['g_weight'], s['g_importance']
        dz = p * (h - (p * h).sum(1, keepdim=True))
        wg = (w * g).sum(1, keepdim=True)
        at = torch.where(there, expert, 0)
        dz = dz.scatter_add(1, at, torch.where(there, w * (g - wg) if case['renorm'] else w * g, 0.0))
        if not case['renorm']:
            dz = dz - p * wg
        out.append(dz.to(s['logits'].dtype))
    return out


def _rows_plain(s):
    case = s['case']
    T, k, W = case['T'], case['k'], case['W']
    dt = s['x'].dtype
    at = s['position'].long()
    there = (s['position'] < s['offsets'][-1])[..., None]

    def rows(t):
        return torch.where(there, t.float()[at], 0.0)

    w = s['weight'][..., None]
    xs = s['x'].new_zeros(T * k, W)
    xs[at.flatten()] = torch.where(there, s['x'][:, None], 0).view(T * k, W)
    out = [xs, (w * rows(s['y'])).sum(1).to(dt)]
    if case['train']:
        dout = s['dout'].float()[:, None]
        dy = torch.zeros_like(s['y'])
        dy[at.flatten()] = torch.where(there, w * dout, 0.0).view(T * k, W).to(dt)
        out += [dy, (dout * rows(s['y'])).sum(-1), rows(s['dxs']).sum(1).to(dt)]
    return out


def _groups(s):
    """(P, most) row numbers of the members' rows, one after the last row where a member has fewer."""
    first, end = s['offsets'][:-1].long()[:, None], s['offsets'][1:].long()[:, None]
    at = first + torch.arange(s['most'], device=first.device)
    return torch.where(at < end, at, s['case']['R'])


def _take(x, at):
    return torch.nn.functional.pad(x.float(), (0, 0, 0, 1))[at]


def _put(y, at, rows):
    out = y.new_zeros(rows + 1, y.shape[-1])
    out[at.flatten()] = y.flatten(0, 1)
    return out[:rows]


def _ragged_plain(s):
    case = s['case']
    R, K, N = case['R'], case['K'], case['N']
    dt = s['x'].dtype
    at = _groups(s)
    x, w, b = _take(s['x'], at), s['w'].float(), s['b']
    if case['widths']:
        keep_in = torch.arange(K, device=w.device) < s['in_f'][:, None]
        keep_out = torch.arange(N, device=w.device) < s['out_f'][:, None]
        x = torch.where(keep_in[:, None], x, 0.0)
        w = torch.where(keep_out[..., None] & keep_in[:, None], w, 0.0)
        b = torch.where(keep_out, b, 0.0)
    y = x @ w.mT + b[:, None]
    if case['relu']:
        y = torch.clamp(y, min=0.0)
    out = [_put(y, at, R).to(dt)]
    if case['train']:
        g = _take(s['dy'], at)
        if case['relu']:
            g = torch.where(_take(s['saved'], at) > 0, g, 0.0)
        if case['widths']:
            g = torch.where(keep_out[:, None], g, 0.0)
        out += [_put(g @ w, at, R).to(dt), g.mT @ x, g.sum(1)]
    return out


def _blocks(x, format):
    """(..., K) as (..., blocks, block), zeros after the end."""
    n = BLOCK[format]
    k = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -k % n)).unflatten(-1, (-1, n))


def _power(n):
    """2^n in fp32, -126 <= n <= 127, from its bits."""
    return ((n.int() + 127) << 23).view(torch.float32)


def _encode(x, format):
    """fp32 (..., K) -> codes (..., blocks, block) 0 to 15, the blocks' scales as bytes, the rows' scales."""
    x = _blocks(x.float(), format)
    big = x.abs().amax(-1)
    if format == 'mxfp4':
        power = torch.clamp(torch.frexp(big)[1] - 3, min=-100)
        power = torch.where(big > 0, power, -100)
        scale = _power(power)
        byte = (power + 127).to(torch.uint8)
        row = torch.ones_like(big[..., 0])
    else:
        part, power = torch.frexp(big.amax(-1))
        row = _power(torch.clamp(torch.where(part > 2688 / 4096, power - 11, power - 12), min=-100))
        small = (big / (6 * row[..., None])).to(torch.float8_e4m3fn)
        scale = small.float() * row[..., None]
        byte = small.view(torch.uint8)
    q = torch.where(scale[..., None] > 0, x.abs() / scale[..., None], 0.0)
    # the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6; in the middle the even code
    code = ((q > 0.25).to(torch.uint8) + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5) + (q > 5))
    return code + 8 * (x < 0).to(torch.uint8), byte, row


def _decode(code, byte, row, format, K):
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=code.device)[(code & 7).long()]
    value = torch.where(code > 7, -value, value)
    if format == 'mxfp4':
        scale = _power(byte.int() - 127)
    else:
        scale = byte.view(torch.float8_e4m3fn).float() * row[..., None]
    return (value * scale[..., None]).flatten(-2)[..., :K]


def _pack(code, byte, row, format):
    """Two codes a byte, the even column's in the low half, rows padded to 32 columns; scales in tiles of 128 rows
    by 4 blocks, byte 16 (row % 32) + 4 (row / 32) + block % 4 of a tile, tiles of a row padded to 256 columns."""
    code = code.flatten(-2)
    code = torch.nn.functional.pad(code, (0, -code.shape[-1] % 32))
    N, B = byte.shape[-2:]
    byte = torch.nn.functional.pad(byte, (0, -B % (256 // BLOCK[format]), 0, -N % 128))
    byte = byte.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32)).permute(0, 1, 4, 3, 2, 5).flatten(-3)
    return code[..., ::2] + 16 * code[..., 1::2], byte.contiguous(), row


def _unpack(codes, scales, row, format, K):
    N, n = codes.shape[-2], BLOCK[format]
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., : (K + n - 1) // n * n].unflatten(-1, (-1, n))
    byte = scales.unflatten(-1, (32, 4, 4)).permute(0, 1, 4, 3, 2, 5).flatten(-2).flatten(1, 3)
    return _decode(code, byte[:, :N, : (K + n - 1) // n].contiguous(), row, format, K)


def _quantize_plain(s):
    case = s['case']
    return [_decode(*_encode(s['x'], case['format']), case['format'], case['K']).bfloat16()]


def _fp4_plain(s):
    case = s['case']
    x = _decode(*_encode(s['x'], case['format']), case['format'], case['K'])
    w = _unpack(s['codes'], s['scales'], s['row_scale'], case['format'], case['K'])
    if case['ragged']:
        at = _groups(s)
        x = _take(x, at)
    y = x @ w.mT + s['b'][:, None]
    if case['relu']:
        y = torch.clamp(y, min=0.0)
    return [(_put(y, at, case['R']) if case['ragged'] else y).to(s['x'].dtype)]


# ------------------------------------------------------------------ the framework's calls


def _route_own(s):
    from tabpack_b200 import ops

    case = s['case']
    weight, expert, position, offsets, importance = ops.route_forward(s['logits'], case['k'], renormalize=case['renorm'])
    out = [weight, expert, position, offsets, importance]
    if case['train']:
        out.append(ops.route_backward(s['g_weight'], s['g_importance'], s['logits'], weight, expert,
                                      renormalize=case['renorm']))
    return out


def _rows_own(s):
    from tabpack_b200 import ops

    plan = s['position'], s['offsets']
    out = [ops.dispatch_rows(s['x'], *plan), ops.combine_rows(s['y'], s['weight'], *plan)]
    if s['case']['train']:
        out += ops.combine_rows_backward(s['dout'], s['y'], s['weight'], *plan)
        out.append(ops.combine_rows(s['dxs'], None, *plan))
    return out


def _ragged_own(s):
    from tabpack_b200 import ops

    relu = s['case']['relu']
    kw = dict(in_features=s['in_f'], out_features=s['out_f'], relu=relu)
    out = [ops.ragged_linear_forward(s['x'], s['w'], s['b'], s['offsets'], **kw)]
    if s['case']['train']:
        out += ops.ragged_linear_backward(s['dy'], s['x'], s['w'], s['saved'] if relu else None, s['offsets'], **kw)
    return out


def _quantize_own(s):
    from tabpack_b200 import ops

    return [ops.fp4_values(ops.fp4_quantize(s['x'], s['case']['format']))]


def _fp4_own(s):
    from tabpack_b200 import ops

    case = s['case']
    weight = ops.Fp4Rows(s['codes'], s['scales'], s['row_scale'], case['K'], case['format'])
    return [ops.fp4_linear_forward(s['x'], weight, s['b'], s['offsets'] if case['ragged'] else None, relu=case['relu'])]


def run(state):
    op = state['case']['op']
    if own:
        return {'route': _route_own, 'rows': _rows_own, 'ragged': _ragged_own, 'quantize': _quantize_own,
                'fp4': _fp4_own}[op](state)
    return {'route': _route_plain, 'rows': _rows_plain, 'ragged': _ragged_plain, 'quantize': _quantize_plain,
            'fp4': _fp4_plain}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    size = 2 if case['dtype'] == 'bf16' else 4
    if case['op'] == 'route':
        T, E, k = case['T'], case['E'], case['k']
        n = T * E * size + T * k * 12 + E * 8
        return {'bytes': n + (T * E * size + T * k * 4 if case['train'] else 0),
                'flops': T * E * (12 if case['train'] else 6)}
    if case['op'] == 'rows':
        T, k, W = case['T'], case['k'], case['W']
        one, many, plan = T * W * size, T * k * W * size, T * k * 8
        if not case['train']:
            return {'bytes': 2 * one + 2 * many + plan, 'flops': 2 * T * k * W}
        # x, out, dout, dx; xs, y, dy, dxs
        return {'bytes': 4 * one + 4 * many + plan + T * k * 4, 'flops': 6 * T * k * W}
    if case['op'] == 'quantize':
        # the rows read, their 4-bit form written and read again, the values written
        R, K = case['R'], case['K']
        return {'bytes': R * K * (size + 2) + R * K * (1 + 2 / BLOCK[case['format']]), 'flops': 8 * R * K}
    P, R, K, N = (case[k] for k in ('P', 'R', 'K', 'N'))
    if case['op'] == 'ragged':
        used = min(P, R)
        n = R * (K + N) * size + used * N * (K * size + 4)
        # a member's widths are three quarters of the largest on average
        share = 0.5625 if case['widths'] else 1.0
        if not case['train']:
            return {'bytes': n, 'flops': 2 * R * K * N * share}
        n += R * (K + N) * size + P * N * (K + 1) * 4 + (R * N * size if case['relu'] else 0)
        return {'bytes': n, 'flops': 6 * R * K * N * share}
    used, rows = (min(P, R), R) if case['ragged'] else (P, P * R)
    n = rows * (K + N) * size + used * N * (K * (0.5 + 1 / BLOCK[case['format']]) + 8)
    return {'bytes': n, 'flops': 2 * rows * K * N}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {'route': _route_exact, 'rows': _rows_exact, 'ragged': _ragged_exact, 'quantize': _quantize_exact,
            'fp4': _fp4_exact}[case['op']](s)


def _route_exact(s):
    """With autograd's gradients of a softmax over the members that are left."""
    case = s['case']
    T, E, k = case['T'], case['E'], case['k']
    z = s['logits'].double().requires_grad_(case['train'])
    expert = torch.argsort(-z.detach(), dim=1, stable=True)[:, :k]
    chosen = z.gather(1, expert)
    there = chosen.detach() > -math.inf
    some = there.any(1, keepdim=True)
    p = torch.softmax(torch.where(some, z, 0.0), 1) * some
    w = torch.softmax(torch.where(some, chosen, 0.0), 1) * some if case['renorm'] else p.gather(1, expert)
    importance = p.sum(0)
    expert = torch.where(there, expert, -1)
    # each pair's place: the pairs of lower members, and the earlier ones of its own
    flat = torch.where(there, expert, E).flatten()
    order = torch.argsort(flat * (T * k) + torch.arange(T * k, device='cuda'))
    position = torch.argsort(order).view(T, k)
    offsets = torch.cumsum(torch.bincount(flat, minlength=E + 1), 0) - torch.bincount(flat, minlength=E + 1)
    out = [w.detach(), expert, position, offsets, importance.detach()]
    if case['train']:
        loss = (w * s['g_weight'].double()).sum() + (importance * s['g_importance'].double()).sum()
        out.append(torch.autograd.grad(loss, z)[0].nan_to_num())
    return out


def _rows_exact(s):
    """From the plan's inverse, pair by pair of a row."""
    case = s['case']
    T, k, W = case['T'], case['k'], case['W']
    used = int(s['offsets'][-1])
    back = torch.argsort(s['position'].flatten())[:used]
    token = back // k
    w = s['weight'].flatten()[back].double()[:, None]
    x, y = s['x'].double(), s['y'][:used].double()
    fill = lambda t: torch.nn.functional.pad(t, (0, 0, 0, T * k - used))  # noqa: E731
    zero = lambda: torch.zeros(T, W, dtype=torch.float64, device='cuda')  # noqa: E731
    out = [fill(x[token]), zero().index_add_(0, token, w * y)]
    if case['train']:
        dout = s['dout'].double()[token]
        dw = torch.zeros(T * k, dtype=torch.float64, device='cuda')
        dw[back] = torch.einsum('rw,rw->r', dout, y)
        out += [fill(w * dout), dw.view(T, k), zero().index_add_(0, token, s['dxs'][:used].double())]
    return out


def _ragged_exact(s):
    """Member by member."""
    case = s['case']
    P, R, K, N = (case[k] for k in ('P', 'R', 'K', 'N'))
    edge = s['offsets'].tolist()
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device='cuda')  # noqa: E731
    y, dx, dw, db = new(R, N), new(R, K), new(P, N, K), new(P, N)
    for m in range(P):
        a, b = edge[m], edge[m + 1]
        i, o = (int(s['in_f'][m]), int(s['out_f'][m])) if case['widths'] else (K, N)
        x, w = s['x'][a:b, :i].double(), s['w'][m, :o, :i].double()
        t = torch.addmm(s['b'][m, :o].double(), x, w.T)
        y[a:b, :o] = t.relu() if case['relu'] else t
        if case['train']:
            g = s['dy'][a:b, :o].double()
            if case['relu']:
                g = g * (s['saved'][a:b, :o] > 0)
            dx[a:b, :i], dw[m, :o, :i], db[m, :o] = g @ w, g.T @ x, g.sum(0)
    return [y, dx, dw, db] if case['train'] else [y]


def _power_exact(n):
    """2^n for whole n from -200 to 200, from a table."""
    return torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=n.device)[n.long() + 200]


def _floor_log2(x):
    return torch.frexp(x)[1] - 1


def _round_exact(x, format):
    """(..., K) to 4 bits and back, on grids of powers of two."""
    n, K = BLOCK[format], x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -K % n))
    x = x.view(*x.shape[:-1], -1, n)
    big = x.abs().amax(-1, keepdim=True)
    if format == 'mxfp4':
        scale = _power_exact(_floor_log2(big.clamp(min=2.0 ** -98)) - 2)
    else:
        row = _power_exact((-_floor_log2(2688 / big.amax(-2, keepdim=True).clamp(min=2.0 ** -120))).clamp(min=-100))
        t = big / 6 / row
        # e4m3: three bits after the leading one, steps of 2^-9 at least
        step = _power_exact(_floor_log2(t.clamp(min=2.0 ** -6)) - 3)
        scale = torch.round(t / step) * step * row
    t = torch.where(scale > 0, x.abs() / scale, 0.0).clamp(max=6.0)
    step = _power_exact(_floor_log2(t.clamp(min=1.0)) - 1)
    return (torch.sign(x) * torch.round(t / step) * step * scale).flatten(-2)[..., :K]


def _quantize_exact(s):
    # six significant bits at most: 32 hold them
    return [_round_exact(s['x'], s['case']['format']).float()]


def _fp4_exact(s):
    """Member by member, the weights' values from tables of the codes and scale bytes."""
    case = s['case']
    P, R, K, N = (case[k] for k in ('P', 'R', 'K', 'N'))
    n = BLOCK[case['format']]
    sign = torch.tensor([1.0, -1.0], dtype=torch.float64, device='cuda')
    small = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device='cuda')
    byte = torch.arange(256, device='cuda', dtype=torch.float64)
    if case['format'] == 'mxfp4':
        table = _power_exact(byte - 127)
    else:
        e, f = torch.floor(byte / 8) % 16, byte % 8
        table = torch.where(e > 0, (1 + f / 8) * _power_exact(e - 7), f / 512)
    row, col = torch.arange(N, device='cuda')[:, None], torch.arange(K, device='cuda')
    tile, block = row // 128, col // n
    inside = row % 32 * 16 + row % 128 // 32 * 4 + block % 4
    x = _round_exact(s['x'], case['format'])
    y = torch.zeros(*x.shape[:-1], N, dtype=torch.float64, device='cuda')
    edge = s['offsets'].tolist() if case['ragged'] else None
    for m in range(P):
        code = (s['codes'][m][:, col // 2] >> (col % 2 * 4).to(torch.uint8)).long() & 15
        w = sign[code >> 3] * small[code & 7] * table[s['scales'][m][tile, block // 4, inside].long()]
        w = w * s['row_scale'][m].double()[:, None]
        rows = slice(edge[m], edge[m + 1]) if case['ragged'] else m
        t = torch.addmm(s['b'][m].double(), x[rows], w.T)
        y[rows] = t.relu() if case['relu'] else t
    return [y]
