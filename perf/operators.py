"""Cases of the packed layer norm, the label log probabilities and the AdamW step with 8-bit moments.

Each case is one pass through an operator, in its plain form (elementary torch operations, `own` false)
or through this package's kernels (`own` true).

layer norm, member m over its first n_m of W columns (zero beyond):
    xhat = (x - mean) / sqrt(var + eps),  y = xhat w_m + b_m
    dx = (dy w - mean(dy w) - xhat mean(dy w xhat)) / sqrt(var + eps),  dw = sum_r dy xhat,  db = sum_r dy
label log probabilities, per row of logits z:
    log p_c = z_c - log sum_c' exp z_c',  H = -sum_c p_c log p_c,  the top k classes (ties: lowest index)
    dz_c = g_l (1[c = label] - p_c) - g_H p_c (log p_c + H)
AdamW with moments in 8 bits, blocks of 128 elements of a member, one fp32 scale each:
    p <- p (1 - lr wd),  m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2
    p <- p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
    m is stored as e4m3 times max|m| / 448, sqrt(v) as an unsigned 4-bit exponent and 4-bit mantissa
    times max sqrt(v) / 1.9375; both are rounded up or down at random in proportion to the distance, with
    16 bits each of Philox4x32-10 keyed by the seed, counter (element / 4, tensor, member, step).
"""

import math

import torch

own = False

EPS = 1e-5
BLOCK = 128
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def listed():
    return [
        # one row of every member: a single prediction of a 32-member pack
        dict(name='norm one row', op='norm', P=32, B=1, W=512, dtype='bf16', ragged=True, shared=False, train=False),
        # a batch shared by the members, odd sizes, fp32: the first layer of a small pack
        dict(name='norm shared odd', op='norm', P=7, B=333, W=771, dtype='fp32', ragged=True, shared=True, train=True),
        # a training step's hidden activations: 64 members of different widths
        dict(name='norm pack train', op='norm', P=64, B=1024, W=512, dtype='bf16', ragged=True, shared=False,
             train=True),
        # one wide model on a long batch
        dict(name='norm wide train', op='norm', P=1, B=16384, W=8192, dtype='bf16', ragged=False, shared=False,
             train=True),
        # a few rows over a long list of labels, with the best alternatives: serving
        dict(name='labels serve', op='labels', P=1, B=4, C=51200, dtype='bf16', k=10, masked=False, train=False),
        # evaluation with classes masked out per row
        dict(name='labels eval masked', op='labels', P=3, B=2571, C=1009, dtype='fp32', k=5, masked=True, train=False),
        # the loss of a 512-member pack on 10 classes: log probabilities, entropies and their gradient
        dict(name='labels pack train', op='labels', P=512, B=1024, C=10, dtype='bf16', k=0, masked=False, train=True),
        # the loss of one model over a long list of labels
        dict(name='labels long train', op='labels', P=1, B=8192, C=65536, dtype='bf16', k=0, masked=False, train=True),
        # a single small model: launch latency
        dict(name='adamw8 small', op='adamw8', P=1, d_in=24, width=64, layers=2, classes=3, per_member=False),
        # odd sizes (no row starts on a 16-byte boundary), every member with its own hyperparameters and step
        dict(name='adamw8 odd pack', op='adamw8', P=5, d_in=37, width=531, layers=3, classes=7, per_member=True),
        # a pack's training step
        dict(name='adamw8 pack', op='adamw8', P=64, d_in=100, width=512, layers=2, classes=10, per_member=True),
        # one large model
        dict(name='adamw8 large', op='adamw8', P=1, d_in=8192, width=8192, layers=3, classes=1000, per_member=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'labels', 'adamw8'])
    if op == 'norm':
        P, W = _log(rng, 1, 128), _log(rng, 2, 8192)
        B = _log(rng, 1, max(1, min(16384, 2 ** 26 // (P * W))))
        return dict(op=op, P=P, B=B, W=W, dtype=rng.choice(['bf16', 'bf16', 'fp32']), ragged=rng.random() < 0.6,
                    shared=rng.random() < 0.25, train=rng.random() < 0.7)
    if op == 'labels':
        P, C = _log(rng, 1, 256), _log(rng, 2, 131072)
        B = _log(rng, 1, max(1, min(16384, 2 ** 27 // (P * C))))
        train = rng.random() < 0.6
        return dict(op=op, P=P, B=B, C=C, dtype=rng.choice(['bf16', 'bf16', 'fp32']),
                    k=0 if train else min(C, rng.randint(0, 16)), masked=rng.random() < 0.4, train=train)
    P, width, layers = _log(rng, 1, 64), _log(rng, 8, 4096), rng.randint(1, 4)
    while P * layers * width * width > 2 ** 26:
        width = max(8, width * 2 // 3)
    return dict(op=op, P=P, d_in=_log(rng, 1, 1024), width=width, layers=layers, classes=_log(rng, 1, 1000),
                per_member=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs


def _shapes(case):
    P, w = case['P'], case['width']
    shapes = [(P, w, case['d_in']), (P, w)]
    shapes += [(P, w, w), (P, w)] * (case['layers'] - 1)
    return shapes + [(P, case['classes'], w), (P, case['classes'])]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=gen, device='cuda')  # noqa: E731
    normal = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    state = {'case': case}
    if case['op'] == 'norm':
        P, B, W = case['P'], case['B'], case['W']
        dt = DTYPES[case['dtype']]
        lead = (B,) if case['shared'] else (P, B)
        n = (torch.randint((W + 3) // 4, W + 1, (P,), generator=gen, device='cuda', dtype=torch.int32)
             if case['ragged'] else None)
        # activations after a linear layer: a mean of their own and a spread per row
        state['x'] = (normal(*lead, W) * (0.5 + rand(*lead, 1)) + 0.3 * normal(*lead, 1)).to(dt)
        state['n'] = n
        state['w'], state['b'] = 1 + 0.2 * normal(P, W), 0.2 * normal(P, W)
        if case['train']:
            state['dy'] = (normal(P, B, W) / B).to(dt)
        return state
    if case['op'] == 'labels':
        P, B, C = case['P'], case['B'], case['C']
        dt = DTYPES[case['dtype']]
        # the output layer's rows are padded to a multiple of eight columns: a bf16 pack's raw outputs
        ld = (C + 7) // 8 * 8 if dt == torch.bfloat16 else C
        logits = (normal(P, B, ld) * 2.5).to(dt)[..., :C]
        labels = torch.randint(0, C, (P, B), generator=gen, device='cuda')
        if case['masked']:
            off = torch.rand(logits.shape, generator=gen, device='cuda') < 0.3
            off.scatter_(-1, labels[..., None], False)
            logits.masked_fill_(off, -math.inf)
        state.update(logits=logits, labels=labels)
        if case['train']:
            # the gradients of a mean over rows: per-row weights of the label's term and of the entropy bonus
            state['g_l'] = -rand(P, B) / B
            state['g_h'] = -0.05 * rand(P, B) / B
        return state
    P = case['P']
    shapes = _shapes(case)
    state['params'], state['grads'] = [], []
    for s in ('exp_avgs', 'exp_avg_scales', 'exp_avg_sqs', 'exp_avg_sq_scales'):
        state[s] = []
    for shape in shapes:
        inner = math.prod(shape[1:])
        state['params'].append((2 * rand(*shape) - 1) * shape[-1] ** -0.5)
        # gradients whose size varies from element to element over a few orders of magnitude
        size = torch.exp(1.5 * normal(P, inner)) * 1e-3
        state['grads'].append((normal(P, inner) * size).view(shape))
        m, u = 0.3 * normal(P, inner) * size, size * (0.5 + rand(P, inner))
        r = torch.randint(0, 1 << 16, (P, inner), generator=gen, device='cuda')
        for name, (codes, scales) in (('exp_avg', _store_first(m, r)), ('exp_avg_sq', _store_root(u, r))):
            state[name + 's'].append(codes.view(shape))
            state[name + '_scales'].append(scales)
    state['seed'] = seed * 1_000_003 + 17
    if case['per_member']:
        state['step'] = torch.randint(1, 2000, (P,), generator=gen, device='cuda')
        state['hp'] = dict(lr=1e-3 * (0.3 + rand(P)), beta1=0.85 + 0.1 * rand(P), beta2=0.99 + 0.0095 * rand(P),
                           eps=1e-8, weight_decay=0.02 * rand(P))
    else:
        state['step'] = 40
        state['hp'] = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)
    return state


# ------------------------------------------------------------------ plain forms


def _norm_plain(s):
    case = s['case']
    P, B, W = case['P'], case['B'], case['W']
    x = s['x'].float().expand(P, B, W)
    n = torch.full((P,), W, device=x.device) if s['n'] is None else s['n']
    keep = torch.arange(W, device=x.device) < n[:, None, None]
    n = n[:, None, None].float()
    mean = torch.where(keep, x, 0).sum(-1, keepdim=True) / n
    d = torch.where(keep, x - mean, 0)
    rstd = 1 / torch.sqrt((d * d).sum(-1, keepdim=True) / n + EPS)
    xhat = d * rstd
    w, b = s['w'][:, None], s['b'][:, None]
    y = torch.where(keep, xhat * w + b, 0).to(s['x'].dtype)
    if not case['train']:
        return [y]
    dy = torch.where(keep, s['dy'].float(), 0)
    g = dy * w
    c1 = g.sum(-1, keepdim=True) / n
    c2 = (g * xhat).sum(-1, keepdim=True) / n
    dx = torch.where(keep, rstd * (g - c1 - xhat * c2), 0)
    if case['shared']:
        dx = dx.sum(0)
    return [y, dx.to(s['x'].dtype), (dy * xhat).sum(1), dy.sum(1)]


def _labels_plain(s):
    case = s['case']
    z = s['logits'].float()
    z = z - z.amax(-1, keepdim=True)
    logp = z - torch.log(torch.exp(z).sum(-1, keepdim=True))
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, 0)
    entropy = -plogp.sum(-1)
    out = [logp.gather(-1, s['labels'][..., None])[..., 0], entropy]
    if case['k']:
        top = torch.sort(s['logits'], dim=-1, descending=True, stable=True)[1][..., : case['k']]
        out += [logp.gather(-1, top), top]
    if case['train']:
        hot = torch.arange(case['C'], device=z.device) == s['labels'][..., None]
        dz = s['g_l'][..., None] * (hot.float() - p) - s['g_h'][..., None] * (plogp + p * entropy[..., None])
        out.append(dz.to(s['logits'].dtype))
    return out


def _blocks(x):
    """(P, inner) as (P, blocks, 128), zeros after the end."""
    P, inner = x.shape
    nb = (inner + BLOCK - 1) // BLOCK
    return torch.nn.functional.pad(x, (0, nb * BLOCK - inner)).view(P, nb, BLOCK)


def _scales(x, top):
    """Each block's scale: its largest magnitude over the code's largest value (0 where that is next to nothing)."""
    big = x.abs().amax(-1)
    return torch.where(big < 2.0 ** -100, 0.0, big / top)


def _inverse(scale):
    return torch.where(scale > 0, 1 / scale, 0.0)[..., None]


def _store_first(m, r):
    """(P, inner) first moments and 16 random bits each -> e4m3 codes and scales."""
    inner = m.shape[1]
    x, r = _blocks(m), _blocks(r).to(torch.int32)
    scale = _scales(x, 448.0)
    y = torch.clamp(x.abs() * _inverse(scale), max=448.0)
    normal = ((y.view(torch.int32) + (r << 4)) >> 20) - (120 << 3)
    small = torch.floor(y * 512 + r * 2.0 ** -16).to(torch.int32)
    code = torch.where(y >= 2.0 ** -6, normal, small) + torch.where(x < 0, 128, 0)
    code = torch.where(scale[..., None] > 0, code, 0)
    return code.to(torch.uint8).flatten(1)[:, :inner].contiguous(), scale


def _store_root(u, r):
    """(P, inner) roots of the second moments and 16 random bits each -> e4m4 codes and scales."""
    inner = u.shape[1]
    x, r = _blocks(u), _blocks(r).to(torch.int32)
    scale = _scales(x, 1.9375)
    y = torch.clamp(x * _inverse(scale), max=1.9375)
    code = torch.clamp(((y.view(torch.int32) + (r << 3)) >> 19) - (112 << 4), 1, 255)
    code = torch.where((x > 0) & (scale[..., None] > 0), code, 0)
    return code.to(torch.uint8).flatten(1)[:, :inner].contiguous(), scale


def _load_first(codes, scales):
    inner = codes[0].numel()
    return (_blocks(codes.flatten(1)).view(torch.float8_e4m3fn).float() * scales[..., None]).flatten(1)[:, :inner]


def _load_root(codes, scales):
    inner = codes[0].numel()
    c = _blocks(codes.flatten(1)).to(torch.int32)
    value = torch.where(c > 0, ((c + (112 << 4)) << 19).view(torch.float32), 0.0)
    return (value * scales[..., None]).flatten(1)[:, :inner]


def _philox(c0, c1, c2, c3, seed):
    """Philox4x32-10 of counters that broadcast together, int64 words below 2^32."""
    low = 0xFFFFFFFF
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), -1)


def _bits(P, inner, tensor, step, seed, device):
    """(P, inner) 32 random bits each."""
    groups = torch.arange((inner + 3) // 4, device=device)[None]
    member = torch.arange(P, device=device)[:, None]
    step = step[:, None] if isinstance(step, torch.Tensor) else torch.tensor(step, device=device)
    words = _philox(groups, torch.tensor(tensor, device=device), member, step, seed)
    return words.flatten(1)[:, :inner]


def _column(v):
    return v[:, None] if isinstance(v, torch.Tensor) else v


def _adamw8_tensor(s, i):
    p, g = s['params'][i].flatten(1), s['grads'][i].flatten(1)
    lr, b1, b2, eps, wd = (_column(s['hp'][k]) for k in ('lr', 'beta1', 'beta2', 'eps', 'weight_decay'))
    t = _column(s['step'])
    m = _load_first(s['exp_avgs'][i], s['exp_avg_scales'][i])
    u = _load_root(s['exp_avg_sqs'][i], s['exp_avg_sq_scales'][i])
    # 1 - b^t in 64 bits: next to 0 for the first steps
    bc1, bc2 = ((1 - torch.as_tensor(b, dtype=torch.float64, device=p.device) ** t).float() for b in (b1, b2))
    m = m * b1 + g * (1 - b1)
    u = torch.sqrt((u * u) * b2 + (g * g) * (1 - b2))
    p = p * (1 - lr * wd) - (lr / bc1) * m / (u / torch.sqrt(bc2) + eps)
    s['params'][i].copy_(p.view(s['params'][i].shape))
    words = _bits(*p.shape, i, s['step'], s['seed'], p.device)
    for name, (codes, scales) in (('exp_avg', _store_first(m, words & 0xFFFF)),
                                  ('exp_avg_sq', _store_root(u, words >> 16))):
        s[name + 's'][i].copy_(codes.view(s[name + 's'][i].shape))
        s[name + '_scales'][i].copy_(scales)


def _adamw8_plain(s):
    s['step'] = s['step'] + 1
    which = range(len(s['params']))
    for i in which:
        _adamw8_tensor(s, i)
    # the stored moments' values: a code has at most five significant bits, bf16 eight
    first = [_load_first(s['exp_avgs'][i], s['exp_avg_scales'][i]).bfloat16() for i in which]
    root = [_load_root(s['exp_avg_sqs'][i], s['exp_avg_sq_scales'][i]) for i in which]
    shape = [q.shape for q in s['params']]
    return [s['params'], [f.view(t) for f, t in zip(first, shape)],
            [(r * r).bfloat16().view(t) for r, t in zip(root, shape)]]


# ------------------------------------------------------------------ the framework's calls


def _norm_own(s):
    from tabpack_b200 import ops

    y, mean, rstd = ops.layer_norm_forward(s['x'], s['w'], s['b'], n_features=s['n'], eps=EPS)
    if not s['case']['train']:
        return [y]
    dx, dw, db = ops.layer_norm_backward(s['dy'], s['x'], s['w'], mean, rstd, n_features=s['n'])
    return [y, dx, dw, db]


def _labels_own(s):
    from tabpack_b200 import ops

    case = s['case']
    log_prob, entropy, top, which, stats = ops.label_log_probs_forward(s['logits'], s['labels'], top_k=case['k'])
    out = [log_prob, entropy]
    if case['k']:
        out += [top, which]
    if case['train']:
        out.append(ops.label_log_probs_backward(s['g_l'], s['g_h'], s['logits'], s['labels'], stats))
    return out


def _adamw8_own(s):
    from tabpack_b200 import ops

    moments = (s['exp_avgs'], s['exp_avg_scales'], s['exp_avg_sqs'], s['exp_avg_sq_scales'])
    if s['case']['per_member']:
        s['step'] = s['step'] + 1
        ops.adamw8_step(s['params'], s['grads'], *moments, steps=[s['step']] * len(s['params']), seed=s['seed'],
                        **s['hp'])
    else:
        s['step'] += 1
        ops.adamw8_step(s['params'], s['grads'], *moments, step=s['step'], seed=s['seed'], **s['hp'])
    first, second = ops.adamw8_moments(*moments, dtype=torch.bfloat16)
    return [s['params'], first, second]


def run(state):
    op = state['case']['op']
    if own:
        return {'norm': _norm_own, 'labels': _labels_own, 'adamw8': _adamw8_own}[op](state)
    return {'norm': _norm_plain, 'labels': _labels_plain, 'adamw8': _adamw8_plain}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case['op'] == 'norm':
        P, B, W = case['P'], case['B'], case['W']
        size = 2 if case['dtype'] == 'bf16' else 4
        x, y, par = (1 if case['shared'] else P) * B * W * size, P * B * W * size, P * W * 4
        if not case['train']:
            return {'bytes': x + y + 2 * par, 'flops': 8 * P * B * W}
        return {'bytes': x + y + y + x + 4 * par, 'flops': 22 * P * B * W}
    if case['op'] == 'labels':
        rows, C = case['P'] * case['B'], case['C']
        size = 2 if case['dtype'] == 'bf16' else 4
        n = rows * C * size + rows * (8 + 8) + rows * case['k'] * 12
        if case['train']:
            n += rows * C * size + rows * 8
        return {'bytes': n, 'flops': rows * C * (14 if case['train'] else 6)}
    n = sum(math.prod(s) for s in _shapes(case))
    # parameter read and written, gradient read, both codes read and written; the values returned as bf16
    return {'bytes': n * (8 + 4 + 4) + n * 4 + 16 * (n // BLOCK), 'flops': 25 * n}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {'norm': _norm_exact, 'labels': _labels_exact, 'adamw8': _adamw8_exact}[case['op']](s)


def _norm_exact(s):
    """Member by member, with autograd's gradients."""
    case = s['case']
    P, B, W = case['P'], case['B'], case['W']
    y, dx, dw, db = [], [], [], []
    for m in range(P):
        n = W if s['n'] is None else int(s['n'][m])
        x = (s['x'] if case['shared'] else s['x'][m])[:, :n].double().requires_grad_(case['train'])
        w, b = (s[k][m, :n].double().requires_grad_(case['train']) for k in ('w', 'b'))
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        out = (x - mean) * torch.rsqrt(var + EPS) * w + b
        wide = lambda t: torch.nn.functional.pad(t.detach(), (0, W - n))  # noqa: E731
        if case['train']:
            got = torch.autograd.grad(out, (x, w, b), s['dy'][m, :, :n].double())
            for to, t in zip((dx, dw, db), got):
                to.append(wide(t))
        y.append(wide(out))
    if not case['train']:
        return [torch.stack(y)]
    dx = torch.stack(dx)
    return [torch.stack(y), dx.sum(0) if case['shared'] else dx, torch.stack(dw), torch.stack(db)]


def _labels_exact(s):
    """In pieces of rows, from the softmax."""
    case = s['case']
    P, B, C = case['P'], case['B'], case['C']
    z, labels = s['logits'].reshape(P * B, C), s['labels'].reshape(-1)
    rows = max(1, 2 ** 26 // C)
    parts = []
    for i in range(0, P * B, rows):
        zi, li = z[i: i + rows].double(), labels[i: i + rows]
        p = torch.softmax(zi, -1)
        surprise = torch.logsumexp(zi, -1, keepdim=True) - zi
        h = torch.special.xlogy(p, p).sum(-1).neg()
        part = [-surprise.gather(-1, li[:, None])[:, 0], h]
        if case['k']:
            # a stable order over (value, position): one sort of the negated values
            top = torch.argsort(-zi, dim=-1, stable=True)[:, : case['k']]
            part += [-surprise.gather(-1, top), top]
        if case['train']:
            gl, gh = (s[k].reshape(-1)[i: i + rows, None].double() for k in ('g_l', 'g_h'))
            dz = -gl * p - gh * (torch.special.xlogy(p, p) + p * h[:, None])
            dz.scatter_add_(1, li[:, None], gl)
            # kept in 32 bits: a long case's gradient in 64 would be several GB
            part.append(dz.float())
        parts.append(part)
    return [torch.cat(t).view(P, B, *t[0].shape[1:]) for t in zip(*parts)]


def _random_words(counter, seed):
    """Philox4x32-10 (Salmon et al., 2011), round by round on a list of four words of counters."""
    mask = (1 << 32) - 1
    key = [seed & mask, (seed >> 32) & mask]
    x = list(counter)
    for r in range(10):
        k = [(key[j] + r * w) & mask for j, w in enumerate((0x9E3779B9, 0xBB67AE85))]
        # 32 x 32 -> 64 bits in halves of the multiplicand, so that no product leaves 63 bits
        wide = []
        for word, c in ((x[0], 0xD2511F53), (x[2], 0xCD9E8D57)):
            lo, hi = (word & 0xFFFF) * c, (word >> 16) * c
            mid = hi + (lo >> 16)
            wide.append((mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)))
        x = [wide[1][0] ^ x[1] ^ k[0], wide[1][1], wide[0][0] ^ x[3] ^ k[1], wide[0][1]]
    return x


def _adamw8_exact(s):
    case = s['case']
    P = case['P']
    step = s['step'] + 1
    f64 = lambda v: v.double()[:, None] if isinstance(v, torch.Tensor) else float(v)  # noqa: E731
    lr, b1, b2, eps, wd = (f64(s['hp'][k]) for k in ('lr', 'beta1', 'beta2', 'eps', 'weight_decay'))
    t = f64(step)
    out = [[], [], []]
    for i, shape in enumerate(_shapes(case)):
        inner = math.prod(shape[1:])
        at = torch.arange(inner, device='cuda')
        block = at // BLOCK
        # what the codes stand for
        code = s['exp_avgs'][i].view(P, inner).long()
        e, f = code >> 3 & 15, code & 7
        m = torch.where(e > 0, (8 + f) * 2.0 ** (e - 10).double(), f * 2.0 ** -9) * torch.where(code > 127, -1.0, 1.0)
        m = m * s['exp_avg_scales'][i].double()[:, block]
        code = s['exp_avg_sqs'][i].view(P, inner).long()
        u = torch.where(code > 0, (16 + code % 16) * 2.0 ** (code // 16 - 19).double(), 0.0)
        v = (u * s['exp_avg_sq_scales'][i].double()[:, block]) ** 2
        p, g = (s[k][i].view(P, inner).double() for k in ('params', 'grads'))
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        u = torch.sqrt(v)
        p = p - lr * wd * p - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
        zero = torch.zeros(1, 1, dtype=torch.int64, device='cuda')
        when = step[:, None] if isinstance(step, torch.Tensor) else zero + step
        group, member = at[None, : (inner + 3) // 4], torch.arange(P, device='cuda')[:, None]
        words = _random_words([group + zero, zero + i, member + zero, when], s['seed'])
        words = torch.stack([w.expand(P, (inner + 3) // 4) for w in words], -1).reshape(P, -1)[:, :inner]
        # a block's largest value is the code's largest; each value goes to a neighbour in the code's grid
        for x, top, digits, lowest, r, to, power in ((m, 448.0, 3, -6, words % 65536, 1, 1),
                                                     (u, 1.9375, 4, -15, words // 65536, 2, 2)):
            big = torch.zeros(P, int(block[-1]) + 1, dtype=torch.float64, device='cuda')
            big.scatter_reduce_(1, block.expand(P, -1), x.abs(), 'amax')
            scale = (big / top)[:, block]
            y = torch.where(scale > 0, x.abs() / scale, 0.0).clamp(max=top)
            grid = 2.0 ** (torch.frexp(y)[1].clamp(min=lowest + 1) - 1 - digits).double()
            y = torch.floor(y / grid + r / 65536.0) * grid
            if power == 2:
                # the roots have no values between 0 and the lowest code above 2^-15
                y = torch.where(x > 0, y.clamp(min=(1 + 1 / 16) * 2.0 ** lowest), 0.0)
            out[to].append((torch.sign(x) * y * scale).pow(power).view(shape))
        out[0].append(p.view(shape))
    return out
