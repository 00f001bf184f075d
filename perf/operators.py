"""Cases of the training operators: ``ops.linear_cross_entropy``, ``ops.orthogonalize`` and ``optim.muon_step_``.

``run`` computes a case through the package's operators where ``own`` is true, and in elementary torch operations where it is false.
``exact`` is the same in 64 bits, written from the definitions.

    linear_cross_entropy   z = scale * h w^T,  loss_i = log sum_v exp(z_iv) - z_i,t(i)  (0 where t(i) is ignored), with dh and dw
    orthogonalize          x = g / (|g|_F + eps);  five times  x = a x + (b s + c s s) x,  s = x x^T  (on the transpose of a tall matrix)
    muon_step_             m += (1 - mu)(g - m);  u = g + mu (m - g);  p = p (1 - lr wd) - lr sqrt(max(1, rows / cols)) orthogonalize(u)
"""
import math

import torch

own = False

IGNORED = -100
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}

# 3x3 convolution weights of the flow network (pyramid encoder, five decoder levels, context network): (output, input channels, how many)
FLOW_NETWORK = ((16, 3, 1), (16, 16, 1), (32, 16, 1), (32, 32, 1), (64, 32, 1), (64, 64, 1), (96, 64, 1), (96, 96, 1), (128, 96, 1),
                (128, 128, 8), (196, 128, 1), (196, 196, 1), (128, 81, 1), (96, 256, 5), (64, 224, 5), (32, 160, 5), (2, 96, 5),
                (128, 211, 1), (128, 179, 1), (128, 147, 1), (128, 115, 1), (128, 34, 1), (96, 128, 1), (64, 96, 1), (32, 64, 1), (2, 32, 1))


def _lce(name, rows, vocab, dim, dtype, train, reduction, scale=1.0, ignored=0.0):
    return {'name': name, 'op': 'linear_cross_entropy', 'rows': rows, 'vocab': vocab, 'dim': dim, 'dtype': dtype, 'train': train,
            'reduction': reduction, 'scale': scale, 'ignored': ignored}


def listed():
    return [
        # the log-probability of one next token
        _lce('score_token_bf16', 1, 32000, 2048, 'bf16', False, 'none'),
        # a ragged handful of continuations scored together
        _lce('score_batch_fp16', 61, 50257, 1024, 'fp16', False, 'none'),
        # positions of one frame against all positions of the next, feature maps of levels 4 and 3 at 832 x 256, 30 % occluded
        _lce('match_level4_fp32', 832, 832, 96, 'fp32', True, 'mean', 1 / 0.07, 0.3),
        _lce('match_level3_fp32', 3328, 3328, 64, 'fp32', True, 'mean', 1 / 0.07, 0.3),
        # odd sizes, a weight of its own for every row
        _lce('train_ragged_fp32', 1013, 10007, 777, 'fp32', True, 'none', 1.0, 0.1),
        # one micro-batch of a middle-sized and of a large language model
        _lce('train_bf16', 4096, 32000, 2048, 'bf16', True, 'mean', 1.0, 0.1),
        _lce('train_large_bf16', 8192, 131072, 4096, 'bf16', True, 'sum', 1.0, 0.02),
        # the eight equal convolutions of the flow network at once
        {'name': 'orthogonalize_conv_fp32', 'op': 'orthogonalize', 'batch': 8, 'rows': 128, 'cols': 1152, 'dtype': 'fp32'},
        # a pair of tall projections, and one large square matrix
        {'name': 'orthogonalize_tall_fp32', 'op': 'orthogonalize', 'batch': 2, 'rows': 4096, 'cols': 1024, 'dtype': 'fp32'},
        {'name': 'orthogonalize_square_bf16', 'op': 'orthogonalize', 'batch': 1, 'rows': 4096, 'cols': 4096, 'dtype': 'bf16'},
        # one optimiser step of the flow network's weights, and of four transformer blocks of width 1024
        {'name': 'muon_flow_network_fp32', 'op': 'muon', 'network': 'flow', 'width': 128, 'layers': 1, 'dtype': 'fp32'},
        {'name': 'muon_blocks_bf16', 'op': 'muon', 'network': 'blocks', 'width': 1024, 'layers': 4, 'dtype': 'bf16'},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(('score', 'train', 'match', 'orthogonalize', 'muon'))
    dtype = rng.choice(('fp32', 'bf16', 'fp16'))
    if kind == 'score':
        c = _lce('', _spread(rng, 1, 512), _spread(rng, 500, 131072), _spread(rng, 32, 4096), dtype, False, 'none')
    elif kind == 'train':
        c = _lce('', _spread(rng, 16, 8192), _spread(rng, 500, 65536), _spread(rng, 32, 4096), dtype, True,
                 rng.choice(('mean', 'sum', 'none')), 1.0, rng.choice((0.0, 0.1, 0.5)))
    elif kind == 'match':
        n = rng.randint(4, 72) * rng.randint(8, 180)
        c = _lce('', n, n, rng.choice((32, 64, 96, 128, 196)), rng.choice(('fp32', 'bf16')), True, 'mean', 1 / 0.07, rng.choice((0.1, 0.3)))
    elif kind == 'orthogonalize':
        rows, cols = _spread(rng, 8, 4096), _spread(rng, 8, 4096)
        c = {'op': 'orthogonalize', 'batch': rng.randint(1, max(1, min(16, (1 << 24) // (rows * cols)))), 'rows': rows, 'cols': cols, 'dtype': dtype}
    else:
        network = rng.choice(('flow', 'blocks'))
        c = {'op': 'muon', 'network': network, 'width': _spread(rng, 24, 256) if network == 'flow' else _spread(rng, 64, 1024),
             'layers': rng.randint(1, 4), 'dtype': dtype}
    c.pop('name', None)
    return c


def _shapes(case):
    """The weights of a network: convolutions as (out, in, 3, 3), projections as (out, in)."""
    w = case['width']
    if case['network'] == 'flow':
        return [(max(2, o * w // 128), max(2, i * w // 128), 3, 3) for o, i, n in FLOW_NETWORK for _ in range(n)]
    return [s for _ in range(case['layers']) for s in ((w, w), (w, w), (w, w), (w, w), (4 * w, w), (w, 4 * w))]


def _gradient(rows, cols, gen, batch=None):
    """What a gradient looks like: a few strong directions over a floor of noise."""
    lead = () if batch is None else (batch,)
    rank = max(1, min(rows, cols) // 8)
    n = lambda *s: torch.randn(*lead, *s, generator=gen, device='cuda')  # noqa: E731
    strong = n(rows, rank) * torch.linspace(1.0, 0.1, rank, device='cuda') @ n(rank, cols)
    return 1e-3 * (strong / math.sqrt(rank) + 0.3 * n(rows, cols))


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    if case['op'] == 'linear_cross_entropy':
        n, v, d = case['rows'], case['vocab'], case['dim']
        weight = torch.randn(v, d, generator=gen, device='cuda')
        target = torch.randint(v, (n,), generator=gen, device='cuda')
        if case['scale'] == 1.0:        # final hidden states and an output embedding: logits of a few units, the target's somewhat larger
            weight *= 1.3 / math.sqrt(d)
            hidden = torch.randn(n, d, generator=gen, device='cuda') + 3 * weight[target]
        else:                           # unit feature vectors, a position's match being near to it
            weight /= weight.norm(dim=1, keepdim=True)
            hidden = weight[target] + 0.7 / math.sqrt(d) * torch.randn(n, d, generator=gen, device='cuda')
            hidden /= hidden.norm(dim=1, keepdim=True)
        target[torch.rand(n, generator=gen, device='cuda') < case['ignored']] = IGNORED
        # (a mean's gradients are below what 16 bits with 5 of exponent hold: such a run scales its loss)
        upstream = torch.full((), 4096.0 if dtype == torch.float16 and case['reduction'] != 'sum' else 1.0, device='cuda')
        if case['reduction'] == 'none':
            upstream = upstream / n * torch.rand(n, generator=gen, device='cuda')
        return {'case': case, 'hidden': hidden.to(dtype).requires_grad_(case['train']), 'weight': weight.to(dtype).requires_grad_(case['train']),
                'target': target, 'upstream': upstream}
    if case['op'] == 'orthogonalize':
        return {'case': case, 'x': _gradient(case['rows'], case['cols'], gen, case['batch']).to(dtype)}
    params, grads = [], []
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    buffer = torch.zeros(sum(sizes), device='cuda')
    momenta = []
    for shape, size, part in zip(shapes, sizes, buffer.split(sizes)):
        cols = size // shape[0]
        p = torch.randn(shape, generator=gen, device='cuda') / math.sqrt(cols)
        g = _gradient(shape[0], cols, gen).view(shape)
        m = _gradient(shape[0], cols, gen).view(shape)
        if len(shape) == 4:             # the flow network keeps its convolution weights in channels_last order
            p, g, m = (t.contiguous(memory_format=torch.channels_last) for t in (p, g, m))
        view = part.as_strided(shape, p.stride())
        view.copy_(m)
        params.append(p.to(dtype))
        grads.append(g.to(dtype))
        momenta.append(view)
    return {'case': case, 'params': params, 'grads': grads, 'momenta': momenta, 'buffer': buffer}


def _plain_orthogonalize(x):
    a, b, c = COEFFICIENTS
    rows, cols = x.shape[-2:]
    x = x.mT if rows > cols else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if rows > cols else x


def _plain_loss(case, hidden, weight, target, upstream):
    h, w = hidden.float(), weight.float()
    valid = target != IGNORED
    count = valid.sum().clamp(min=1)
    row = torch.arange(len(target), device=target.device)
    at = target.where(valid, 0)
    z = case['scale'] * (h @ w.T)
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    losses = ((total.log() + top).squeeze(1) - z[row, at]).where(valid, 0)
    loss = losses if case['reduction'] == 'none' else losses.sum() / count if case['reduction'] == 'mean' else losses.sum()
    if not case['train']:
        return {'loss': loss}
    g = upstream / count if case['reduction'] == 'mean' else upstream
    g = (case['scale'] * g * valid).unsqueeze(1)
    p = e / total
    p[row, at] -= 1
    p *= g
    return {'loss': loss, 'dhidden': (p @ w).to(hidden.dtype), 'dweight': (p.T @ h).to(weight.dtype)}


def _plain_muon(params, grads, momenta):
    for p, g, m in zip(params, grads, momenta):
        g32 = g.float()
        m.add_((1 - MOMENTUM) * (g32 - m))
        u = g32 + MOMENTUM * (m - g32)
        o = _plain_orthogonalize(u.reshape(len(u), -1))
        lr = LR * math.sqrt(max(1.0, o.shape[0] / o.shape[1]))
        p.copy_(p.float() * (1 - LR * DECAY) - lr * o.view(p.shape))


def run(state):
    case = state['case']
    if case['op'] == 'linear_cross_entropy':
        h, w, target = state['hidden'], state['weight'], state['target']
        if own:
            from unopticalflow_amd import ops
            loss = ops.linear_cross_entropy(h, w, target, ignore_index=IGNORED, scale=case['scale'], reduction=case['reduction'])
            if not case['train']:
                return {'loss': loss}
            dh, dw = torch.autograd.grad(loss, (h, w), state['upstream'])
            return {'loss': loss.detach(), 'dhidden': dh, 'dweight': dw}
        with torch.no_grad():
            return _plain_loss(case, h, w, target, state['upstream'])
    if case['op'] == 'orthogonalize':
        if own:
            from unopticalflow_amd import ops
            return ops.orthogonalize(state['x'], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        return _plain_orthogonalize(state['x'].float()).to(state['x'].dtype)
    if own:
        from unopticalflow_amd import optim
        optim.muon_step_(state['params'], state['grads'], state['momenta'], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, nesterov=True,
                         steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    else:
        _plain_muon(state['params'], state['grads'], state['momenta'])
    return {'params': state['params'], 'momenta': state['buffer']}


def _orthogonalize_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m * m * m + 2 * m * m * n)      # x x^T and s s are symmetric: half of each suffices


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'linear_cross_entropy':
        n, v, d = case['rows'], case['vocab'], case['dim']
        times = 2 if case['train'] else 1
        return {'bytes': times * (n + v) * d * size + 8 * n + (4 * n if case['reduction'] == 'none' else 4), 'flops': (6 if case['train'] else 2) * n * v * d}
    if case['op'] == 'orthogonalize':
        b, r, c = case['batch'], case['rows'], case['cols']
        return {'bytes': 2 * b * r * c * size, 'flops': b * _orthogonalize_flops(r, c)}
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    return {'bytes': sum(sizes) * (3 * size + 8), 'flops': sum(_orthogonalize_flops(s[0], n // s[0]) for s, n in zip(shapes, sizes))}


def _exact_orthogonalize(g):
    """The polynomial p(s) = a s + b s^3 + c s^5, five times, on the left factor of g / (|g| + eps): x <- x (a + b x^T x + c (x^T x)^2) is the same map."""
    a, b, c = COEFFICIENTS
    x = g / (torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True) + EPS)
    wide = g.shape[-1] > g.shape[-2]
    eye = torch.eye(min(g.shape[-2:]), dtype=torch.float64, device=g.device)
    for _ in range(STEPS):
        t = torch.matmul(x, x.transpose(-2, -1).contiguous()) if wide else torch.matmul(x.transpose(-2, -1).contiguous(), x)
        q = a * eye + torch.matmul(t, b * eye + c * t)
        x = torch.matmul(q, x) if wide else torch.matmul(x, q)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'linear_cross_entropy':
        h, w, target = s['hidden'].detach().double(), s['weight'].detach().double(), s['target']
        valid = target != IGNORED
        z = torch.matmul(h, w.t()) * case['scale']
        lse = torch.logsumexp(z, 1)
        at = target.clamp(min=0)
        losses = torch.where(valid, lse - z.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
        n = max(1, int(valid.sum()))
        loss = {'none': losses, 'sum': losses.sum(), 'mean': losses.sum() / n}[case['reduction']]
        if not case['train']:
            return {'loss': loss}
        z = torch.softmax(z, 1)
        z.scatter_add_(1, at[:, None], torch.full_like(z[:, :1], -1.0))
        z *= (s['upstream'].double() * valid * case['scale'] / (n if case['reduction'] == 'mean' else 1))[:, None]
        return {'loss': loss, 'dhidden': torch.matmul(z, w), 'dweight': torch.matmul(z.t().contiguous(), h)}
    if case['op'] == 'orthogonalize':
        return _exact_orthogonalize(s['x'].double())
    params, buffer = [], []
    for p, g, m in zip(s['params'], s['grads'], s['momenta']):
        new = MOMENTUM * m.double() + (1 - MOMENTUM) * g.double()
        u = (1 - MOMENTUM) * g.double() + MOMENTUM * new
        o = _exact_orthogonalize(u.flatten(1))
        params.append((1 - LR * DECAY) * p.double() - LR * max(1.0, o.shape[0] / o.shape[1]) ** 0.5 * o.view_as(p))
        buffer.append(torch.empty_like(m, dtype=torch.float64).copy_(new).as_strided((m.numel(),), (1,)))
    return {'params': params, 'momenta': torch.cat(buffer)}
