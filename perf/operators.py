"""Cases and plain forms of the attention-block operators over active sites
(``bevfusion_triton_b200.ops.spconv``): ``packed_attention``,
``qk_norm_rotary`` and ``residual_dropout``.

``run`` computes a case in its plain form (elementary torch operations in
fp32) or, with ``own`` set, through the framework's operators; ``exact``
gives the same outputs from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}
BYTES = {'fp32': 4, 'fp16': 2, 'bf16': 2}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # decoder queries of six camera views attending within their view: the latency of one small call
        {'name': 'attention views', 'op': 'attention', 'dtype': 'fp16', 'heads': 8, 'kv_heads': 8, 'dim': 16,
         'causal': False, 'train': False, 'cache': False, 'seqs': 6, 'shortest': 20, 'longest': 200, 'queries': 0,
         'shape': 1, 'spare': 0},
        # voxels grouped by window, the usual voxel-transformer layer: many short ragged sequences
        {'name': 'attention windows', 'op': 'attention', 'dtype': 'bf16', 'heads': 8, 'kv_heads': 8, 'dim': 32,
         'causal': False, 'train': False, 'cache': False, 'seqs': 64, 'shortest': 1, 'longest': 900, 'queries': 0,
         'shape': 2, 'spare': 37},
        # one packed prompt of scans in serialised order, causal, four query heads to a key head
        {'name': 'attention prompt', 'op': 'attention', 'dtype': 'bf16', 'heads': 16, 'kv_heads': 4, 'dim': 128,
         'causal': True, 'train': False, 'cache': False, 'seqs': 4, 'shortest': 1500, 'longest': 6001, 'queries': 0,
         'shape': 3, 'spare': 0},
        # every cell of a 180 x 90 BEV map against every other
        {'name': 'attention bev map', 'op': 'attention', 'dtype': 'fp16', 'heads': 8, 'kv_heads': 8, 'dim': 64,
         'causal': False, 'train': False, 'cache': False, 'seqs': 1, 'shortest': 16200, 'longest': 16200,
         'queries': 0, 'shape': 4, 'spare': 0},
        # serving a stream: the newest token of each of 24 streams against its cache
        {'name': 'attention stream', 'op': 'attention', 'dtype': 'bf16', 'heads': 32, 'kv_heads': 8, 'dim': 128,
         'causal': True, 'train': False, 'cache': True, 'seqs': 24, 'shortest': 1, 'longest': 30001, 'queries': 1,
         'shape': 5, 'spare': 0},
        # a training step over packed sequences, causal, shared key heads
        {'name': 'attention train prompt', 'op': 'attention', 'dtype': 'bf16', 'heads': 16, 'kv_heads': 4,
         'dim': 128, 'causal': True, 'train': True, 'cache': False, 'seqs': 4, 'shortest': 700, 'longest': 4096,
         'queries': 0, 'shape': 6, 'spare': 0},
        # a training step over the voxels of a batch, each sample one sequence
        {'name': 'attention train voxels', 'op': 'attention', 'dtype': 'fp16', 'heads': 8, 'kv_heads': 8, 'dim': 64,
         'causal': False, 'train': True, 'cache': False, 'seqs': 8, 'shortest': 300, 'longest': 2500, 'queries': 0,
         'shape': 7, 'spare': 11},
        # queries and keys of the active voxels of a batch, positions (z, y, x)
        {'name': 'rotary voxels', 'op': 'rotary', 'dtype': 'bf16', 'heads': 8, 'kv_heads': 8, 'dim': 64,
         'axes': 3, 'rotated': 64, 'tokens': 90001, 'interleaved': False, 'norm': True, 'positions': 'int32',
         'reach': 1440, 'train': False},
        # the same in a training step with shared key heads: gradients of both and of the norms' weights
        {'name': 'rotary train', 'op': 'rotary', 'dtype': 'bf16', 'heads': 16, 'kv_heads': 4, 'dim': 128,
         'axes': 3, 'rotated': 128, 'tokens': 24003, 'interleaved': False, 'norm': True, 'positions': 'float32',
         'reach': 200000, 'train': True},
        # serving: one token for each of 24 streams
        {'name': 'rotary token', 'op': 'rotary', 'dtype': 'bf16', 'heads': 32, 'kv_heads': 8, 'dim': 128,
         'axes': 1, 'rotated': 128, 'tokens': 24, 'interleaved': True, 'norm': True, 'positions': 'int32',
         'reach': 1000000, 'train': False},
        # a block's output onto the residual stream, a training step over the voxels of a batch
        {'name': 'dropout train', 'op': 'dropout', 'dtype': 'bf16', 'rows': 90001, 'width': 512, 'p': 0.1,
         'residual': True, 'train': True},
        # the same for one sample's decoder queries in fp32, forward only
        {'name': 'dropout queries', 'op': 'dropout', 'dtype': 'fp32', 'rows': 601, 'width': 128, 'p': 0.25,
         'residual': True, 'train': False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'attention', 'attention', 'rotary', 'rotary', 'dropout'])
    if op == 'rotary':
        kv = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([16, 32, 48, 64, 80, 96, 128, 256])
        interleaved = rng.random() < 0.5
        rotated = rng.choice([dim, dim, 16 * rng.randint(1, dim // 16)])
        heads = kv * rng.choice([1, 1, 2, 4, 5])
        return {'op': op, 'dtype': rng.choice(['bf16', 'fp16', 'fp32']), 'heads': heads, 'kv_heads': kv, 'dim': dim,
                'axes': rng.choice([1, 2, 3, 4]), 'rotated': rotated,
                'tokens': _log(rng, 1, max(2, 30_000_000 // ((heads + kv) * dim))), 'interleaved': interleaved,
                'norm': rng.random() < 0.8, 'positions': rng.choice(['int32', 'int64', 'float32']),
                'reach': _log(rng, 100, 2_000_000), 'train': rng.random() < 0.5}
    if op == 'dropout':
        return {'op': op, 'dtype': rng.choice(['bf16', 'fp16', 'fp32']), 'rows': _log(rng, 1, 44000),
                'width': rng.choice([1, 80, 128, 131, 256, 512]), 'p': round(rng.uniform(0.0, 0.7), 3),
                'residual': rng.random() < 0.7, 'train': rng.random() < 0.6}
    kind = rng.choice(['encode', 'stream', 'train'])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4, 7])
    dim = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128])
    case = {'op': op, 'dtype': rng.choice(['bf16', 'fp16']), 'heads': heads, 'kv_heads': kv, 'dim': dim,
            'causal': rng.random() < 0.5, 'train': kind == 'train', 'cache': kind == 'stream',
            'seqs': _log(rng, 1, 48), 'shortest': rng.choice([0, 1, 1, 30]), 'longest': 0, 'queries': 0,
            'shape': rng.randrange(1 << 20), 'spare': rng.choice([0, 0, 1, 200])}
    if kind == 'stream':
        case['queries'] = rng.choice([1, 1, 1, 2, 5])
        most = 300_000_000 // (case['seqs'] * kv * dim)  # values in each cache
        case['longest'] = _log(rng, 1, max(2, min(60000, most)))
    else:
        if rng.random() < 0.3:
            case['queries'] = _log(rng, 1, 600)  # queries of their own: cross attention
        most = (0.28e9 if kind == 'train' else 1.2e9) / (case['seqs'] * heads)  # entries of a padded score matrix
        longest = most / case['queries'] if case['queries'] else math.sqrt(most)
        case['longest'] = _log(rng, 1, max(2, min(9000, int(longest))))
    case['shortest'] = min(case['shortest'], case['longest'])
    return case


def _lengths(case):
    """Queries, keys and key capacity of each sequence."""
    rng = random.Random(case['shape'])
    lo, hi = case['shortest'], case['longest']
    keys = [hi] + [lo if lo == hi else min(hi, max(lo, _log(rng, max(lo, 0.7), hi))) for _ in range(case['seqs'] - 1)]
    rng.shuffle(keys)
    room = [hi] * len(keys) if case['cache'] else keys
    if case['cache']:
        queries = [case['queries']] * len(keys)
    elif case['queries']:
        queries = [rng.randint(0, case['queries']) for _ in keys]
        queries[rng.randrange(len(keys))] = case['queries']
    else:
        queries = list(keys)
    return queries, keys, room


def _pairs(nq, nk, causal):
    """Pairs of a query and a key it sees, in one sequence."""
    if not causal:
        return nq * nk
    most, least = nk, max(0, nk - nq + 1)  # keys of the last query and of the first that sees any
    seeing = min(nq, nk)
    return seeing * (most + least if nq <= nk else nk + 1) // 2


def work(case):
    size = BYTES[case['dtype']]
    if case['op'] == 'attention':
        queries, keys, _ = _lengths(case)
        d = case['dim']
        pairs = sum(_pairs(a, b, case['causal']) for a, b in zip(queries, keys)) * case['heads']
        nq, nk = (sum(queries) + case['spare']) * case['heads'] * d, sum(keys) * case['kv_heads'] * d
        if case['train']:
            return {'bytes': size * (4 * nq + 4 * nk), 'flops': 14 * d * pairs}
        return {'bytes': size * (2 * nq + 2 * nk), 'flops': 4 * d * pairs}
    if case['op'] == 'rotary':
        n = case['tokens'] * (case['heads'] + case['kv_heads']) * case['dim']
        place = {'int32': 4, 'float32': 4, 'int64': 8}[case['positions']] * case['tokens'] * case['axes']
        return {'bytes': size * n * (4 if case['train'] else 2) + place, 'flops': n * (22 if case['train'] else 8)}
    n = case['rows'] * case['width']
    moved = 2 + case['residual'] + (2 if case['train'] else 0)
    return {'bytes': size * n * moved, 'flops': n * (4 if case['train'] else 2)}


# -------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device='cuda') * scale).to(dtype)


def _starts(lengths):
    total, at = 0, [0]
    for n in lengths:
        total += n
        at.append(total)
    return at


def _sections(case):
    """Frequencies of each axis: near equal shares, the first the smallest."""
    pairs, axes = case['rotated'] // 2, case['axes']
    return tuple(pairs // axes + (1 if a >= axes - pairs % axes else 0) for a in range(axes))


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case['dtype']]
    state = {'case': dict(case)}
    if case['op'] == 'attention':
        queries, keys, room = _lengths(case)
        d = case['dim']
        nq, nk = sum(queries) + case['spare'], sum(room) + (0 if case['cache'] else case['spare'])
        qkv = [_normal(g, (nq, case['heads'], d), dtype, 1.5), _normal(g, (nk, case['kv_heads'], d), dtype),
               _normal(g, (nk, case['kv_heads'], d), dtype)]
        if case['train']:
            qkv = [t.requires_grad_(True) for t in qkv]
            state['grad'] = _normal(g, (nq, case['heads'], d), dtype)
        starts_q, starts_k = _starts(queries), _starts(room)
        state.update(q=qkv[0], k=qkv[1], v=qkv[2], scale=d ** -0.5, most_q=max(queries), most_k=max(keys),
                     cu_q=torch.tensor(starts_q, dtype=torch.int32, device='cuda'),
                     cu_k=torch.tensor(starts_k, dtype=torch.int32, device='cuda'),
                     lengths=torch.tensor(keys, dtype=torch.int32, device='cuda') if case['cache'] else None)
    elif case['op'] == 'rotary':
        n, d = case['tokens'], case['dim']
        q = _normal(g, (n, case['heads'], d), dtype, 3.0)
        k = _normal(g, (n, case['kv_heads'], d), dtype, 2.0)
        where = torch.rand((n, case['axes']), generator=g, device='cuda', dtype=torch.float64) * case['reach']
        where = where.to(torch.float32) if case['positions'] == 'float32' else where.floor().to(
            getattr(torch, case['positions']))
        half = case['rotated'] // 2
        inv_freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device='cuda') / half)
        state.update(q=q, k=k, positions=where, inv_freq=inv_freq.float(), sections=_sections(case), qw=None, kw=None)
        if case['norm']:
            state['qw'] = 1 + _normal(g, (d,), torch.float32, 0.1)
            state['kw'] = 1 + _normal(g, (d,), torch.float32, 0.1)
        if case['train']:
            state['gq'], state['gk'] = _normal(g, q.shape, dtype), _normal(g, k.shape, dtype)
            state['leaves'] = [t.requires_grad_(True) for t in (q, k, state['qw'], state['kw']) if t is not None]
    else:
        shape = (case['rows'], case['width'])
        state['x'] = _normal(g, shape, dtype)
        state['residual'] = _normal(g, shape, dtype, 2.0) if case['residual'] else None
        state['seed'] = torch.randint(-(1 << 62), 1 << 62, (2,), generator=g, device='cuda')
        if case['train']:
            state['grad'] = _normal(g, shape, dtype)
            state['leaves'] = [t.requires_grad_(True) for t in (state['x'], state['residual']) if t is not None]
    return state


# --------------------------------------------------------------- plain forms
def _padded(rows, starts, lengths, most):
    """[rows, H, D] -> [sequences, H, most, D] fp32, zeros behind each sequence; and where the rows went."""
    at = torch.arange(most, device=rows.device)
    there = at[None, :] < lengths[:, None]
    index = torch.where(there, starts[:, None].long() + at[None, :], 0)
    padded = torch.where(there[:, :, None, None], rows.detach()[index].float(), 0.0)
    return padded.transpose(1, 2), index, there


def _packed(padded, index, there, like):
    """Back to rows; rows of no sequence are zeros."""
    out = torch.zeros_like(like, requires_grad=False)
    out[index[there]] = padded.transpose(1, 2)[there].to(out.dtype)
    return out


def _plain_attention(s):
    c = s['case']
    nq = s['cu_q'][1:] - s['cu_q'][:-1]
    nk = s['lengths'] if s['lengths'] is not None else s['cu_k'][1:] - s['cu_k'][:-1]
    q, iq, hq = _padded(s['q'], s['cu_q'][:-1], nq, s['most_q'])
    k, ik, hk = _padded(s['k'], s['cu_k'][:-1], nk, s['most_k'])
    v, _, _ = _padded(s['v'], s['cu_k'][:-1], nk, s['most_k'])
    n, heads, rows, d = q.shape
    group = heads // c['kv_heads']
    q = q.reshape(n, c['kv_heads'], group * rows, d)
    sees = hk[:, None, None, None, :]
    if c['causal']:
        i, j = torch.arange(rows, device=q.device), torch.arange(s['most_k'], device=q.device)
        sees = sees & (j[None, None, :] <= i[None, :, None] + (nk - nq)[:, None, None])[:, None, None]
    score = (q @ k.transpose(-1, -2) * s['scale']).view(n, c['kv_heads'], group, rows, -1)
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, 1.0)).view(n, c['kv_heads'], group * rows, -1)
    out = p @ v
    spread = lambda x: _packed(x.view(n, heads, rows, d), iq, hq, s['q'])  # noqa: E731
    if not c['train']:
        if not c['cache']:
            return spread(out)
        lse = torch.where(total > 0, top + total.log(), -math.inf).view(n, heads, rows).transpose(1, 2)
        full = torch.full((s['q'].shape[0], heads), -math.inf, device=q.device)
        full[iq[hq]] = lse[hq]
        return spread(out), full.t().contiguous()
    g = _padded(s['grad'], s['cu_q'][:-1], nq, s['most_q'])[0].reshape(n, c['kv_heads'], group * rows, d)
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - (g * out).sum(-1, keepdim=True)) * s['scale']
    back = lambda x: _packed(x, ik, hk, s['k'])  # noqa: E731
    return (spread(out), spread(ds @ k), back(ds.transpose(-1, -2) @ q), back(p.transpose(-1, -2) @ g))


def _turn(x, cos, sin, rotated, interleaved):
    """Rotates pairs of the first `rotated` values: (i, i + half), or neighbours."""
    half = rotated // 2
    if interleaved:
        a, b = x[..., 0:rotated:2], x[..., 1:rotated:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rotated]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rotated:]], -1)


def _plain_rotary(s):
    c = s['case']
    axis = torch.repeat_interleave(torch.arange(c['axes'], device='cuda'),
                                   torch.tensor(s['sections'], device='cuda'), output_size=c['rotated'] // 2)
    angle = s['positions'].double()[:, axis] * s['inv_freq'].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def forward(x, w):
        x = x.detach().float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.detach()
        return _turn(x, cos, sin, c['rotated'], c['interleaved']).to(s['q'].dtype)

    def backward(x, w, g):
        g = _turn(g.float(), cos, -sin, c['rotated'], c['interleaved'])
        if w is None:
            return g.to(x.dtype), None
        x = x.detach().float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        unit = x * r
        gw = (g * unit).sum((0, 1), dtype=torch.float64).float()
        g = g * w.detach()
        return (r * (g - unit * (g * unit).mean(-1, keepdim=True))).to(s['q'].dtype), gw

    outs = [forward(s['q'], s['qw']), forward(s['k'], s['kw'])]
    if c['train']:
        dq, dqw = backward(s['q'], s['qw'], s['gq'])
        dk, dkw = backward(s['k'], s['kw'], s['gk'])
        outs += [t for t in (dq, dk, dqw, dkw) if t is not None]
    return outs


LOW = 0xffffffff


def _product(a, b):
    """High and low words of a 32 x 32 bit product, in 64-bit integers."""
    p = a * b
    return (p >> 32) & LOW, p & LOW


def _plain_words(n, seed):
    """Word i % 4 of Philox 4x32-10 at counter (i // 4, offset) for element i."""
    block = torch.arange((n + 3) // 4, device=seed.device)
    w = [block & LOW, block >> 32, (seed[1] & LOW).expand_as(block), ((seed[1] >> 32) & LOW).expand_as(block)]
    key = [seed[0] & LOW, (seed[0] >> 32) & LOW]
    for _ in range(10):
        h0, l0 = _product(w[0], 0xD2511F53)
        h1, l1 = _product(w[2], 0xCD9E8D57)
        w = [h1 ^ w[1] ^ key[0], l1, h0 ^ w[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & LOW, (key[1] + 0xBB67AE85) & LOW]
    return torch.stack(w, 1).flatten()[:n]


def _plain_dropout(s):
    c = s['case']
    x = s['x'].detach()
    keep = (_plain_words(x.numel(), s['seed']) >= int(c['p'] * 2.0 ** 32)).view_as(x)
    scale = 1.0 / (1.0 - c['p'])
    y = torch.where(keep, x.float() * scale, 0.0)
    if s['residual'] is not None:
        y = y + s['residual'].detach().float()
    if not c['train']:
        return y.to(x.dtype)
    outs = [y.to(x.dtype), torch.where(keep, s['grad'].float() * scale, 0.0).to(x.dtype)]
    return outs + ([s['grad']] if s['residual'] is not None else [])


# ------------------------------------------------------- the framework's calls
def _own(s):
    from bevfusion_triton_b200.ops.spconv import packed_attention, qk_norm_rotary, residual_dropout
    c = s['case']
    if c['op'] == 'attention':
        got = packed_attention(s['q'], s['k'], s['v'], s['cu_q'], s['cu_k'], kv_lengths=s['lengths'],
                               causal=c['causal'], scale=s['scale'], return_lse=c['cache'])
        if not c['train']:
            return got
        return (got.detach(), *torch.autograd.grad(got, (s['q'], s['k'], s['v']), s['grad']))
    if c['op'] == 'rotary':
        q, k = qk_norm_rotary(s['q'], s['k'], s['positions'], s['inv_freq'], s['sections'], s['qw'], s['kw'],
                              eps=1e-6, interleaved=c['interleaved'])
        if not c['train']:
            return [q, k]
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), s['leaves'], (s['gq'], s['gk']))]
    y = residual_dropout(s['x'], s['residual'], c['p'], s['seed'])
    return [y.detach(), *torch.autograd.grad(y, s['leaves'], s['grad'])] if c['train'] else y


def run(state):
    if own:
        return _own(state)
    return {'attention': _plain_attention, 'rotary': _plain_rotary, 'dropout': _plain_dropout}[state['case']['op']](
        state)


# ------------------------------------------------------------------ 64 bits
def _exact_attention(s):
    """Sequence by sequence and head by head; gradients by differentiating the definition."""
    c = s['case']
    queries, keys, room = _lengths(c)
    at_q, at_k = _starts(queries), _starts(room)
    train = c['train']
    q, k, v = (s[n].detach().double() for n in 'qkv')
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device='cuda')
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    for n, (nq, nk) in enumerate(zip(queries, keys)):
        if not nq or not nk:
            continue
        a, b = slice(at_q[n], at_q[n] + nq), slice(at_k[n], at_k[n] + nk)
        hidden = None
        if c['causal']:
            hidden = torch.ones((nq, nk), dtype=torch.bool, device='cuda').triu(nk - nq + 1)
        blind = hidden.all(1) if hidden is not None else torch.zeros(nq, dtype=torch.bool, device='cuda')
        for h in range(c['heads']):
            m = h * c['kv_heads'] // c['heads']
            x, y, z = q[a, h].requires_grad_(train), k[b, m].requires_grad_(train), v[b, m].requires_grad_(train)
            with torch.set_grad_enabled(train):
                score = torch.mm(x, y.t()) * s['scale']
                if hidden is not None:
                    score = score.masked_fill(hidden, -math.inf).masked_fill(blind[:, None], 0.0)
                p = torch.softmax(score, 1)
                o = torch.mm(p, z).masked_fill(blind[:, None], 0.0)
            out[a, h] = o.detach()
            lse[a, h] = torch.logsumexp(score.detach(), 1).masked_fill(blind, -math.inf)
            if train:
                got = torch.autograd.grad(o, (x, y, z), s['grad'][a, h].double())
                for total, part, rows, head in zip(grads, got, (a, b, b), (h, m, m)):
                    total[rows, head] += part
            del score, p, o
    if train:
        return (out, *grads)
    return (out, lse.t().contiguous()) if c['cache'] else out


def _exact_rotary(s):
    """Pair by pair as a complex number turned by exp(i angle); gradients by differentiating that."""
    c = s['case']
    axis = [a for a, n in enumerate(s['sections']) for _ in range(n)]
    angle = s['positions'].double()[:, axis] * s['inv_freq'].double()
    spin = torch.polar(torch.ones_like(angle), angle)[:, None]
    order = torch.arange(c['dim'], device='cuda')
    if not c['interleaved']:  # neighbours first, so that one form serves both
        order = torch.cat([order[:c['rotated']].view(2, -1).t().flatten(), order[c['rotated']:]])
    leaves = {n: s[n].detach().double().requires_grad_(c['train']) for n in ('q', 'k', 'qw', 'kw') if s[n] is not None}

    def apply(x, w):
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c['dim'] + 1e-6) * w
        x = x[..., order]
        z = torch.view_as_complex(x[..., :c['rotated']].unflatten(-1, (-1, 2)).contiguous())
        x = torch.cat([torch.view_as_real(z * spin).flatten(-2), x[..., c['rotated']:]], -1)
        return x[..., torch.argsort(order)]

    outs = [apply(leaves['q'], leaves.get('qw')), apply(leaves['k'], leaves.get('kw'))]
    got = torch.autograd.grad(outs, list(leaves.values()), (s['gq'].double(), s['gk'].double())) if c['train'] else ()
    return [o.detach() for o in outs] + list(got)


def _exact_dropout(s):
    import numpy as np
    c = s['case']
    n = c['rows'] * c['width']
    seed, offset = (int(v) & (2 ** 64 - 1) for v in s['seed'].tolist())
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    low = np.uint64(LOW)
    x0, x1 = block & low, block >> np.uint64(32)
    x2, x3 = np.full_like(block, offset & LOW), np.full_like(block, offset >> 32)
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(10):
        u, w = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = ((w >> np.uint64(32)) ^ x1 ^ np.uint64(k0), w & low,
                          (u >> np.uint64(32)) ^ x3 ^ np.uint64(k1), u & low)
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = np.stack([x0, x1, x2, x3], 1).reshape(-1)[:n]
    kept = torch.from_numpy(words >= np.uint64(int(c['p'] * 2.0 ** 32))).cuda().view(c['rows'], c['width'])
    factor = kept.double() / (1.0 - c['p'])
    y = s['x'].detach().double() * factor
    if c['residual']:
        y = y + s['residual'].detach().double()
    if not c['train']:
        return y
    return [y, s['grad'].double() * factor] + ([s['grad'].double()] if c['residual'] else [])


def exact(case, seed):
    state = prepare(case, seed)
    return {'attention': _exact_attention, 'rotary': _exact_rotary, 'dropout': _exact_dropout}[case['op']](state)
