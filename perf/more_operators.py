"""The operators of Qwen3.5's linear-attention layers for several requests: what is measured, and their plain forms.

  conv   delta.conv        the short causal convolution in front of the rule, with the last rows of each request kept
  rule   delta.rule        the gated delta rule: one token per request, or whole prompts and pieces of them
  norm   layer.rms_norm    root-mean-square norm of rows: with the residual's addition, with a gate, to 8 bits

A request's state is row slots[b] of a pool: the rule's [heads, key dim, value dim], the convolution's last width - 1
input rows. Its new tokens are rows starts[b] .. starts[b + 1] - 1 (one row a request without starts); lengths counts
them and all before, so a request all of whose tokens are new starts from zeros.
"""
from __future__ import annotations

import math
import random

import torch

own = False     # whether run() makes the package's calls, or computes their plain forms

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}
EPS = 1e-6
WIDTH = 4       # taps of the convolution
# (key heads, value heads, key dim, value dim): the package's own delta-net benchmark, and others
HEADS = [(16, 32, 128, 128), (32, 32, 128, 128), (16, 16, 128, 128), (4, 8, 64, 64), (2, 6, 128, 64), (2, 4, 256, 256),
         (3, 3, 64, 128)]
HIDDEN = [4096, 2048, 1024, 5120, 768, 2560, 14336]
MOST_STEP = 256 * 32 * 128 * 128          # state values of a drawn step
MOST_PROMPTS = 8192 * 32 * 128 * 128      # tokens x state values of drawn prompts
MOST_CONV = 16384 * 8192
MOST_NORM = 16384 * 4096


def _rule(name, heads, requests, dtype, longest=1, cached=1000, gates=True, order='grouped', idle=0):
    """`longest`: the most new tokens of a request (1: a decode step, one row a request); `cached`: the most tokens
    that a request has before them (0: every request starts from zeros); `gates`: decay and beta as projected."""
    return {'name': name, 'kind': 'rule', 'key_heads': heads[0], 'value_heads': heads[1], 'key_dim': heads[2],
            'value_dim': heads[3], 'requests': requests, 'dtype': dtype, 'longest': longest, 'cached': cached,
            'gates': gates, 'order': order, 'idle': idle}


def _conv(name, channels, requests, dtype, longest=1, cached=1000, bias=False, idle=0):
    return {'name': name, 'kind': 'conv', 'channels': channels, 'requests': requests, 'dtype': dtype,
            'longest': longest, 'cached': cached, 'bias': bias, 'idle': idle}


def _norm(name, rows, dim, dtype, residual=False, heads=0, out=''):
    """heads: rows of [heads, dim] with a gate, views of one projection; out: the results' type, '' for x's own."""
    return {'name': name, 'kind': 'norm', 'rows': rows, 'dim': dim, 'dtype': dtype, 'residual': residual,
            'heads': heads, 'out': out or dtype}


def listed():
    return [
        # one chat's next token: the package's delta-net benchmark with norms and gates inside
        _rule('rule_one_f32', (16, 32, 128, 128), 1, 'f32'),
        # a server's decode batch, empty places among its requests, 16-bit activations
        _rule('rule_b70_bf16', (16, 32, 128, 128), 70, 'bf16', idle=3),
        # the largest decode batch of a server, gates computed by its program
        _rule('rule_b256_f32', (32, 32, 128, 128), 256, 'f32', gates=False),
        # one short prompt of a small model: latency
        _rule('rule_t77_hd64_f16', (4, 8, 64, 64), 1, 'f16', longest=77, cached=0),
        # one long document from its beginning
        _rule('rule_t8192_bf16', (16, 32, 128, 128), 1, 'bf16', longest=8192, cached=0),
        # pieces of prompts, drafted tokens and decoding requests in one call, heads in GGUF's tiled order
        _rule('rule_pieces_b6_f32', (16, 32, 128, 128), 6, 'f32', longest=2048, order='tiled', idle=1),
        # a decode step's convolution over q, k and v
        _conv('conv_b5_f32', 8192, 5, 'f32'),
        # pieces of prompts through it
        _conv('conv_pieces_b9_bf16', 8192, 9, 'bf16', longest=4096, idle=1),
        # a decode step's norm with the residual of one token
        _norm('norm_one_f32', 1, 4096, 'f32', residual=True),
        # the same for a long prompt
        _norm('norm_t8192_f32', 8192, 4096, 'f32', residual=True),
        # behind the rule: every head of every token, gated
        _norm('norm_gated_t4096_bf16', 4096, 128, 'bf16', heads=32),
        # an odd number of rows kept in 8 bits
        _norm('norm_t2049_q8_0', 2049, 5120, 'bf16', residual=True, out='q8_0'),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(['rule', 'rule', 'rule', 'conv', 'norm', 'norm'])
    dtype = rng.choice(list(DTYPES))
    cached = rng.choice([0, 5, 1000])
    if kind == 'rule':
        heads = rng.choice(HEADS)
        values = heads[1] * heads[2] * heads[3]
        longest, requests = 1, _log(rng, 1, min(300, MOST_STEP // values))
        if rng.random() < 0.6:
            requests = _log(rng, 1, 24)
            longest = _log(rng, 2, min(8192, max(2, MOST_PROMPTS // (values * requests))))
        c = _rule('', heads, requests, dtype, longest, cached, rng.random() < 0.6, rng.choice(['grouped', 'tiled']),
                  rng.randrange(0, 1 + requests // 6))
    elif kind == 'conv':
        heads = rng.choice(HEADS)
        channels = rng.choice([2 * heads[0] * heads[2] + heads[1] * heads[3], _log(rng, 1, 9000)])
        requests = _log(rng, 1, 300)
        longest = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, MOST_CONV // (channels * requests)))
        c = _conv('', channels, requests, dtype, min(longest, 16384), cached, rng.random() < 0.5,
                  rng.randrange(0, 1 + requests // 6))
    else:
        rows = _log(rng, 1, 16384)
        eight = ['q8_0'] if dtype != 'f32' else []     # what is kept in 8 bits was of 16
        if rng.random() < 0.35:
            heads, dim = rng.choice([3, 8, 16, 32]), rng.choice([64, 128, 256])
            c = _norm('', min(rows, MOST_NORM // (heads * dim)), dim, dtype, heads=heads,
                      out=rng.choice(['', 'f32', 'bf16', *eight]))
        else:
            out = rng.choice(['', 'f32', 'f16', 'bf16', *eight])
            dim = rng.choice(HIDDEN) if out == 'q8_0' or rng.random() < 0.4 else _log(rng, 1, 16384)
            c = _norm('', max(1, min(rows, MOST_NORM // dim)), dim, dtype, rng.random() < 0.6, out=out)
    del c['name']
    return c


def _requests(case):
    """(cached tokens, new tokens) of each request: from the case alone. The first has the most new tokens, the others
    spread over their logarithms; idle ones have none (in a decode step: no slot)."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != 'name')))
    n, most = case['requests'], case['longest']
    new = [most] + [_log(rng, 1, most) for _ in range(n - 1)]
    old = [rng.randrange(0, case['cached'] + 1) for _ in range(n)]
    for i in range(case['idle']):
        new[n - 1 - i] = 0
    return old, new


def work(case):
    e = BYTES[case['dtype']]
    if case['kind'] == 'norm':
        values = case['rows'] * max(1, case['heads']) * case['dim']
        out = 34 / 32 if case['out'] == 'q8_0' else BYTES[case['out']]
        moved = e * (2 if case['heads'] else 1) + (8 if case['residual'] else 0) + out
        return {'bytes': int(values * moved) + 4 * case['dim'], 'flops': values * (4 + 5 * bool(case['heads']))}
    old, new = _requests(case)
    tokens, busy = sum(new), sum(1 for x in new if x)
    kept = sum(1 for o, x in zip(old, new) if x and o)     # states that are read
    tables = 4 * case['requests'] * (2 if case['longest'] == 1 else 3)
    if case['kind'] == 'conv':
        c = case['channels']
        return {'bytes': 2 * tokens * c * e + 4 * (WIDTH - 1) * c * (busy + kept) + 4 * c * (WIDTH + case['bias']) + tables,
                'flops': tokens * c * (2 * WIDTH + 4)}
    hk, hv, kd, vd = case['key_heads'], case['value_heads'], case['key_dim'], case['value_dim']
    return {'bytes': tokens * ((2 * hk * kd + 2 * hv * vd) * e + 8 * hv) + 4 * hv * kd * vd * (busy + kept) + tables,
            'flops': 6 * tokens * hv * kd * vd}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, dtype=dtype, device='cuda', generator=gen)

    dtype = DTYPES[case['dtype']]
    if case['kind'] == 'norm':
        rows, dim, heads = case['rows'], case['dim'], case['heads']
        s = {'case': case, 'weight': 1 + 0.2 * normal(dim), 'residual': None, 'gate': None}
        if heads:     # the rule's result, and z beside other columns of a projection
            s['x'] = 0.1 * normal(rows, heads, dim, dtype=dtype)
            s['gate'] = normal(rows, 2 * heads * dim, dtype=dtype)[:, heads * dim:].unflatten(-1, (heads, dim))
        else:
            s['x'] = normal(rows, dim, dtype=dtype)
        if case['residual']:
            s['residual'] = 3 * normal(rows, dim)
        return s
    old, new = _requests(case)
    n = case['requests']
    step = case['longest'] == 1
    rows = n if step else sum(new)
    pool = n + 2
    slots = torch.randperm(pool, generator=gen, device='cuda')[:n].to(torch.int32)
    if step and case['idle']:
        slots[n - case['idle']:] = -1
    s = {'case': case, 'slots': slots, 'lengths': _ints([o + x for o, x in zip(old, new)]),
         'starts': None if step else _ints([0] + [sum(new[:b + 1]) for b in range(n)])}
    if case['kind'] == 'conv':
        c = case['channels']
        s.update(x=normal(rows, c, dtype=dtype), weight=0.5 * normal(c, WIDTH), state=normal(pool, WIDTH - 1, c),
                 bias=0.1 * normal(c) if case['bias'] else None,
                 out=torch.zeros((rows, c), dtype=dtype, device='cuda'))     # rows without a slot stay as they are
        return s
    hk, hv, kd, vd = case['key_heads'], case['value_heads'], case['key_dim'], case['value_dim']
    x = normal(rows, 2 * hk * kd + hv * vd)     # the convolution's output: silu of it, q, k and v side by side
    x = (x / (1 + torch.exp(-x))).to(dtype)
    q, k, v = (y.unflatten(-1, (-1, d)) for y, d in zip(x.split([hk * kd, hk * kd, hv * vd], dim=1), (kd, kd, vd)))
    decay, beta = normal(rows, hv), 2 * normal(rows, hv)
    # forgetting rates from a thousandth of a token's state to most of it, as trained models have them
    a = -torch.exp(torch.empty(hv, device='cuda').uniform_(0, math.log(16), generator=gen))
    dt_bias = torch.log(torch.expm1(torch.exp(torch.empty(hv, device='cuda').uniform_(math.log(1e-3), math.log(1e-1),
                                                                                     generator=gen))))
    if not case['gates']:
        decay, beta = a * torch.log1p(torch.exp(decay + dt_bias)), 1 / (1 + torch.exp(-beta))
        a = dt_bias = None
    s.update(q=q, k=k, v=v, decay=decay, beta=beta, a=a, dt_bias=dt_bias, state=0.3 * normal(pool, hv, kd, vd),
             out=torch.zeros((rows, hv, vd), dtype=dtype, device='cuda'))
    return s


def run(state):
    kind = state['case']['kind']
    if own:
        return _own(kind, state)
    return {'rule': _plain_rule, 'conv': _plain_conv, 'norm': _plain_norm}[kind](state)


def _own(kind, s):
    from localai_amd import delta, dequant, layer
    c = s['case']
    if kind == 'norm':
        x, q8 = s['x'], c['out'] == 'q8_0'
        y = layer.rms_norm(x, s['weight'], eps=EPS, residual=s['residual'], gate=s['gate'],
                           dtype='q8_0' if q8 else DTYPES[c['out']])
        if q8:     # read again as activations of x's type
            y = dequant.dequantize_device(y, 8, x.shape).to(x.dtype)
        return [y] if s['residual'] is None else [y, s['residual']]
    if kind == 'conv':
        y = delta.conv(s['x'], s['weight'], s['state'], slots=s['slots'], starts=s['starts'], lengths=s['lengths'],
                       bias=s['bias'], out=s['out'])
    else:
        y = delta.rule(s['q'], s['k'], s['v'], s['decay'], s['beta'], s['state'], slots=s['slots'],
                       starts=s['starts'], lengths=s['lengths'], a=s['a'], dt_bias=s['dt_bias'], order=c['order'],
                       norm_eps=EPS, out=s['out'])
    return [y, s['state']]


def _silu(x):
    return x / (1 + torch.exp(-x))


def _rows_of(s):
    """(starts [requests + 1], count [requests]) of a step or of prompts; requests without a slot count 0."""
    n = s['case']['requests']
    starts = torch.arange(n + 1, device='cuda') if s['starts'] is None else s['starts'].long()
    return starts, (starts[1:] - starts[:-1]) * (s['slots'] >= 0)


def _plain_rule(s):
    c, pool, out = s['case'], s['state'], s['out']
    hv, kd, rows = c['value_heads'], c['key_dim'], s['v'].shape[0]
    group = hv // c['key_heads']
    q, k = (x.float() for x in (s['q'], s['k']))
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + EPS) / math.sqrt(kd)
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + EPS)
    if c['order'] == 'grouped':
        q, k = (x.repeat_interleave(group, dim=1) for x in (q, k))
    else:
        q, k = (x.repeat(1, group, 1) for x in (q, k))
    v, decay, beta = s['v'].float(), s['decay'], s['beta']
    if s['a'] is not None:
        x = decay + s['dt_bias']
        decay = s['a'] * (torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x))))
        beta = 1 / (1 + torch.exp(-beta))
    factor = torch.exp(decay)
    starts, count = _rows_of(s)
    old = (s['lengths'] > count) & (count > 0)
    state = torch.where(old[:, None, None, None], pool[s['slots'].clamp(min=0).long()], 0.0)
    result = torch.cat([out, out[:1]])     # one row more: where requests that have ended write
    for i in range(c['longest']):
        live = i < count
        t = (starts[:-1] + i).clamp(max=rows - 1)
        state = state * torch.where(live[:, None], factor[t], 1.0)[..., None, None]
        kt = k[t][..., None]
        change = (v[t] - (state * kt).sum(-2)) * torch.where(live[:, None], beta[t], 0.0)[..., None]
        state = state + kt * change[..., None, :]
        result[torch.where(live, t, rows)] = (state * q[t][..., None]).sum(-2).to(out.dtype)
    # idle requests are the last ones: without a slot, or with their states unchanged
    kept = c['requests'] - c['idle']
    pool[s['slots'][:kept].long()] = state[:kept]
    return [result[:rows], pool]


def _plain_conv(s):
    c, x, pool = s['case'], s['x'], s['state']
    rows, w = x.shape[0], s['weight']
    starts, count = _rows_of(s)
    old = (s['lengths'] > count) & (count > 0)
    before = torch.where(old[:, None, None], pool[s['slots'].clamp(min=0).long()], 0.0)
    t = torch.arange(rows, device=x.device)
    b = torch.searchsorted(starts[1:], t, right=True)
    y = torch.zeros_like(x, dtype=torch.float32) if s['bias'] is None else s['bias'].expand(x.shape)
    for j in range(WIDTH):
        at = t - (WIDTH - 1) + j - starts[b]
        value = torch.where((at >= 0)[:, None], x[(t - (WIDTH - 1) + j).clamp(min=0)].float(),
                            before[b, (WIDTH - 1 + at).clamp(max=WIDTH - 2)])
        y = y + w[:, j] * value
    y = torch.where((count[b] > 0)[:, None], _silu(y).to(x.dtype), s['out'])
    after = []
    for j in range(WIDTH - 1):
        at = count - (WIDTH - 1) + j
        row = (starts[:-1] + at).clamp(0, rows - 1)
        place = (WIDTH - 1 + at).clamp(0, WIDTH - 2)
        after.append(torch.where((at >= 0)[:, None], x[row].float(),
                                 before[torch.arange(len(at), device=x.device), place]))
    kept = c['requests'] - c['idle']
    pool[s['slots'][:kept].long()] = torch.stack(after, 1)[:kept]
    return [y, pool]


def _plain_norm(s):
    c, x = s['case'], s['x'].float()
    if s['residual'] is not None:
        x = s['residual'].add_(x)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s['weight']
    if s['gate'] is not None:
        y = y * _silu(s['gate'].float())
    if c['out'] == 'q8_0':
        blocks = y.unflatten(-1, (-1, 32))
        d = (blocks.abs().amax(-1, keepdim=True) / 127).half().float()
        y = (torch.round(blocks / torch.where(d == 0, 1.0, d)).clamp(-127, 127) * d).flatten(-2).to(s['x'].dtype)
    else:
        y = y.to(DTYPES[c['out']])
    return [y] if s['residual'] is None else [y, x]


def exact(case, seed):
    s = prepare(case, seed)
    return {'rule': _exact_rule, 'conv': _exact_conv, 'norm': _exact_norm}[case['kind']](s)


def _pieces(s):
    """(slot, first row, rows, state before in 64 bits) of each request that has new tokens."""
    n = s['case']['requests']
    starts = list(range(n + 1)) if s['starts'] is None else s['starts'].tolist()
    for b, (slot, length) in enumerate(zip(s['slots'].tolist(), s['lengths'].tolist())):
        count = starts[b + 1] - starts[b]
        if slot >= 0 and count:
            state = s['state'][slot].double()
            yield slot, starts[b], count, state if length > count else torch.zeros_like(state)


def _exact_rule(s):
    """Request by request, 64 tokens at a time: their changes of the state from one triangular system."""
    c = s['case']
    heads = torch.arange(c['value_heads'], device='cuda')
    key = heads // (c['value_heads'] // c['key_heads']) if c['order'] == 'grouped' else heads % c['key_heads']
    unit = [x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + EPS) for x in (s['q'], s['k'])]
    q, k = ((x.transpose(0, 1)[key]) for x in unit)     # [heads, tokens, key dim]
    q = q * c['key_dim'] ** -0.5
    v, decay, beta = s['v'].double().transpose(0, 1), s['decay'].double().t(), s['beta'].double().t()
    if s['a'] is not None:
        decay = s['a'].double()[:, None] * torch.logaddexp(decay + s['dt_bias'].double()[:, None], decay.new_zeros(()))
        beta = torch.sigmoid(beta)
    out, pool = s['out'].double(), s['state'].double()
    for slot, first, count, state in _pieces(s):
        for at in range(first, first + count, 64):
            part = slice(at, min(at + 64, first + count))
            n = part.stop - part.start
            total = torch.cumsum(decay[:, part], 1)
            since = torch.exp((total[:, :, None] - total[:, None, :]).tril()).tril()
            grown = torch.exp(total)[..., None]
            b = beta[:, part, None]
            qs, ks, vs = (x[:, part].contiguous() for x in (q, k, v))
            kt = ks.transpose(1, 2).contiguous()
            system = torch.eye(n, device='cuda', dtype=torch.float64) + (b * (ks @ kt) * since).tril(-1)
            change = torch.linalg.solve_triangular(system, b * (vs - grown * (ks @ state)), upper=False)
            out[part] = (grown * (qs @ state) + ((qs @ kt) * since) @ change).transpose(0, 1)
            left = torch.exp(total[:, -1:] - total)[:, None, :]
            state = grown[:, -1:] * state + (kt * left) @ change
        pool[slot] = state
    return [out, pool]


def _exact_conv(s):
    out, pool = s['out'].double(), s['state'].double()
    w = s['weight'].double()
    for slot, first, count, state in _pieces(s):
        line = torch.cat([state, s['x'][first:first + count].double()])
        pool[slot] = line[count:]
        for at in range(0, count, 1024):
            part = line[at:min(at + 1024, count) + WIDTH - 1]
            y = (part.unfold(0, WIDTH, 1) * w).sum(-1)
            if s['bias'] is not None:
                y = y + s['bias'].double()
            out[first + at:first + at + len(y)] = y * torch.sigmoid(y)
    return [out, pool]


def _exact_norm(s):
    c, h = s['case'], s['x'].double()
    if s['residual'] is not None:
        h = h + s['residual'].double()
    y = h / torch.sqrt(h.square().sum(-1, keepdim=True) / c['dim'] + EPS) * s['weight'].double()
    if s['gate'] is not None:
        z = s['gate'].double()
        y = y * z * torch.sigmoid(z)
    if c['out'] == 'q8_0':
        blocks = y.reshape(*y.shape[:-1], -1, 32)
        d = (blocks.abs().amax(-1, keepdim=True) / 127).to(torch.float16).double()
        y = torch.where(d == 0, 0.0, (blocks / d).round().clamp(-127, 127) * d).reshape(y.shape)
    return [y] if s['residual'] is None else [y, h]
