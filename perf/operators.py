"""The operators that serve several requests from a paged key/value cache: what is measured, and their plain forms.

  extend     paged.extend            the requests' page tables and the slots of a step's new tokens, from their lengths
  store      paged.norm_rope_store   q / k norms per head, the position rotation, and k / v written to their slots
  attention  paged.attention         the new tokens' attention over the pages: one token a request, or several

A cache of one layer is k and v [pages, kv heads, page size, head dim]; a page table row lists a request's pages in
the order of their positions; slot = page * page size + place in the page.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False     # whether run() makes the package's calls, or computes their plain forms

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}
EPS = 1e-6
ROPE_BASE = 500000.0
# (query heads, kv heads, head dim) that the package's tests and benchmark use
HEADS = [(32, 8, 128), (64, 8, 128), (28, 4, 128), (16, 4, 256), (8, 8, 64), (6, 2, 64), (4, 4, 256)]
# bytes of padded k and v (requests x longest) that a drawn attention does not exceed, and pairs of a drawn prompt
MOST_PADDED = 64 * 8192 * 2 * 8 * 128 * 2
MOST_PAIRS = 4 * 512 * 2048
MOST_TOKENS = 131072
MOST_STORE = 8192 * (64 + 16) * 128


def _extend(name, requests, longest, page, new, idle=0):
    """`new`: the most new tokens of a request (1: a decode step); `longest`: positions after the step."""
    return {'name': name, 'kind': 'extend', 'requests': requests, 'longest': longest, 'page': page, 'new': new,
            'idle': idle}


def _store(name, heads, tokens, dtype, page, rope, rotary, norm):
    return {'name': name, 'kind': 'store', 'heads': heads[0], 'kv_heads': heads[1], 'head_dim': heads[2],
            'tokens': tokens, 'dtype': dtype, 'page': page, 'rope': rope, 'rotary': rotary, 'norm': norm}


def _attention(name, heads, requests, longest, dtype, page, new=1, window=0, gate=False, idle=0):
    return {'name': name, 'kind': 'attention', 'heads': heads[0], 'kv_heads': heads[1], 'head_dim': heads[2],
            'requests': requests, 'longest': longest, 'dtype': dtype, 'page': page, 'new': new, 'window': window,
            'gate': gate, 'idle': idle}


def listed():
    return [
        # one chat's next token: the smallest bookkeeping there is, once per token
        _extend('extend_one', 1, 4096, 64, 1),
        # a decode step of a server with 256 places, some of them empty
        _extend('extend_decode_b256', 256, 32768, 16, 1, idle=9),
        # prompts and decoding requests in one step: slots for tens of thousands of tokens
        _extend('extend_prompts_b48', 48, 8191, 16, 8000),
        # one token through Qwen3-like q / k norms and the half-split rotation, cache in fp32
        _store('store_one_f32', (32, 8, 128), 1, 'f32', 64, 'halves', 128, True),
        # an odd number of tokens through Qwen3.5's partial rotation, head dim 256
        _store('store_t777_hd256_f16', (16, 4, 256), 777, 'f16', 32, 'halves', 64, True),
        # a long prompt with Llama's adjacent pairs and no norms, 64 query heads
        _store('store_t8192_bf16', (64, 8, 128), 8192, 'bf16', 16, 'pairs', 128, False),
        # short requests of a small multi-head model, an empty place among them: latency
        _attention('attention_b7_hd64_f32', (8, 8, 64), 7, 301, 'f32', 16, idle=1),
        # one chat of 4096 positions, fp32 pages: the package's own decode benchmark, paged
        _attention('attention_one_4096_f32', (32, 8, 128), 1, 4096, 'f32', 64),
        # one long document
        _attention('attention_one_131072_f16', (32, 8, 128), 1, 131072, 'f16', 64),
        # a server's decode batch of very different lengths
        _attention('attention_b64_8192_bf16', (32, 8, 128), 64, 8192, 'bf16', 16, idle=2),
        # gated full attention with head dim 256 under a sliding window
        _attention('attention_b16_hd256_window_f16', (16, 4, 256), 16, 5000, 'f16', 32, window=1024, gate=True),
        # pieces of prompts and drafted tokens, each over what its request has cached
        _attention('attention_prompts_b4_f16', (32, 8, 128), 4, 2048, 'f16', 16, new=512),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(['extend', 'store', 'attention', 'attention'])
    page = rng.choice([16, 32, 64, 128])
    if kind == 'extend':
        requests = _log(rng, 1, 256)
        longest = _log(rng, 2, 32768)
        new = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, min(longest, MOST_TOKENS // requests)))
        c = _extend('', requests, longest, page, new, idle=rng.randrange(0, 1 + requests // 8))
    elif kind == 'store':
        heads = rng.choice(HEADS)
        most = MOST_STORE // ((heads[0] + 2 * heads[1]) * heads[2])
        c = _store('', heads, _log(rng, 1, min(16384, most)), rng.choice(list(DTYPES)), page,
                   rng.choice(['halves', 'pairs']), rng.choice([heads[2], heads[2] // 2, heads[2] // 4]),
                   rng.random() < 0.6)
    else:
        heads, dtype = rng.choice(HEADS), rng.choice(list(DTYPES))
        requests = _log(rng, 1, 96)
        most = MOST_PADDED // (requests * 2 * heads[1] * heads[2] * BYTES[dtype])
        longest = _log(rng, 1, min(131072, most))
        new, window = 1, 0
        if rng.random() < 0.3:
            requests = _log(rng, 1, 8)
            new = _log(rng, 2, 512)
            longest = new + _log(rng, 1, max(1, MOST_PAIRS // (requests * new) // max(1, heads[0] // 32) - new))
        if rng.random() < 0.3:
            window = _log(rng, 1, max(2, longest))
        c = _attention('', heads, requests, longest, dtype, page, new=new, window=window, gate=rng.random() < 0.25,
                       idle=rng.randrange(0, 1 + requests // 8))
    del c['name']
    return c


def _requests(case):
    """(cached positions before the step, new tokens) of each request: from the case alone. The first request is the
    longest one and has the most new tokens; others spread over their logarithms; idle ones have none of either."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != 'name')))
    n, longest, most = case['requests'], case['longest'], case['new']
    old, new = [longest - most], [most]
    for _ in range(n - 1):
        x = _log(rng, 1, most)
        total = max(x, _log(rng, max(1, longest // 32), longest))
        old.append(total - x)
        new.append(x)
    for i in range(case['idle']):
        old[n - 1 - i] = new[n - 1 - i] = 0
    return old, new


def _pages(positions, page):
    return -(-positions // page)


def _span(case, old, new):
    """(first position read, positions after the step) of a request."""
    first = old + 1 - case['window'] if case['window'] else 0
    return (max(0, first), old + new) if new else (0, 0)


def _pairs(case, old, new):
    """(query token, position) pairs of a request."""
    w = case['window'] or old + new
    return sum(min(old + i + 1, w) for i in range(new))


def work(case):
    if case['kind'] == 'extend':
        old, new = _requests(case)
        tokens = sum(new)
        fresh = sum(_pages(o + n, case['page']) - _pages(o, case['page']) for o, n in zip(old, new))
        partly = sum(1 for o, n in zip(old, new) if n and o % case['page'])
        # lengths and new counts read, lengths and starts written; a fresh page's id read and written; the page that
        # a request goes on filling read; slot and position of each token written
        return {'bytes': 16 * len(old) + 8 * fresh + 4 * partly + 8 * tokens + 12, 'flops': 0}
    nh, nkv, hd = case['heads'], case['kv_heads'], case['head_dim']
    if case['kind'] == 'store':
        t, e = case['tokens'], BYTES[case['dtype']]
        values = (nh + 2 * nkv) * hd
        return {'bytes': t * (4 * values + 4 * nh * hd + 2 * e * nkv * hd + 8),
                'flops': t * (nh + nkv) * (5 * hd * case['norm'] + 3 * case['rotary'])}
    old, new = _requests(case)
    spans = [_span(case, o, n) for o, n in zip(old, new)]
    read = sum(b - a for a, b in spans)
    pages = sum(_pages(b, case['page']) - a // case['page'] for a, b in spans if b)
    io = sum(new) * nh * hd * (12 if case['gate'] else 8)
    return {'bytes': read * 2 * nkv * hd * BYTES[case['dtype']] + io + 4 * pages + 8 * len(old),
            'flops': 4 * nh * hd * sum(_pairs(case, o, n) for o, n in zip(old, new))}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _normal(shape, dtype, gen):
    return torch.randn(shape, dtype=dtype, device='cuda', generator=gen)


def _tables(held, pool, width, gen):
    """(table [requests, width], page list [pool]): requests that hold `held` pages each, handed out from the front of
    the list as requests that grow side by side take them (page j of each before page j + 1 of any); -1 elsewhere."""
    pages = torch.randperm(pool, generator=gen, device='cuda').to(torch.int32)
    taken = torch.arange(width, device='cuda')[:, None] < _ints(held)[None, :]
    table = torch.full((width, len(held)), -1, dtype=torch.int32, device='cuda')
    table[taken] = pages[:sum(held)]
    return table.t().contiguous(), pages


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    page = case['page']
    if case['kind'] == 'extend':
        old, new = _requests(case)
        held, need = [_pages(o, page) for o in old], [_pages(o + n, page) for o, n in zip(old, new)]
        table, pages = _tables(held, sum(need) + 8, max(need), gen)
        return {'case': case, 'lengths': _ints(old), 'new': _ints(new), 'table': table, 'free': pages,
                'used': _ints([sum(held)]), 'tokens': sum(new) + 5}     # five places of padding behind the last token
    nh, nkv, hd, dtype = case['heads'], case['kv_heads'], case['head_dim'], DTYPES[case['dtype']]
    if case['kind'] == 'store':
        t, n = case['tokens'], case['rotary'] // 2
        pool = _pages(t, page) + 3
        qkv = _normal((t, (nh + 2 * nkv) * hd), torch.float32, gen)     # the fused projection's output
        q, k, v = (x.view(t, -1, hd) for x in qkv.split([nh * hd, nkv * hd, nkv * hd], dim=1))
        places, order = torch.arange(t, device='cuda'), torch.randperm(pool, generator=gen, device='cuda')
        first = torch.randint(0, 100000, (1,), generator=gen, device='cuda')
        weights = [1 + 0.2 * _normal((hd,), torch.float32, gen) if case['norm'] else None for _ in range(2)]
        return {'case': case, 'q': q, 'k': k, 'v': v, 'positions': (first + places).to(torch.int32),
                'slots': (order[places // page] * page + places % page).to(torch.int32),
                'freq': ROPE_BASE ** (-torch.arange(n, dtype=torch.float64, device='cuda') / n),
                'q_weight': weights[0], 'k_weight': weights[1],
                'k_cache': _normal((pool, nkv, page, hd), dtype, gen),
                'v_cache': _normal((pool, nkv, page, hd), dtype, gen)}
    old, new = _requests(case)
    total = [o + n for o, n in zip(old, new)]
    held = [_pages(x, page) for x in total]
    table, _ = _tables(held, sum(held) + 8, max(held), gen)
    # a decode batch has one row a place, empty places among them; pieces of prompts follow each other
    starts = None if case['new'] == 1 else _ints([0] + np.cumsum(new).tolist())
    rows = case['requests'] if starts is None else sum(new)
    return {'case': case, 'q': 2 * _normal((rows, nh, hd), torch.float32, gen), 'table': table,
            'lengths': _ints(total), 'starts': starts,
            'k_cache': _normal((sum(held) + 8, nkv, page, hd), dtype, gen),
            'v_cache': _normal((sum(held) + 8, nkv, page, hd), dtype, gen),
            'gate': _normal((rows, nh, hd), torch.float32, gen) if case['gate'] else None}


def run(state):
    kind = state['case']['kind']
    if own:
        return _own(kind, state)
    return {'extend': _plain_extend, 'store': _plain_store, 'attention': _plain_attention}[kind](state)


def _own(kind, s):
    from localai_amd import paged
    c = s['case']
    if kind == 'extend':
        step = paged.extend(s['lengths'], s['new'], s['table'], s['free'], s['used'], c['page'], s['tokens'])
        return [step.lengths, step.used, step.starts, step.slots, step.positions, step.status, s['table']]
    if kind == 'store':
        q = paged.norm_rope_store(s['q'], s['k'], s['v'], s['positions'], s['slots'], s['k_cache'], s['v_cache'],
                                  freq=s['freq'], q_weight=s['q_weight'], k_weight=s['k_weight'], eps=EPS,
                                  rope=c['rope'])
        return [q, s['k_cache'], s['v_cache']]
    return paged.attention(s['q'], s['k_cache'], s['v_cache'], s['table'], s['lengths'], starts=s['starts'],
                           window=c['window'], gate=s['gate'])


def _plain_extend(s):
    page, (n, width), table = s['case']['page'], s['table'].shape, s['table']
    old, total = s['lengths'], s['lengths'] + s['new']
    held, want = (old + page - 1) // page, (total + page - 1) // page
    need = want - held
    before = torch.cumsum(need, 0, dtype=torch.int32) - need
    starts = torch.cat([torch.zeros_like(s['used']), torch.cumsum(s['new'], 0, dtype=torch.int32)])
    used = s['used'] + need.sum(dtype=torch.int32)
    short = (used > s['free'].numel()).to(torch.int32)
    narrow = ((want > width) | (s['new'] < 0) | (old < 0)).any().to(torch.int32)
    many = (starts[-1:] > s['tokens']).to(torch.int32)
    status = short + 2 * narrow + 4 * many
    fits = status == 0
    j = torch.arange(width, dtype=torch.int32, device=table.device)[None, :]
    fresh = (j >= held[:, None]) & (j < want[:, None]) & fits
    take = (s['used'] + before[:, None] + j - held[:, None]).clamp(0, s['free'].numel() - 1)
    table = torch.where(fresh, s['free'][take], table)
    t = torch.arange(s['tokens'], dtype=torch.int32, device=table.device)
    b = torch.searchsorted(starts[1:], t, right=True, out_int32=True).clamp(max=n - 1)
    live = (t < starts[-1]) & fits
    position = torch.where(live, old[b] + t - starts[b], -1)
    at = position.clamp(0, width * page - 1)
    slots = torch.where(live, table[b, at // page] * page + at % page, -1)
    return [torch.where(fits, total, old), torch.where(fits, used, s['used']), torch.where(fits, starts, 0), slots,
            position, status, table]


def _rotate(x, cos, sin, rope):
    n = cos.shape[-1]
    pick = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if rope == 'pairs' else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., pick[0]], x[..., pick[1]]
    y = x.clone()
    y[..., pick[0]] = a * cos - b * sin
    y[..., pick[1]] = b * cos + a * sin
    return y


def _plain_store(s):
    c, kc, vc = s['case'], s['k_cache'], s['v_cache']
    angle = (s['positions'].double()[:, None] * s['freq'])[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = s['q'], s['k']
    if c['norm']:
        q, k = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
                for x, w in ((q, s['q_weight']), (k, s['k_weight'])))
    page, place = s['slots'].long() // c['page'], s['slots'].long() % c['page']
    kc[page, :, place] = _rotate(k, cos, sin, c['rope']).to(kc.dtype)
    vc[page, :, place] = s['v'].to(vc.dtype)
    return [_rotate(q, cos, sin, c['rope']), kc, vc]


def _plain_attention(s):
    c, q, lengths = s['case'], s['q'], s['lengths'].long()
    (n, width), rows, nkv, hd, most = s['table'].shape, q.shape[0], c['kv_heads'], c['head_dim'], c['new']
    group, span = c['heads'] // nkv, width * c['page']
    pages = s['table'].clamp(min=0).long()
    s_ = torch.arange(span, device=q.device)
    keys, values = (x[pages].permute(0, 2, 1, 3, 4).reshape(n, nkv, span, hd).float()
                    for x in (s['k_cache'], s['v_cache']))
    values = torch.where((s_ < lengths[:, None])[:, None, :, None], values, 0.0)
    starts = torch.arange(n + 1, device=q.device) if s['starts'] is None else s['starts'].long()
    count = starts[1:] - starts[:-1]
    i = torch.arange(most, device=q.device)
    row = (starts[:-1, None] + i).clamp(max=rows - 1)
    x = q[row].view(n, most, nkv, group, hd).permute(0, 2, 1, 3, 4).reshape(n, nkv, most * group, hd)
    score = (x @ keys.transpose(2, 3) * (1 / math.sqrt(hd))).view(n, nkv, most, group, span)
    position = lengths[:, None] - count[:, None] + i
    seen = s_ <= position[..., None]
    if c['window']:
        seen &= s_ > position[..., None] - c['window']
    score = torch.where(seen[:, None, :, None, :], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(n, nkv, most * group, span)
    y = (p @ values).view(n, nkv, most, group, hd).permute(0, 2, 1, 3, 4).reshape(n, most, c['heads'], hd)
    t = torch.arange(rows, device=q.device)
    b = torch.searchsorted(starts[1:], t, right=True)
    y = y[b, t - starts[b]]
    return y if s['gate'] is None else y / (1 + torch.exp(-s['gate']))


def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] == 'extend':
        return _exact_extend(s)
    if case['kind'] == 'store':
        return _exact_store(s)
    return _exact_attention(s)


def _exact_extend(s):
    """Request by request and token by token, as a list of what each has and takes."""
    page = s['case']['page']
    table, free = s['table'].tolist(), s['free'].tolist()
    lengths, slots, positions, starts, used = [], [], [], [0], int(s['used'])
    for row, old, new in zip(table, s['lengths'].tolist(), s['new'].tolist()):
        for p in range(old, old + new):
            if p % page == 0:
                row[p // page] = free[used]
                used += 1
            slots.append(row[p // page] * page + p % page)
            positions.append(p)
        lengths.append(old + new)
        starts.append(len(slots))
    rest = [-1] * (s['tokens'] - len(slots))
    return [np.array(x, dtype=np.int32) for x in (lengths, [used], starts, slots + rest, positions + rest, [0], table)]


def _exact_store(s):
    """The rotation as a product of complex numbers."""
    c = s['case']
    n, page, hd = c['rotary'] // 2, c['page'], c['head_dim']
    turn = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'),
                       torch.outer(s['positions'].double(), s['freq']))[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / hd + EPS) * w.double()
        head, tail = x[..., :2 * n], x[..., 2 * n:]
        if c['rope'] == 'pairs':
            z = torch.complex(*head.unflatten(-1, (n, 2)).unbind(-1)) * turn
            return torch.cat([torch.stack([z.real, z.imag], -1).flatten(-2), tail], -1)
        z = torch.complex(*head.unflatten(-1, (2, n)).unbind(-2)) * turn
        return torch.cat([z.real, z.imag, tail], -1)

    q, k = turned(s['q'], s['q_weight']), turned(s['k'], s['k_weight'])
    caches = []
    for cache, x in ((s['k_cache'], k), (s['v_cache'], s['v'].double())):
        y = cache.double().transpose(1, 2).reshape(-1, c['kv_heads'], hd)
        y[s['slots'].long()] = x
        caches.append(y.view(-1, page, c['kv_heads'], hd).transpose(1, 2))
    return [q, *caches]


def _exact_attention(s):
    """One request after another, its pages joined to one run of positions."""
    c, q = s['case'], s['q'].double()
    nkv, hd, page = c['kv_heads'], c['head_dim'], c['page']
    group, out = c['heads'] // nkv, torch.zeros_like(q)
    starts = list(range(len(q) + 1)) if s['starts'] is None else s['starts'].tolist()
    for b, length in enumerate(s['lengths'].tolist()):
        rows = range(starts[b], starts[b + 1])
        if not length or not len(rows):
            continue
        ids = s['table'][b, :_pages(length, page)].long()
        keys, values = (torch.cat(x[ids].unbind(0), dim=1)[:, :length].double()
                        for x in (s['k_cache'], s['v_cache']))
        position = torch.arange(length - len(rows), length, device='cuda')
        at = torch.arange(length, device='cuda')
        gone = at[None, :] > position[:, None]
        if c['window']:
            gone |= at[None, :] <= position[:, None] - c['window']
        for h in range(c['heads']):
            score = q[rows.start:rows.stop, h] @ keys[h // group].t() / math.sqrt(hd)
            p = torch.softmax(score.masked_fill(gone, -math.inf), dim=-1)
            out[rows.start:rows.stop, h] = p @ values[h // group]
    return out if s['gate'] is None else out * torch.sigmoid(s['gate'].double())
