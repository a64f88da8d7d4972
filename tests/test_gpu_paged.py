"""The paged cache on the GPU against oracle/paged.py.

Tables: whole numbers, equal. Norm + rotation: a value is a sum of two products
of x, 1 / rms, the weight and a cosine: with u = 2^-24 the mean square carries
at most (3 + 6 + 2) u (a tree over 4 values and 64 lanes, the scale, eps), half
of it in the root, then the root, the quotient and two products, the cosine's
own 4 u and 2 pi 2^-25 of angle, and two more roundings: under 24 u of |a| + |b|;
an angle from a fp64 turn count of size n adds n 2^-52. The cache adds half a
step of its type. Attention: a score is off by at most (hd + 8) u of its sum of
|q k| (hd products and sums, the scale, the split query), a probability by
twice the largest of these (its own and the maximum's) plus (L + 64) u for the
exponential and the sums over L positions, and the output by the numerator's
and the denominator's, all times sum p |v|. That bounds every element; as
roundings are independent, the whole result is off far less: its 2-norm is held
to 1e-5 (a query or probability cut to one 11-bit or two 8-bit pieces, or one
dropped position of 100 000, is off by more)."""
import numpy as np
import pytest

from oracle import paged as opaged

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ['float32', 'float16', 'bfloat16']
HALF = {'float32': U, 'float16': 2.0 ** -11, 'bfloat16': 2.0 ** -8}


def _ints(x):
    import torch
    return torch.tensor(np.asarray(x, dtype=np.int32), device='cuda')


# ---------------------------------------------------------------- page tables

def _tables(rng, lengths, page, width, spare, pad=0):
    """Device and oracle tables of requests with `lengths` cached and a shuffled pool; pad: table columns behind."""
    held = [-(-x // page) for x in lengths]
    pool = sum(held) + spare
    free = rng.permutation(pool)
    table = np.full((len(lengths), width + pad), -1)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = free[at:at + n]
        at += n
    oracle = opaged.Tables(lengths, table[:, :width], free, at, page)
    return oracle, dict(lengths=_ints(lengths), table=_ints(table)[:, :width], free=_ints(free), used=_ints([at]))


def _extend_both(oracle, d, new, tokens, page, in_place):
    from localai_amd import paged
    import torch
    out = None
    if in_place:
        e = lambda n: torch.empty(n, dtype=torch.int32, device='cuda')
        out = paged.Step(d['lengths'], d['used'], e(len(new) + 1), e(tokens), e(tokens), e(1))
    before = d['lengths'].clone(), d['used'].clone()
    step = paged.extend(d['lengths'], _ints(new), d['table'], d['free'], d['used'], page, tokens, out=out)
    status, starts, slots, positions = oracle.extend(new, tokens)
    if not in_place:
        assert torch.equal(d['lengths'], before[0]) and torch.equal(d['used'], before[1])
    np.testing.assert_array_equal(step.status.cpu(), [status])
    np.testing.assert_array_equal(step.starts.cpu(), starts)
    np.testing.assert_array_equal(step.positions.cpu(), positions)
    np.testing.assert_array_equal(step.slots.cpu(), slots)
    np.testing.assert_array_equal(step.lengths.cpu(), oracle.lengths)
    np.testing.assert_array_equal(step.used.cpu(), [oracle.used])
    np.testing.assert_array_equal(d['table'].cpu(), oracle.table)
    d['lengths'], d['used'] = step.lengths, step.used
    return step


@pytest.mark.parametrize('in_place', [False, True])
@pytest.mark.parametrize('lengths,new,page,spare', [
    ([0], [1], 16, 1), ([15], [1], 16, 0), ([16], [1], 16, 1), ([0], [0], 16, 1),
    ([5, 0, 16, 31, 0], [11, 0, 1, 2, 40], 16, 9),
    ([0, 0, 0], [0, 100, 0], 64, 5),
    ([7] * 70, [1] * 70, 32, 3),
    ([1, 4095, 300], [5000, 1, 700], 16, 400),          # several workgroups
    ([0] * 5, [1024, 0, 1, 1023, 2049], 128, 40),
])
def test_extend(lengths, new, page, spare, in_place):
    rng = np.random.default_rng(len(lengths) + sum(new))
    width = max(1, max(-(-(a + b) // page) for a, b in zip(lengths, new))) + 2
    oracle, d = _tables(rng, lengths, page, width, spare, pad=3)
    _extend_both(oracle, d, new, sum(new), page, in_place)
    oracle, d = _tables(rng, lengths, page, width, spare)
    _extend_both(oracle, d, new, sum(new) + 7, page, in_place)


@pytest.mark.parametrize('n', [63, 64, 65, 256, 1023, 1024, 1025, 4096])
def test_extend_many_requests_over_steps(n):
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, 100, n).tolist()
    oracle, d = _tables(rng, lengths, 16, 12, 6 * n)
    for _ in range(3):
        new = np.where(rng.random(n) < 0.3, 0, rng.integers(0, 25, n)).tolist()
        _extend_both(oracle, d, new, sum(new) + 3, 16, in_place=True)


@pytest.mark.parametrize('big', [False, True])
@pytest.mark.parametrize('fault', ['pool', 'width', 'tokens', 'negative new', 'negative length', 'used'])
def test_extend_that_does_not_fit_changes_nothing(fault, big):
    import torch
    from localai_amd import paged
    rng = np.random.default_rng(3)
    lengths, new = [20, 3, 0], [13, 4000 if big else 40, 5]
    width = 300
    oracle, d = _tables(rng, lengths, 16, width, 1 if fault == 'pool' else 300)
    tokens = sum(new)
    want = {'pool': 1, 'width': 2, 'tokens': 4, 'negative new': 2, 'negative length': 2, 'used': 2}[fault]
    if fault == 'width':
        d['table'] = d['table'][:, :2]
    if fault == 'tokens':
        tokens -= 1
    if fault == 'negative new':
        new[2] = -1
    if fault == 'negative length':
        d['lengths'][1] = -4
    if fault == 'used':
        d['used'][0] = -1
    kept = {k: v.clone() for k, v in d.items()}
    step = paged.extend(d['lengths'], _ints(new), d['table'], d['free'], d['used'], 16, tokens)
    assert int(step.status) & want
    assert torch.equal(step.lengths, kept['lengths']) and torch.equal(step.used, kept['used'])
    assert torch.equal(d['table'], kept['table']) and torch.equal(d['free'], kept['free'])
    assert not step.starts.any() and (step.slots == -1).all() and (step.positions == -1).all()
    with pytest.raises(RuntimeError, match='nothing was changed'):
        step.check()


def test_extend_gives_no_slot_for_pages_outside_the_pool():
    from localai_amd import paged
    table, free = _ints([[9, -1], [-7, -1], [1, -1]]), _ints([0, 99, 1, 2])
    step = paged.extend(_ints([3, 3, 16]), _ints([2, 2, 2]), table, free, _ints([1]), 16, 6)
    np.testing.assert_array_equal(step.slots.cpu(), [-1, -1, -1, -1, -1, -1])   # pages 9, -7, and 99 from the list
    np.testing.assert_array_equal(step.positions.cpu(), [3, 4, 3, 4, 16, 17])


@pytest.mark.parametrize('n', [1, 5, 64, 1500])
def test_shrink(n):
    from localai_amd import paged
    rng = np.random.default_rng(n)
    oracle, d = _tables(rng, rng.integers(0, 700, n).tolist(), 16, 60, 40 * n)
    for _ in range(2):
        before = {k: v.clone() for k, v in d.items()}
        new = rng.integers(0, 90, n).tolist()
        kept = list(oracle.lengths)
        _extend_both(oracle, d, new, sum(new), 16, in_place=True)
        status = paged.shrink(d['lengths'], _ints(kept), d['table'], d['free'], d['used'], 16)   # drafts taken back
        oracle.shrink(kept)
        for k in d:
            assert bool((d[k] == before[k]).all()), k
        keep = rng.integers(0, 800, n).tolist()
        paged.shrink(d['lengths'], _ints(keep), d['table'], d['free'], d['used'], 16)
        oracle.shrink(keep)
        assert int(status) == 0
        np.testing.assert_array_equal(d['lengths'].cpu(), oracle.lengths)
        np.testing.assert_array_equal(d['table'].cpu(), oracle.table)
        np.testing.assert_array_equal(d['free'].cpu(), oracle.free)
        assert int(d['used']) == oracle.used


@pytest.mark.parametrize('n', [1, 5, 64, 1500])
def test_shrink_says_that_it_was_done(n):
    """Status 0 of drafts taken back and of a second cut, from a buffer that held something else."""
    import torch
    from localai_amd import paged
    rng = np.random.default_rng(n + 1)
    oracle, d = _tables(rng, rng.integers(0, 700, n).tolist(), 16, 60, 40 * n)
    kept = list(oracle.lengths)
    new = rng.integers(0, 90, n).tolist()
    _extend_both(oracle, d, new, sum(new), 16, in_place=True)
    for keep in (kept, rng.integers(0, 800, n).tolist(), [0] * n):
        torch.full((1,), 77, dtype=torch.int32, device='cuda')
        status = paged.shrink(d['lengths'], _ints(keep), d['table'], d['free'], d['used'], 16)
        oracle.shrink(keep)
        assert int(status) == 0
        paged.check(status)
        np.testing.assert_array_equal(d['lengths'].cpu(), oracle.lengths)
        np.testing.assert_array_equal(d['free'].cpu(), oracle.free)
    assert int(d['used']) == 0 and (d['table'] == -1).all()


@pytest.mark.parametrize('fault,want', [('keep', 2), ('length', 2), ('used', 1), ('pool', 2)])
def test_shrink_that_cannot_be_changes_nothing(fault, want):
    import torch
    from localai_amd import paged
    _, d = _tables(np.random.default_rng(1), [40, 20], 16, 4, 3)
    keep = _ints([3, 2])
    if fault == 'keep':
        keep[1] = -1
    if fault == 'length':
        d['lengths'][0] = 65
    if fault == 'used':
        d['used'][0] = 2
    if fault == 'pool':
        d['used'][0] = 99
    kept = {k: v.clone() for k, v in d.items()}
    status = paged.shrink(d['lengths'], keep, d['table'], d['free'], d['used'], 16)
    assert int(status) & want
    for k in d:
        assert torch.equal(d[k], kept[k]), k


# ---------------------------------------------------------------- norm, rotation, store

def _store(tokens, heads, dtype, page, rope, n, norm, seed=0, views=False, token_major=False, pad=(), far=0,
           in_place=False):
    import torch
    from localai_amd import paged
    nh, nkv, hd = heads
    rng = np.random.default_rng(seed)
    q, k, v = (rng.standard_normal((tokens, h, hd)).astype(np.float32) * s for h, s in ((nh, 3), (nkv, .1), (nkv, 1)))
    w = [(1 + .2 * rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2)]
    freq = 10000.0 ** (-np.arange(n) / max(n, 1))
    positions = far + rng.permutation(4 * tokens)[:tokens]
    pool = -(-tokens // page) + 2
    slots = rng.permutation(pool * page)[:tokens]
    for i, s in pad:
        slots[i] = s
    tt = getattr(torch, dtype)
    shape = (pool, page, nkv, hd) if token_major else (pool, nkv, page, hd)
    caches = [torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda().to(tt) for _ in range(2)]
    kc, vc = (c.transpose(1, 2) if token_major else c for c in caches)
    kc0, vc0 = kc.clone(), vc.clone()
    dq, dk, dv = (torch.from_numpy(x).cuda() for x in (q, k, v))
    if views:
        fused = torch.cat([x.reshape(tokens, -1) for x in (dq, dk, dv)], 1)
        dq, dk, dv = (x.view(tokens, -1, hd) for x in fused.split([nh * hd, nkv * hd, nkv * hd], 1))
    out = dq if in_place else torch.full((tokens, nh, hd), 7.0, device='cuda')
    dev = lambda a: torch.from_numpy(a).cuda() if a is not None else None
    got = paged.norm_rope_store(dq, dk, dv, _ints(positions), _ints(slots), kc, vc, dev(freq) if n else None,
                                dev(w[0]), dev(w[1]), eps=1e-6, rope=rope, out=out)
    assert got is out
    torch.cuda.synchronize()
    turns = 1 + abs(positions).max() / 6
    tol = 24 * U + 2 ** -52 * turns * 8

    def near(y, x, want, raw, half):
        raw = np.abs(raw).max(-1, keepdims=True) * 2     # |a| + |b| of a rotated pair
        assert (np.abs(y - want) <= tol * raw + half * (np.abs(want) + tol * raw) + 2.0 ** -24 * (half > U)).all()

    skip = {i for i, _ in pad}
    yq = got.cpu().numpy()
    yk, yv = kc.float().cpu().numpy(), vc.float().cpu().numpy()
    seen = np.zeros((pool, page), bool)
    for t in range(tokens):
        if t in skip:
            np.testing.assert_array_equal(yq[t], q[t] if in_place else np.full((nh, hd), 7.0, np.float32))
            continue
        wq, wk = (opaged.norm_rope(x[t], positions[t], freq, ww, 1e-6, rope) for x, ww in ((q, w[0]), (k, w[1])))
        at = divmod(int(slots[t]), page)
        seen[at] = True
        near(yq[t], q[t], wq, wq, 0)
        near(yk[at[0], :, at[1]], k[t], wk, wk, HALF[dtype])
        want_v = torch.from_numpy(v[t]).to(tt).float().numpy()
        np.testing.assert_array_equal(yv[at[0], :, at[1]], want_v)
    rest = torch.from_numpy(~seen).cuda()
    for c, c0 in ((kc, kc0), (vc, vc0)):                  # every other place of the cache as it was
        assert torch.equal(c.transpose(1, 2)[rest], c0.transpose(1, 2)[rest])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rope', ['halves', 'pairs'])
@pytest.mark.parametrize('heads,n,norm', [((32, 8, 128), 64, True), ((16, 4, 256), 32, True), ((8, 8, 64), 32, False),
                                          ((6, 2, 64), 10, True), ((4, 4, 256), 128, False), ((3, 1, 128), 1, True),
                                          ((28, 4, 128), 63, True), ((1, 1, 64), 0, True)])
def test_norm_rope_store(heads, n, norm, rope, dtype):
    _store(5, heads, dtype, 16, rope, n, norm, seed=n)


@pytest.mark.parametrize('tokens', [1, 2, 63, 500])
def test_norm_rope_store_of_views(tokens):
    _store(tokens, (32, 8, 128), 'float16', 32, 'halves', 64, True, seed=tokens, views=True)
    _store(tokens, (16, 4, 256), 'bfloat16', 64, 'pairs', 32, True, seed=tokens, views=True, token_major=True)


@pytest.mark.parametrize('rope,n', [('halves', 32), ('halves', 10), ('pairs', 32)])
def test_norm_rope_store_in_place_with_padding(rope, n):
    pad = [(0, -1), (3, 2 ** 31 - 1), (6, 3 * 16), (4, -2 ** 31)]   # 7 tokens: a pool of 3 pages, 48 slots
    _store(7, (6, 2, 64), 'float16', 16, rope, n, True, pad=pad, in_place=True)
    _store(7, (6, 2, 64), 'float32', 16, rope, n, False, pad=pad, views=True, in_place=True)
    _store(7, (6, 2, 64), 'bfloat16', 16, rope, n, True, pad=pad)


@pytest.mark.parametrize('far', [100_000, 10_000_000, 2_000_000_000])
def test_norm_rope_store_at_far_positions(far):
    _store(9, (8, 2, 128), 'float32', 16, 'pairs', 64, True, far=far, seed=9)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rope,n', [('halves', 0), ('halves', 12), ('halves', 10), ('pairs', 12), ('pairs', 7),
                                    ('pairs', 0)])
def test_store_leaves_values_that_are_not_rotated_as_they_are(rope, n, dtype):
    """Infinities, NaN and negative zeros behind the rotated values stay, and stay where they are."""
    import torch
    from localai_amd import paged
    hd, nh, nkv, tokens = 64, 4, 2, 5
    gen = torch.Generator('cuda').manual_seed(n)
    q, k, v = (torch.randn((tokens, h, hd), generator=gen, device='cuda') for h in (nh, nkv, nkv))
    freq = torch.from_numpy(100.0 ** (-np.arange(n) / max(n, 1))).cuda() if n else None
    tt = getattr(torch, dtype)

    def run(q, k):
        kc, vc = (torch.zeros((1, nkv, 16, hd), dtype=tt, device='cuda') for _ in range(2))
        y = paged.norm_rope_store(q, k, v, _ints(range(3, 3 + tokens)), _ints(range(tokens)), kc, vc, freq, rope=rope)
        return y, kc[0, :, :tokens].transpose(0, 1)

    clean = run(q, k)
    for x in (q, k):
        x[:, 0, 2 * n + 1], x[:, 1, 2 * n + 2], x[:, 1, hd - 1] = float('inf'), float('-inf'), float('nan')
        x[:, 0, 2 * n + 6] = -0.0
    for got, was, x in zip(run(q, k), clean, (q, k)):
        assert torch.equal(got[..., :2 * n], was[..., :2 * n])
        want = x[..., 2 * n:].to(got.dtype)
        assert torch.equal(got[..., 2 * n:].isnan(), want.isnan())
        assert torch.equal(got[..., 2 * n:].nan_to_num(7.0), want.nan_to_num(7.0))
        assert torch.equal(torch.signbit(got[..., 2 * n:])[~want.isnan()], torch.signbit(want)[~want.isnan()])


def test_store_refuses_outputs_that_overlap():
    import torch
    from localai_amd import _lib, paged
    q, k = torch.zeros((2, 4, 64), device='cuda'), torch.zeros((2, 2, 64), device='cuda')
    kc, vc = (torch.zeros((1, 2, 16, 64), device='cuda') for _ in range(2))
    for out in (q[:1].expand(2, -1, -1), q[:, :1].expand(-1, 4, -1), torch.zeros(600, device='cuda').as_strided((2, 4, 64), (192, 64, 1))):
        with pytest.raises(_lib.HipError, match='overlap'):
            paged.norm_rope_store(q, k, k, _ints([0, 1]), _ints([0, 1]), kc, vc, out=out)


def test_store_rounds_as_the_type_does():
    """Values past fp16's range become infinite; zero rows keep the norm finite."""
    import torch
    from localai_amd import paged
    k = torch.tensor([1e6, -1e6, 65519.0, 65520.0] + [0.0] * 60, device='cuda').view(1, 1, 64)
    kc, vc = (torch.zeros((1, 1, 16, 64), dtype=torch.float16, device='cuda') for _ in range(2))
    q = torch.zeros((1, 2, 64), device='cuda')
    w = torch.ones(64, device='cuda')
    y = paged.norm_rope_store(q, k, k, _ints([0]), _ints([3]), kc, vc, q_weight=w)
    assert torch.equal(y, q)
    want = torch.zeros(64, dtype=torch.float16, device='cuda')
    want[:4] = torch.tensor([float('inf'), float('-inf'), 65504.0, float('inf')])
    assert torch.equal(kc[0, 0, 3], want) and torch.equal(vc[0, 0, 3], want)
    assert not kc[0, 0, :3].any() and not kc[0, 0, 4:].any()


# ---------------------------------------------------------------- attention

def _pages(rng, lengths, page, width, spare=3):
    held = [-(-x // page) for x in lengths]
    ids = rng.permutation(sum(held) + spare)
    table = np.full((len(lengths), width), -1)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, len(ids)


def _attention(heads, lengths, dtype, page=16, new=None, window=0, gate=False, scale=None, seed=0, token_major=False,
               behind=0, q_size=2.0, nan=True, check=True):
    import torch
    from localai_amd import paged
    nh, nkv, hd = heads
    rng = np.random.default_rng(seed)
    width = max(1, max(-(-x // page) for x in lengths)) + 1
    table, pool = _pages(rng, lengths, page, width)
    tt = getattr(torch, dtype)
    shape = (pool, page, nkv, hd) if token_major else (pool, nkv, page, hd)
    gen = torch.Generator('cuda').manual_seed(seed)
    kc, vc = (torch.randn(shape, generator=gen, device='cuda').to(tt) for _ in range(2))
    if token_major:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    dt = _ints(table)
    runs = []
    unseen = torch.ones((pool, page), dtype=torch.bool, device='cuda')
    for b, n in enumerate(lengths):
        ids = dt[b, :-(-n // page)].long()
        runs.append([x[ids].transpose(1, 2).reshape(-1, nkv, hd)[:n].double().cpu().numpy() for x in (kc, vc)])
        flat = (ids[:, None] * page + torch.arange(page, device='cuda')).reshape(-1)[:n]
        unseen.view(-1)[flat] = False
    if nan:                             # what no row sees may be anything
        kc.transpose(1, 2)[unseen] = float('nan')
        vc.transpose(1, 2)[unseen] = float('inf')
    count = [1] * len(lengths) if new is None else new
    rows = sum(count)
    q = (rng.standard_normal((rows + behind, nh, hd)) * q_size).astype(np.float32)
    g = rng.standard_normal((rows + behind, nh, hd)).astype(np.float32) * 3 if gate else None
    starts = None if new is None else _ints(np.concatenate([[0], np.cumsum(count)]))
    out = torch.full((rows + behind, nh, hd), 5.0, device='cuda')
    args = (torch.from_numpy(q).cuda(), kc, vc, dt, _ints(lengths))
    kw = dict(starts=starts, window=window, scale=scale, gate=torch.from_numpy(g).cuda() if gate else None)
    got = paged.attention(*args, out=out, **kw)
    assert got is out
    torch.cuda.synchronize()
    y = got.cpu().numpy()
    want, bound = np.zeros_like(q, np.float64), np.zeros_like(q, np.float64)
    at = 0
    for (k, v), n, c in zip(runs, lengths, count):
        o, weight, spread = opaged.attention(q[at:at + c], k, v, c, scale or opaged.default_scale(hd), window,
                                             g[at:at + c] if gate else None)
        want[at:at + c] = o
        bound[at:at + c] = weight * (4 * (hd + 8) * U * spread[..., None] + 2 * (n + 64) * U)
        at += c
    assert np.isfinite(y).all()
    assert (np.abs(y[:rows] - want[:rows]) <= bound[:rows]).all()
    rel = np.linalg.norm(y[:rows] - want[:rows]) / max(np.linalg.norm(want[:rows]), 1e-30)
    print(f'paged attention {heads} {lengths[:6]} {dtype}: {rel:.2e}')
    assert rel <= 1e-5
    assert (y[rows:] == 5.0).all()
    return args, kw, y


HEADS = [(32, 8, 128), (8, 8, 64), (6, 2, 64), (28, 4, 128), (16, 4, 256), (64, 8, 128), (4, 4, 256), (9, 1, 128),
         (16, 1, 64), (17, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', HEADS)
def test_attention_heads(heads, dtype):
    _attention(heads, [1, 0, 16, 33, 200, 15], dtype, seed=heads[0])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('length', [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513,
                                    1025, 4096])
def test_attention_lengths(length, dtype):
    _attention((8, 2, 128), [length], dtype, page=32, seed=length)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('page', [16, 64, 256])
def test_attention_ragged_batch(page, dtype):
    rng = np.random.default_rng(page)
    lengths = [int(x) for x in np.exp(rng.uniform(0, np.log(3000), 37))]
    lengths[5] = lengths[20] = 0
    _attention((8, 2, 64), lengths, dtype, page=page, seed=page, token_major=page == 64)


@pytest.mark.parametrize('n', [63, 64, 65, 200, 1100, 4096])
def test_attention_many_requests(n):
    rng = np.random.default_rng(n)
    _attention((2, 1, 64), rng.integers(0, 70, n).tolist(), 'float16', seed=n)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [65, 130, 300])
def test_attention_many_requests_of_several_chunks(n, dtype):
    """More requests than a wave has lanes, some long: several requests per lane, each cut by its length."""
    rng = np.random.default_rng(n)
    lengths = np.exp(rng.uniform(0, np.log(2500), n)).astype(int).tolist()
    lengths[3] = lengths[n - 1] = 0
    lengths[7] = 2500
    _attention((2, 1, 64), lengths, dtype, seed=n)
    new = [min(x, y) for x, y in zip(lengths, rng.integers(0, 4, n).tolist())]
    _attention((4, 2, 64), lengths, dtype, new=new, seed=n + 1, window=900)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [12, 64, 300])
def test_attention_few_of_many_places(n, dtype):
    """A batch whose places are mostly empty, of a few requests cut into many chunks, first, last and between."""
    lengths = [0] * n
    for b, x in ((0, 9000), (n // 3, 40), (n // 2, 3001), (n - 1, 6000)):
        lengths[b] = x
    _attention((8, 8, 64), lengths, dtype, page=64, seed=n)
    _attention((4, 2, 128), lengths, dtype, page=64, new=[min(x, 2) for x in lengths], seed=n + 1)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads,tokens', [((2, 1, 64), 40), ((16, 16, 64), 40), ((8, 2, 128), 90)])
def test_attention_many_requests_of_several_blocks(heads, tokens, dtype):
    """More requests than a wave has lanes, several blocks of tokens each, some cut: with one and two column sets."""
    rng = np.random.default_rng(tokens)
    lengths = np.exp(rng.uniform(0, np.log(160), 70)).astype(int).tolist()
    for b, x in ((2, 3000), (3, 2100), (69, 4000)):
        lengths[b] = x
    lengths[5] = lengths[68] = 0
    new = [min(x, int(y)) for x, y in zip(lengths, rng.integers(1, tokens, 70))]
    new[2] = new[69] = tokens
    new[9] = 0
    _attention(heads, lengths, dtype, page=32, new=new, seed=1, behind=2)
    _attention(heads, lengths, dtype, page=32, new=new, seed=2, window=1500)


@pytest.mark.parametrize('window', [0, 700])
@pytest.mark.parametrize('heads', [(8, 8, 64), (32, 32, 64)])
def test_attention_with_many_rows_of_padding(heads, window):
    """Rows behind the last request count for the layout, not for the chunks."""
    _attention(heads, [2500, 60, 1200], 'float16', new=[60, 60, 40], behind=2000, window=window, seed=3)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('window', [1, 2, 17, 128, 1000, 2 ** 40])
def test_attention_window(window, dtype):
    _attention((8, 2, 128), [1, 16, 700, 129, 2000], dtype, window=window, seed=window % 1000)
    _attention((8, 2, 128), [1, 300, 700], dtype, new=[1, 70, 0], window=window, seed=window % 1000 + 1)


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_gate_and_scale(dtype):
    _attention((16, 4, 256), [300, 1, 0, 77], dtype, gate=True, seed=5)
    _attention((16, 4, 256), [300, 5, 0, 77], dtype, gate=True, new=[20, 5, 0, 1], seed=6)
    _attention((8, 8, 64), [300, 77], dtype, scale=0.31, q_size=1.0, seed=7)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', [(32, 8, 128), (6, 2, 64), (16, 4, 256), (8, 8, 64), (7, 1, 128), (20, 1, 64),
                                   (64, 8, 128)])
def test_attention_several_tokens(heads, dtype):
    _attention(heads, [50, 1, 129, 33, 0, 400], dtype, new=[50, 1, 3, 33, 0, 17], behind=3, seed=heads[0])


@pytest.mark.parametrize('new', [[1, 1, 1], [0, 5, 0], [2, 0, 0], [64, 64, 64], [100, 1, 300], [16, 8, 4]])
def test_attention_piece_sizes(new):
    _attention((8, 2, 128), [300, 64, 301], 'float16', new=new, behind=1, page=64, seed=sum(new))
    _attention((8, 2, 128), [300, 64, 301], 'bfloat16', new=new, seed=sum(new), window=40)


# prompts large enough for the kernel's layout with two sets of columns a workgroup: (heads, lengths, new)
PROMPTS = [((32, 32, 64), [300, 130, 70, 0], [200, 100, 70, 0]),
           ((64, 32, 128), [150, 33, 260], [150, 33, 90]),
           ((32, 32, 256), [90, 140, 41], [90, 100, 41]),
           ((40, 2, 64), [210, 5, 1], [200, 5, 1]),
           ((51, 17, 64), [310, 64], [260, 64])]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads,lengths,new', PROMPTS)
def test_attention_prompts(heads, lengths, new, dtype):
    _attention(heads, lengths, dtype, new=new, behind=2, seed=heads[0])
    _attention(heads, lengths, dtype, new=new, window=37, gate=True, page=64, seed=heads[0] + 1, token_major=True)


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_prompts_beside_a_long_request(dtype):
    """One request far longer than the rest: its blocks are cut into chunks and joined, the others' are not."""
    _attention((32, 32, 64), [6000, 130, 150], dtype, new=[3, 130, 120], seed=1)
    _attention((64, 32, 128), [60, 2500, 60, 61], dtype, new=[60, 40, 60, 61], seed=2, page=32, gate=True)


def test_attention_prompts_with_bad_pages():
    import torch
    from localai_amd import paged
    (q, kc, vc, table, dl), kw, y = _attention((32, 32, 64), [200, 150, 170], 'float16', new=[150, 150, 100], nan=False)
    table = table.clone()
    table[1, 4] = 10 ** 6                # positions 64 to 79 of request 1
    bad = paged.attention(q, kc, vc, table, dl, **kw).cpu().numpy()
    np.testing.assert_array_equal(bad[:150], y[:150])
    np.testing.assert_array_equal(bad[300:], y[300:])
    assert np.isnan(bad[150 + 64:300]).all()
    np.testing.assert_array_equal(bad[150:150 + 64], y[150:150 + 64])   # tokens before the bad page do not see it


def test_attention_fewer_positions_than_tokens_sees_nothing():
    """A length below the count of new tokens: the first of them lie before position 0 and are zeros."""
    _attention((8, 2, 64), [3, 40], 'float16', new=[5, 2], seed=1)


def test_attention_rows_ahead_of_the_first_request_stay():
    import torch
    from localai_amd import paged
    (q, kc, vc, table, dl), kw, y = _attention((8, 2, 64), [2000, 40], 'float16', new=[3, 2], seed=5)
    out = torch.full((9, 8, 64), 5.0, device='cuda')
    qq = torch.cat([q[:1], q[:1], q, q[:2]])
    paged.attention(qq, kc, vc, table, dl, starts=_ints([2, 5, 7]), out=out)
    np.testing.assert_array_equal(out[2:7].cpu(), y)
    assert (out[:2] == 5.0).all() and (out[7:] == 5.0).all()


def test_attention_window_past_every_length():
    import torch
    from localai_amd import paged
    args, kw, y = _attention((8, 2, 64), [300, 1, 33], 'float16', seed=6)
    for window in (300, 2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1, 2 ** 70, -1):
        np.testing.assert_array_equal(paged.attention(*args, window=window).cpu(), y)
    with pytest.raises(ValueError, match='page_size'):
        paged.extend(args[4], args[4], args[3], args[4], args[4][:1], 2 ** 32 + 16, 4)


@pytest.mark.parametrize('scale', [0.0, -0.2])
def test_attention_scale_of_zero_and_below(scale):
    import torch
    from localai_amd import paged
    (q, kc, vc, table, dl), _, _ = _attention((8, 2, 64), [300, 1, 33], 'float16', seed=6)
    y = paged.attention(q, kc, vc, table, dl, scale=scale).cpu().numpy()
    for b, n in enumerate([300, 1, 33]):
        k, v = (x[table[b, :-(-n // 16)].long()].transpose(1, 2).reshape(-1, 2, 64)[:n].double().cpu().numpy()
                for x in (kc, vc))
        want = opaged.attention(q[b:b + 1].cpu().numpy(), k, v, 1, scale)[0][0]
        assert np.linalg.norm(y[b] - want) <= 1e-5 * np.linalg.norm(want)


def test_attention_one_long_request():
    _attention((8, 2, 128), [70_001], 'float16', page=64, seed=2)
    _attention((4, 1, 64), [33_000, 5, 9000], 'bfloat16', page=16, seed=3)


def test_attention_small_scores_of_many_positions():
    """A peak of one position against thousands far below it: the small probabilities keep their share."""
    _attention((4, 1, 128), [5000], 'float16', q_size=6.0, seed=8)
    _attention((4, 1, 128), [5000], 'bfloat16', q_size=0.01, seed=9)


@pytest.mark.parametrize('q_size', [1e-6, 300.0])
def test_attention_query_sizes(q_size):
    """Queries far from 1: the split into pieces follows their size."""
    _attention((8, 2, 64), [100, 31], 'float16', q_size=q_size, scale=1 / q_size, seed=4)
    _attention((8, 2, 64), [100, 31], 'bfloat16', q_size=q_size, scale=1 / q_size, seed=4)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('new', [None, [1, 40, 1, 7]])
def test_attention_bad_pages_are_nan_and_others_unharmed(new, dtype):
    import torch
    from localai_amd import paged
    lengths = [900, 640, 100, 333]
    (q, kc, vc, table, dl), kw, y = _attention((8, 2, 128), lengths, dtype, page=16, new=new, nan=False, seed=11)
    table = table.clone()
    table[0, 30] = kc.shape[0]           # one past the pool
    table[1, 0] = -1
    table[3, :] = 2 ** 31 - 1
    bad = paged.attention(q, kc, vc, table, dl, **kw)
    count = new or [1] * 4
    at = 0
    for b, c in enumerate(count):
        rows = bad[at:at + c]
        if b == 2:
            np.testing.assert_array_equal(rows.cpu(), y[at:at + c])
        else:
            assert torch.isnan(rows).all()
        at += c
    dl = dl.clone()
    dl[2] = table.shape[1] * 16 + 1      # a position past the table
    bad = paged.attention(q, kc, vc, table, dl, **kw)
    at = sum(count[:2])
    assert torch.isnan(bad[at:at + count[2]][-1]).all()
    table[0, 30] = 0                     # a page that a window does not reach is not looked at
    table[0, :20] = -9
    if new is None:
        got = paged.attention(q, kc, vc, table, dl, window=500)
        assert torch.isfinite(got[0]).all()


# (heads, lengths, new, window): decode batches, drafts, prompts of one and of two column sets, head_dim 256
LEAKS = [((8, 2, 128), [300, 64], [40, 9], 0), ((8, 2, 128), [300, 64], [40, 9], 19), ((6, 2, 64), [90, 33], [90, 33], 0),
         ((16, 4, 256), [120, 50], [50, 7], 30), ((8, 2, 64), [70, 40, 20], [3, 0, 0], 0), ((8, 8, 64), [700], None, 80),
         ((32, 32, 64), [300, 130, 70], [200, 100, 70], 0), ((64, 32, 128), [150, 33, 260], [150, 33, 90], 37),
         ((9, 1, 128), [2500, 700], [20, 30], 0),
         ((32, 32, 64), [2600, 300], [200, 160], 1500)]     # two column sets, cut, windows that end inside a chunk


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads,lengths,new,window', LEAKS)
def test_attention_values_that_are_not_finite_reach_only_rows_that_see_them(heads, lengths, new, window, dtype):
    """An infinity or NaN in v: that value of the rows and heads that see it is not finite, every other result keeps
    its bits, whatever tokens share the row's tile. In k: the rows that see a NaN are NaN."""
    from localai_amd import paged
    nh, nkv, hd = heads
    (q, kc, vc, table, dl), kw, y = _attention(heads, lengths, dtype, new=new, window=window, nan=False, seed=31)
    pages, group = table.cpu().numpy(), nh // nkv
    count, at = new or [1] * len(lengths), 0
    rng = np.random.default_rng(7)
    for b, (length, n) in enumerate(zip(lengths, count)):
        first = length - n
        spots = {length - 1, first, first + n // 2, max(0, first + 1 - (window or length)), max(0, first - 3)}
        for s in sorted(spots):
            kh, d, bad = int(rng.integers(nkv)), int(rng.integers(hd)), rng.choice([np.inf, -np.inf, np.nan])
            place = (int(pages[b, s // 16]), kh, s % 16, d)
            p = first + np.arange(n)
            sees = np.zeros(len(q), bool)
            sees[at:at + n] = (p >= s) & ((p - s < window) if window else True)
            for cache, value in ((vc, float(bad)), (kc, float('nan'))):
                kept = cache[place].clone()
                cache[place] = value
                got = paged.attention(q, kc, vc, table, dl, **kw).cpu().numpy()
                cache[place] = kept
                hit = np.zeros(y.shape, bool)
                hit[sees, kh * group:(kh + 1) * group, slice(d, d + 1) if cache is vc else slice(None)] = True
                assert not np.isfinite(got[hit]).any(), (b, s, value)
                if cache is kc:
                    assert np.isnan(got[hit]).all(), (b, s)
                np.testing.assert_array_equal(got[~hit], y[~hit], err_msg=f'request {b} position {s} {value}')
        at += n


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads,lengths,new', [((8, 2, 64), [1, 40], None), ((8, 2, 64), [2500, 900], None),
                                               ((8, 8, 64), [600, 2500], [700, 300]), ((4, 2, 64), [290, 700], [300, 2]),
                                               ((32, 32, 64), [300, 130], [320, 100])])
def test_attention_rows_whose_scores_are_all_minus_infinity_are_nan(heads, lengths, new, dtype):
    """Rows that see positions, but every score is -inf, are NaN as the softmax is; rows that see nothing are zeros,
    whole or joined from chunks."""
    import torch
    from localai_amd import paged
    nh, nkv, hd = heads
    (q, kc, vc, table, dl), kw, y = _attention(heads, lengths, dtype, new=new, nan=False, seed=4)
    q = q.clone()
    q[:, :, 3] = 1.0
    ids = table[0, :-(-lengths[0] // 16)].long()
    kc[ids, :, :, 3] = float('-inf')
    got = paged.attention(q, kc, vc, table, dl, **kw).cpu().numpy()
    count = new or [1] * len(lengths)
    none = max(0, count[0] - lengths[0])             # its rows ahead of position 0
    assert (got[:none] == 0).all()
    assert np.isnan(got[none:count[0]]).all()
    assert np.isfinite(got[count[0]:]).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads,lengths,new', [((8, 2, 64), [1, 2, 40, 700], None), ((4, 2, 128), [3, 2500], [2, 1]),
                                               ((32, 32, 64), [300, 130, 70], [200, 100, 70]),
                                               ((64, 8, 128), [900, 60], [40, 60]), ((4, 4, 256), [20, 33], [5, 33])])
def test_attention_infinite_scores(heads, lengths, new, dtype):
    """An infinite k: a score of -inf has probability 0, one of inf makes the row NaN, and so does a row of nothing
    but -inf (the softmax's 0 / 0). q's values are small multiples of 1/8: all their low bits are zero. Beside f16, a
    value of q below 2^-34 of the largest is 0 (2^-24 where the largest is 2^9 to 2^10), and 0 times infinity NaN."""
    import torch
    from localai_amd import paged
    nh, nkv, hd = heads
    group = nh // nkv
    (q, kc, vc, table, dl), kw, _ = _attention(heads, lengths, dtype, new=new, nan=False, seed=3)
    q = torch.round(q * 4) / 8
    q[:, :, 5] = torch.where(q[:, :, 5] == 0, 0.125, q[:, :, 5])
    q[:, :, 9] *= 2.0 ** -40             # far below the row's largest
    pages, count = table.cpu().numpy(), new or [1] * len(lengths)
    rng = np.random.default_rng(8)

    def place(b, s, kh, d):
        return int(pages[b, s // 16]), kh, s % 16, d

    planted = {}
    for b, length in enumerate(lengths):
        for s in {0, length // 2, length - 1}:
            for kh in range(nkv):
                d = int(rng.choice([5, 9]))
                planted[b, s, kh] = d, float(rng.choice([np.inf, -np.inf]))
                kc[place(b, s, kh, d)] = planted[b, s, kh][1]
    got = paged.attention(q, kc, vc, table, dl, **kw).cpu().numpy()
    qn, at, kinds = q.double().cpu().numpy(), 0, set()
    if dtype == 'float16':
        qn[:, :, 9] = 0
    for b, (length, n) in enumerate(zip(lengths, count)):
        k, v = (x[table[b, :-(-length // 16)].long()].transpose(1, 2).reshape(-1, nkv, hd)[:length].double().cpu().numpy()
                for x in (kc, vc))
        for i in range(n):
            p = length - n + i
            for h in range(nh):
                with np.errstate(invalid='ignore'):
                    score = k[:p + 1, h // group] @ qn[at + i, h] / np.sqrt(hd)
                    w = np.exp(score - score.max())
                y = got[at + i, h]
                if not np.isfinite(score.max()):
                    kinds.add(str(score.max()))
                    assert np.isnan(y).all(), (b, i, h, score.max())
                    continue
                kinds.add('finite' if np.isfinite(score).all() else 'some')
                want = (w / w.sum()) @ v[:p + 1, h // group]
                assert np.linalg.norm(y - want) <= 1e-5 * np.linalg.norm(want), (b, i, h)
        at += n
    assert len(qn) < 40 or {'inf', 'some'} <= kinds      # (a few rows may all be NaN)


def test_attention_gate_that_is_not_a_number():
    """The gate's clip keeps NaN; infinities are its ends."""
    import torch
    from localai_amd import paged
    for lengths in ([30, 2500], [30, 40]):
        (q, kc, vc, table, dl), kw, y = _attention((8, 2, 64), lengths, 'float16', gate=True, seed=2)
        gate = kw['gate'].clone()
        gate[0, 3, 7] = gate[1, 5, 60] = float('nan')
        gate[0, 0, 0], gate[1, 0, 0] = float('inf'), float('-inf')
        got = paged.attention(q, kc, vc, table, dl, gate=gate).cpu().numpy()
        assert np.isnan(got[0, 3, 7]) and np.isnan(got[1, 5, 60])
        assert np.isnan(got).sum() == 2
        assert got[0, 0, 0] != 0 and abs(got[1, 0, 0]) <= abs(y[1, 0]).max() * 1e3 * np.exp(-80.0)
    (q, kc, vc, table, dl), kw, y = _attention((8, 2, 64), [30, 0], 'float16', gate=True, seed=2)
    got = paged.attention(q, kc, vc, table, dl, gate=torch.full_like(q, float('nan')))
    assert torch.isnan(got[0]).all() and (got[1] == 0).all()           # a row that sees nothing is zeros


def test_attention_over_offsets_past_32_bits():
    """Pages and positions whose byte and value offsets pass 2^32: strides of a large buffer."""
    import torch
    from localai_amd import paged
    hd, nkv, page, pool = 64, 2, 16, 3
    stride = 3 * 2 ** 30 // 2            # values between pages: 3 GiB of fp16
    buf = torch.empty(2 * stride + nkv * page * hd + 64, dtype=torch.float16, device='cuda')
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((pool, nkv, page, hd)).astype(np.float16) for _ in range(2))
    caches = []
    for x, at in ((k, 0), (v, 0)):
        b = buf if x is k else torch.empty_like(buf)
        view = b.as_strided((pool, nkv, page, hd), (stride, page * hd, hd, 1), at)
        view.copy_(torch.from_numpy(x))
        caches.append(view)
    q = rng.standard_normal((2, 4, hd)).astype(np.float32)
    table, lengths = [[2, 0, 1], [1, 2, 0]], [45, 30]
    y = paged.attention(torch.from_numpy(q).cuda(), *caches, _ints(table), _ints(lengths)).cpu().numpy()
    for b in range(2):
        kk, vv = (x[table[b]].transpose(0, 2, 1, 3).reshape(-1, nkv, hd)[:lengths[b]] for x in (k, v))
        want, weight, _ = opaged.attention(q[b:b + 1], kk, vv, 1, opaged.default_scale(hd))
        assert np.linalg.norm(y[b] - want[0]) <= 1e-5 * np.linalg.norm(want)
    x = torch.from_numpy(rng.standard_normal((1, 2, hd)).astype(np.float32)).cuda()
    paged.norm_rope_store(x, x, x, _ints([0]), _ints([2 * 16 + 5]), *caches)
    assert torch.equal(caches[0][2, :, 5], x[0].half()) and torch.equal(caches[1][2, :, 5], x[0].half())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads,lengths,new', [((8, 2, 64), [3000, 5, 0], None), ((8, 2, 128), [2500, 64], [40, 9]),
                                               ((32, 32, 64), [300, 130, 70], [200, 100, 70])])
def test_attention_into_its_queries(heads, lengths, new, dtype):
    from localai_amd import paged
    (q, *rest), kw, y = _attention(heads, lengths, dtype, new=new, seed=14)
    got = paged.attention(q, *rest, out=q, **kw)
    assert got is q
    np.testing.assert_array_equal(q.cpu().numpy(), y)


def test_attention_same_bits_again_and_on_another_stream():
    import torch
    from localai_amd import paged
    args, kw, y = _attention((32, 8, 128), [5000, 3, 700, 1200], 'bfloat16', seed=21)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    again = [paged.attention(*args, **kw) for _ in range(3)] + [paged.attention(*args, stream=s, **kw)]
    torch.cuda.synchronize()
    for x in again:
        np.testing.assert_array_equal(x.cpu().numpy(), y)


def test_attention_calls_at_once_on_two_streams():
    """Calls that overlap in time have workspaces of their own."""
    import torch
    from localai_amd import paged
    calls = [_attention((32, 8, 128), [3000, 900, 40], 'float16', seed=31),
             _attention((32, 8, 128), [70, 2100, 1500], 'float16', seed=32)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(12):
        for (args, kw, _), s, g in zip(calls, streams, got):
            with torch.cuda.stream(s):
                g.append(paged.attention(*args, **kw))
    torch.cuda.synchronize()
    for (_, _, y), g in zip(calls, got):
        for x in g:
            np.testing.assert_array_equal(x.cpu().numpy(), y)


def test_calls_on_another_stream_hold_their_arguments():
    """A Step and inputs dropped while the other stream still waits: their memory is given out only after it."""
    import torch
    from localai_amd import paged
    nh, nkv, hd = 8, 2, 64
    gen = torch.Generator('cuda').manual_seed(3)
    data = [torch.randn((40, h, hd), generator=gen, device='cuda') for h in (nh, nkv, nkv)]
    freq, w = torch.rand(hd // 2, generator=gen, device='cuda', dtype=torch.float64), torch.ones(hd, device='cuda')
    new, keep = _ints([30, 8]), [25, 0]
    side = torch.cuda.Stream()

    def run(stream):
        cache = paged.PagedKVCache(1, nkv, hd, n_pages=8, page_size=16, requests=2, dtype=torch.float16)
        q, k, v = (x.clone() for x in data)
        step = cache.extend(new.clone(), 40)
        if stream is not None:
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                torch.cuda._sleep(20_000_000)        # some 10 ms
        q = cache.store(0, q, k, v, step, freq.clone(), w.clone(), w.clone(), stream=stream)
        y = cache.attention(0, q, step, gate=data[0].clone(), stream=stream)
        status = cache.shrink(_ints(keep), stream=stream)
        more = paged.extend(cache.lengths, _ints([3, 4]), cache.table, cache.free, cache.used, 16, 7, stream=stream)
        return cache, y, status, more

    def results(cache, y, status, more):
        return [x.cpu() for x in (cache.k, cache.v, cache.table, cache.lengths, cache.free, cache.used, y[:38], status, *more)]

    want = results(*run(None))
    torch.cuda.synchronize()
    made = run(side)
    held = [torch.full((n,), 2 ** 30, dtype=torch.int32, device='cuda') for n in
            [2, 3, 8, 40, 83, 127, 128, 64, 40 * nh * hd, 40 * nkv * hd] for _ in range(8)]
    torch.cuda.synchronize()
    for a, b in zip(results(*made), want):
        assert torch.equal(a, b)
    del held


def test_check_waits_for_the_stream_of_the_call():
    import torch
    from localai_amd import paged
    cache = paged.PagedKVCache(1, 1, 64, n_pages=2, page_size=16, requests=1)
    side, new, keep = torch.cuda.Stream(), _ints([40]), _ints([-1])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)        # some 10 ms
    step = cache.extend(new, 40, stream=side)
    with pytest.raises(RuntimeError, match='too few pages|longer than'):
        step.check(stream=side)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    status = cache.shrink(keep, stream=side)
    with pytest.raises(RuntimeError, match='negative'):
        paged.check(status, side)
    with torch.cuda.stream(side):
        cache.extend(_ints([32]), 32).check()


def test_refusals():
    import torch
    from localai_amd import _lib, paged
    (q, kc, vc, table, dl), _, _ = _attention((8, 2, 64), [30, 40], 'float16')
    for bad in (dict(q=q.double()), dict(q=q[:, :, :32]), dict(q=q.transpose(0, 1)), dict(k_cache=kc.float()),
                dict(v_cache=vc[:-1]), dict(table=table.long()), dict(table=table[:1]), dict(lengths=dl.cpu()),
                dict(starts=dl), dict(gate=q[:1]), dict(out=q[:1]), dict(k_cache=kc.double(), v_cache=vc.double()),
                dict(k_cache=kc[..., ::2], v_cache=vc[..., ::2]), dict(table=table.t().contiguous().t())):
        with pytest.raises((TypeError, ValueError)):
            paged.attention(**{**dict(q=q, k_cache=kc, v_cache=vc, table=table, lengths=dl), **bad})
    with pytest.raises(_lib.HipError):          # 5 heads over 2 kv heads
        paged.attention(q[:, :5].contiguous(), kc, vc, table, dl)
    with pytest.raises(_lib.HipError):
        paged.attention(q, kc[:, :, :8], vc[:, :, :8], table, dl)
    with pytest.raises(_lib.HipError, match='head_dim'):
        z = torch.zeros((2, 2, 16, 96), dtype=torch.float16, device='cuda')
        paged.attention(torch.zeros((2, 8, 96), device='cuda'), z, z.clone(), table, dl)
    k = torch.zeros((2, 2, 64), device='cuda')
    ok = dict(q=q, k=k, v=k, positions=dl, slots=dl, k_cache=kc, v_cache=vc)
    for bad in (dict(k=k[:1]), dict(k=k.half()), dict(positions=dl.long()), dict(slots=dl[:1]), dict(rope='other'),
                dict(freq=torch.zeros(4, device='cuda')), dict(q_weight=torch.zeros(32, device='cuda')),
                dict(out=q[:, :4])):
        with pytest.raises((TypeError, ValueError)):
            paged.norm_rope_store(**{**ok, **bad})
    with pytest.raises(_lib.HipError):
        paged.norm_rope_store(**{**ok, 'freq': torch.zeros(33, dtype=torch.float64, device='cuda')})
    with pytest.raises(_lib.HipError, match='aligned'):
        flat = torch.zeros(2 * 8 * 64 + 1, device='cuda')
        paged.norm_rope_store(**{**ok, 'q': flat[1:].view(2, 8, 64)})
    with pytest.raises(_lib.HipError, match='page_size'):
        paged.extend(dl, dl, table, dl, dl[:1], 24, 4)
    with pytest.raises(ValueError):
        paged.extend(dl, dl, table[:1].expand(2, -1), dl, dl[:1], 16, 4)


# ---------------------------------------------------------------- together

class Model:
    """Two layers' q, k, v of each request's tokens and the oracle's run over them."""

    def __init__(self, heads, dtype, rope, norm, seed=0):
        import torch
        self.heads, self.dtype, self.rope = heads, dtype, rope
        self.rng = np.random.default_rng(seed)
        nh, nkv, hd = heads
        self.freq = 10000.0 ** (-np.arange(hd // 4) / (hd // 4))
        self.w = [(1 + .1 * self.rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2)]
        dev = lambda a: torch.from_numpy(a).cuda() if a is not None else None
        self.args = dict(freq=dev(self.freq), q_weight=dev(self.w[0]), k_weight=dev(self.w[1]), rope=rope)
        self.rows = {}            # (layer, request) -> lists of rounded k, v rows

    def qkv(self, tokens):
        nh, nkv, hd = self.heads
        return [self.rng.standard_normal((tokens, h, hd)).astype(np.float32) for h in (nh, nkv, nkv)]

    def want(self, layer, q, k, v, owners, positions):
        import torch
        tt = getattr(torch, self.dtype)
        hd = self.heads[2]
        out = np.zeros(q.shape)
        for t, (b, p) in enumerate(zip(owners, positions)):
            ks, vs = self.rows.setdefault((layer, b), ([], []))
            del ks[p:], vs[p:]
            kk = opaged.norm_rope(k[t], p, self.freq, self.w[1], 1e-6, self.rope)
            ks.append(torch.from_numpy(kk).float().to(tt).double().numpy())
            vs.append(torch.from_numpy(v[t]).to(tt).double().numpy())
            qq = opaged.norm_rope(q[t], p, self.freq, self.w[0], 1e-6, self.rope)
            out[t] = opaged.attention(qq[None], np.array(ks), np.array(vs), 1, opaged.default_scale(hd))[0][0]
        return out


# a k that rounds to the other neighbour in 16 bits moves a score by up to a step of one value: q k eps / sqrt(hd)
# of about 1e-3 (bf16 2^-8 x 3 x 3 / 11), for the rare value within 24 u of a tie; fp32 has no such jumps
RUN_TOL = {'float32': 1e-5, 'float16': 1e-4, 'bfloat16': 1e-3}


@pytest.mark.parametrize('dtype,heads,rope,norm', [('float32', (8, 2, 64), 'pairs', False),
                                                   ('float16', (32, 8, 128), 'halves', True),
                                                   ('bfloat16', (16, 4, 256), 'halves', True)])
def test_serving_run(dtype, heads, rope, norm):
    """Prompts, decode steps with a request joining, drafts taken back, a request ended and its pages used again."""
    import torch
    from localai_amd import paged
    nh, nkv, hd = heads
    m = Model(heads, dtype, rope, norm)
    cache = paged.PagedKVCache(2, nkv, hd, n_pages=14, page_size=16, requests=3, max_pages=8,
                               dtype=getattr(torch, dtype))
    lengths = [0, 0, 0]
    plan = [([37, 5, 0], None), ([1, 1, 0], None), ([1, 1, 20], None), ([4, 1, 4], [39, 7, 21]), ([1, 1, 1], None),
            ([1, 1, 1], [0, 99, 99]), ([60, 1, 1], None), ([1, 16, 1], None)]
    for new, keep in plan:
        owners = [b for b in range(3) for _ in range(new[b])]
        positions = [lengths[b] + i for b in range(3) for i in range(new[b])]
        tokens = sum(new) + 2
        step = cache.extend(_ints(new), tokens)
        for layer in range(2):
            q, k, v = m.qkv(tokens)
            dq, dk, dv = (torch.from_numpy(x).cuda() for x in (q, k, v))
            qr = cache.store(layer, dq, dk, dv, step, **m.args)
            y = cache.attention(layer, qr, step)
            want = m.want(layer, q, k, v, owners, positions)[:sum(new)]
            got = y.cpu().numpy()[:sum(new)]
            assert np.linalg.norm(got - want) <= RUN_TOL[dtype] * np.linalg.norm(want)
        step.check()
        lengths = [a + b for a, b in zip(lengths, new)]
        if keep:
            paged.check(cache.shrink(_ints(keep)))
            lengths = [min(a, b) for a, b in zip(lengths, keep)]
        np.testing.assert_array_equal(cache.lengths.cpu(), lengths)
        assert int(cache.used) == sum(-(-x // 16) for x in lengths)
    step = cache.extend(_ints([100, 100, 100]), 300)
    with pytest.raises(RuntimeError, match='too few pages|longer than'):
        step.check()
    np.testing.assert_array_equal(cache.lengths.cpu(), lengths)
    cache.reset()
    assert int(cache.used) == 0 and not cache.lengths.any() and (cache.table == -1).all()


def test_decode_steps_from_one_graph():
    """A captured decode step (extend, store, attention) replayed ten times, against the same steps run eagerly."""
    import torch
    from localai_amd import paged
    nh, nkv, hd = 32, 8, 128
    rng = np.random.default_rng(4)

    def fresh():
        c = paged.PagedKVCache(1, nkv, hd, n_pages=40, page_size=16, requests=4, dtype=torch.bfloat16)
        step = c.extend(_ints([30, 0, 7, 100]), 137)
        k = torch.from_numpy(np.random.default_rng(1).standard_normal((137, nkv, hd)).astype(np.float32)).cuda()
        paged.norm_rope_store(k, k, k, step.positions, step.slots, c.k[0], c.v[0])
        return c

    new = _ints([1, 0, 1, 1])
    freq = torch.from_numpy(10000.0 ** (-np.arange(64) / 64)).cuda()
    w = torch.ones(hd, device='cuda')
    q, k, v = (torch.empty((4, h, hd), device='cuda') for h in (nh, nkv, nkv))

    def one(c):
        step = c.extend(new, 4)
        return c.attention(0, c.store(0, q, k, v, step, freq, w, w), step), step.status

    inputs = [[rng.standard_normal(tuple(x.shape)).astype(np.float32) for x in (q, k, v)] for _ in range(10)]

    def fill(xs):
        for t, x in zip((q, k, v), xs):
            t.copy_(torch.from_numpy(x))

    eager, wants = fresh(), []
    for xs in inputs:
        fill(xs)
        wants.append(one(eager)[0][:3].cpu().numpy())
    cache = fresh()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    fill(inputs[0])
    torch.cuda.synchronize()
    kept = [t.clone() for t in (cache.lengths, cache.used, cache.table)]
    with torch.cuda.graph(g, stream=s):
        y, status = one(cache)
    for t, x in zip((cache.lengths, cache.used, cache.table), kept):
        t.copy_(x)
    for xs, want in zip(inputs, wants):
        fill(xs)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(y[:3].cpu().numpy(), want)
        paged.check(status)
        one(eager)                               # other work between the replays
        torch.cuda.synchronize()
    np.testing.assert_array_equal(cache.lengths.cpu(), [40, 0, 17, 110])
