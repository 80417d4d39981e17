"""Token operators (eo_vae_amd.token_ops) against their definitions in 64 bits.

Tolerances are bounds worked out from the operands, value by value: `h` is half a step of the output type, `u` half a step
of the type in which probabilities and score gradients enter a product (0 for fp32), `f` = 2^-24, and a sum of n fp32 terms is
off by at most n f times the sum of their magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def reference_bucket(rel, buckets, max_distance, two_sided):
    side = buckets // 2 if two_sided else buckets
    e, m = side // 2, side - side // 2
    n = abs(rel) if two_sided else max(-rel, 0)
    if n < e:
        b = n
    else:
        b = e + max(t for t in range(m) if n ** m >= e ** (m - t) * max_distance ** t)
    return b + (side if two_sided and rel > 0 else 0)


def reference(q, k, v, do, maps, scale, bias=None, lam=None, max_distance=128, two_sided=True, causal=False, kv_len=None, start=None):
    """(values, bounds): dicts of out, dq, dk, dv, dbias, dlam in fp64 and how far the operator may be from them."""
    t = q.dtype
    h, u = HALF[t], 0.0 if t == torch.float32 else HALF[t]
    q, k, v, do = (x.detach().cpu().double() for x in (q, k, v, do))
    b, sq, nh, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    w = d // maps
    share = nh // hk
    bt = None if bias is None else bias.detach().cpu().double()
    lm = torch.ones(nh, dtype=torch.float64) if lam is None else lam.detach().cpu().double()
    val = {'out': torch.zeros_like(q), 'dq': torch.zeros_like(q), 'dk': torch.zeros_like(k), 'dv': torch.zeros_like(v)}
    if bt is not None:
        val['dbias'] = torch.zeros_like(bt)
    if lam is not None:
        val['dlam'] = torch.zeros_like(lm)
    err = {n: torch.zeros_like(x) for n, x in val.items()}
    for i in range(b):
        n = sk if kv_len is None else int(kv_len[i])
        s0 = sk - sq if start is None else int(start if isinstance(start, int) else start[i])
        if n == 0:
            continue
        rel = torch.arange(n)[None] - (s0 + torch.arange(sq))[:, None]
        seen = rel <= 0 if causal else torch.ones_like(rel, dtype=torch.bool)
        if bt is not None:
            lo, hi = int(rel.min()), int(rel.max())
            table = torch.tensor([reference_bucket(r, bt.shape[0], max_distance, two_sided) for r in range(lo, hi + 1)])
            bucket = table[rel - lo]
        for j in range(nh):
            kj, vj, qj, gj = k[i, :n, j // share], v[i, :n, j // share], q[i, :, j], do[i, :, j]
            add = bt[:, j][bucket] if bt is not None else torch.zeros(sq, n, dtype=torch.float64)
            P, rP = [], []
            for m in range(maps):
                sl = slice(m * w, (m + 1) * w)
                s = scale * qj[:, sl] @ kj[:, sl].T + add
                e_s = F * (w + 8) * (abs(scale) * qj[:, sl].abs() @ kj[:, sl].abs().T + add.abs()) + 4 * F * s.abs()
                s = s.masked_fill(~seen, -math.inf)
                p = torch.softmax(s, 1).nan_to_num(0.0)
                e_s = e_s.masked_fill(~seen, 0.0)
                P.append(p)
                rP.append(e_s + e_s.amax(1, keepdim=True) + F * (n + 16))
            wts = [1.0, -float(lm[j])][:maps]
            A = sum(c * p for c, p in zip(wts, P))
            o = A @ vj
            aA = sum(abs(c) * p * (r + u + n * F) for c, p, r in zip(wts, P, rP))          # error of the weights in a product
            eo = aA @ vj.abs() + h * o.abs()
            val['out'][i, :, j] = o
            err['out'][i, :, j] = eo
            # backward
            da = gj @ vj.T
            ada = gj.abs() @ vj.abs().T
            aA2 = sum(abs(c) * p * (r + (sq * share + 2) * F) for c, p, r in zip(wts, P, rP)) + u * A.abs()
            val['dv'][i, :n, j // share] += A.T @ gj
            err['dv'][i, :n, j // share] += aA2.T @ gj.abs() + sq * F * (A.abs().T @ gj.abs())
            ds_all, e_all = 0, 0
            for m in range(maps):
                sl = slice(m * w, (m + 1) * w)
                c = wts[m]
                om = P[m] @ vj
                dm = (c * gj * om).sum(1, keepdim=True)
                # delta is formed from stored outputs: each off by its own rounding and by the weights' error
                eom = (P[m] * (rP[m] + u + n * F)) @ vj.abs() + h * om.abs()
                if maps == 2 and m == 0:                       # O_0 = O + lambda O_1 from two stored values
                    eom = eom + eo + abs(float(lm[j])) * ((P[1] * (rP[1] + u + n * F)) @ vj.abs() + h * (P[1] @ vj).abs())
                ed = abs(c) * (gj.abs() * eom).sum(1, keepdim=True) + (d + 4) * F * abs(c) * (gj.abs() * om.abs()).sum(1, keepdim=True)
                ds = P[m] * (c * da - dm)
                eds = ds.abs() * (rP[m] + u + 4 * F) + P[m] * (abs(c) * (d + 4) * F * ada + ed)
                val['dq'][i, :, j, sl] = scale * ds @ kj[:, sl]
                err['dq'][i, :, j, sl] = abs(scale) * (eds + n * F * ds.abs()) @ kj[:, sl].abs()
                val['dk'][i, :n, j // share, sl] += scale * ds.T @ qj[:, sl]
                err['dk'][i, :n, j // share, sl] += abs(scale) * (eds + (sq * share + 2) * F * ds.abs()).T @ qj[:, sl].abs()
                ds_all, e_all = ds_all + ds, e_all + eds - u * ds.abs() + ((sq + n) * F) * ds.abs()
            if bt is not None:
                val['dbias'][:, j].index_add_(0, bucket.reshape(-1), ds_all.reshape(-1))
                err['dbias'][:, j].index_add_(0, bucket.reshape(-1), e_all.reshape(-1))
            if lam is not None:
                o1 = P[1] @ vj
                val['dlam'][j] -= (gj * o1).sum()
                e1 = (P[1] * (rP[1] + u + n * F)) @ vj.abs() + h * o1.abs()
                err['dlam'][j] += (gj.abs() * e1).sum() + (sq * d) * F * (gj * o1).abs().sum()
    for n in ('dq', 'dk', 'dv'):
        err[n] += h * val[n].abs() + (h * 1e-30)
    for n, x in (('dbias', bias), ('dlam', lam)):
        if n in val:
            err[n] += HALF[x.dtype] * val[n].abs()
    return val, err


def inside(got, want, bound, name):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), f'{name}: not finite'
    over = (got - want).abs() - bound * (1 + 1e-6) - 1e-37
    assert (over <= 0).all(), f'{name}: {int((over > 0).sum())} values outside, worst off by {float((got - want).abs().max()):.3g}, ' \
                              f'largest excess {float(over.max()):.3g}'


def make(b, sq, sk, h, hk, d, dtype, maps, buckets=0, seed=0, param=None):
    g = torch.Generator().manual_seed(seed + 1000 * sq + sk)
    r = lambda *s: torch.randn(*s, generator=g)                                            # noqa: E731
    x = {'q': r(b, sq, h, d), 'k': r(b, sk, hk, d), 'v': r(b, sk, hk, d), 'do': r(b, sq, h, d)}
    x = {n: t.to(dtype).cuda() for n, t in x.items()}
    x['bias'] = r(buckets, h).to(param or dtype).cuda() if buckets else None
    x['lam'] = (0.5 + 0.2 * r(h)).to(param or dtype).cuda() if maps == 2 else None
    return x


def call(x, maps, **kw):
    from eo_vae_amd import token_ops as T
    if maps == 2:
        return T.diff_attention(x['q'], x['k'], x['v'], x['lam'], x['bias'], **kw)
    return T.rel_pos_attention(x['q'], x['k'], x['v'], x['bias'], **kw)


def run_and_check(x, maps, max_distance=128, two_sided=True, causal=False, kv_len=None, start=None, scale=None):
    leaves = {n: x[n].requires_grad_(True) for n in ('q', 'k', 'v', 'bias', 'lam') if x[n] is not None}
    dev = lambda t: t if t is None or isinstance(t, int) else torch.tensor(t, dtype=torch.int32, device='cuda')   # noqa: E731
    out = call(x, maps, max_distance=max_distance, bidirectional=two_sided, causal=causal, kv_len=dev(kv_len), query_start=dev(start),
               scale=scale)
    grads = torch.autograd.grad(out, list(leaves.values()), x['do'])
    with torch.no_grad():        # the call that keeps nothing for a backward gives the same values
        assert torch.equal(out, call(x, maps, max_distance=max_distance, bidirectional=two_sided, causal=causal, kv_len=dev(kv_len),
                                     query_start=dev(start), scale=scale))
    w = x['q'].shape[-1] // maps
    val, err = reference(x['q'], x['k'], x['v'], x['do'], maps, w ** -0.5 if scale is None else scale, x['bias'], x['lam'], max_distance,
                         two_sided, causal, kv_len, start)
    inside(out, val['out'], err['out'], 'out')
    for n, g in zip(leaves, grads):
        assert g.dtype == x[n].dtype and g.shape == x[n].shape
        inside(g, val['d' + n], err['d' + n], 'd' + n)
    return out, grads


BF, FP = torch.bfloat16, torch.float32


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps,d', [(1, 32), (1, 64), (1, 128), (2, 64), (2, 128)])
@pytest.mark.parametrize('shape', [
    dict(b=1, sq=1, sk=1, h=1, hk=1),
    dict(b=2, sq=33, sk=65, h=2, hk=1, buckets=8, max_distance=20),
    dict(b=1, sq=141, sk=141, h=4, hk=4, buckets=32),
    dict(b=2, sq=70, sk=70, h=4, hk=2, causal=True, buckets=32, two_sided=False, max_distance=40),
    dict(b=1, sq=130, sk=300, h=2, hk=2, causal=True, buckets=16, two_sided=True, max_distance=64),
    dict(b=3, sq=40, sk=90, h=2, hk=2, kv_len=[90, 17, 0], buckets=6, max_distance=9, start=[0, 5, -3]),
    dict(b=2, sq=200, sk=64, h=2, hk=1, causal=True),                                  # the first 136 rows see nothing
    dict(b=2, sq=96, sk=96, h=2, hk=2, causal=True, kv_len=[96, 31], start=0, buckets=4, max_distance=3),
    dict(b=1, sq=64, sk=257, h=3, hk=1, scale=0.31),
    dict(b=2, sq=70, sk=70, h=2, hk=2, causal=True, scale=-0.2, kv_len=[70, 44], start=0),
    dict(b=1, sq=70, sk=100, h=1, hk=1, causal=True, scale=0.0, buckets=8, max_distance=10),
])
def test_attention_and_gradients(maps, d, dtype, shape):
    s = dict(shape)
    x = make(s.pop('b'), s.pop('sq'), s.pop('sk'), s.pop('h'), s.pop('hk'), d, dtype, maps, s.pop('buckets', 0))
    run_and_check(x, maps, **s)


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps,d', [(1, 32), (1, 64), (1, 128), (2, 64), (2, 128)])
@pytest.mark.parametrize('shape', [
    dict(b=64, sq=37, sk=75, h=4, hk=4, buckets=8, max_distance=20),
    dict(b=32, sq=150, sk=150, h=4, hk=4, causal=True, two_sided=False, buckets=16, max_distance=30, kv_len=[150, 0, 1, 64] * 8, start=0),
    dict(b=32, sq=131, sk=200, h=8, hk=2)])
def test_calls_that_fill_the_chip(maps, d, dtype, shape):
    """At least 256 blocks of 128 rows: the forms that smaller calls do not take."""
    s = dict(shape)
    x = make(s.pop('b'), s.pop('sq'), s.pop('sk'), s.pop('h'), s.pop('hk'), d, dtype, maps, s.pop('buckets', 0), seed=17)
    run_and_check(x, maps, **s)


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps,d', [(1, 32), (1, 64), (1, 128), (2, 64), (2, 128)])
@pytest.mark.parametrize('b,sq,sk,h,hk,lens', [
    (3, 1, 700, 8, 2, [700, 1, 333]), (2, 2, 129, 4, 4, [2, 129]), (1, 1, 4000, 1, 1, [3999]), (2, 5, 260, 6, 1, [5, 257]),
    (2, 1, 50, 32, 1, [50, 0]), (70, 1, 300, 2, 2, [(37 * i) % 301 for i in range(70)]), (3, 4, 3000, 8, 1, [3000, 129, 2047])])
def test_single_tokens_on_a_cache(maps, d, dtype, b, sq, sk, h, hk, lens):
    x = make(b, sq, sk, h, hk, d, dtype, maps, 32, seed=5)
    for i, n in enumerate(lens):            # nothing behind a sequence's length is read
        x['k'][i, n:] = float('nan')
        x['v'][i, n:] = float('inf')
    run_and_check_padded(x, maps, lens, [n - sq for n in lens])


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps,d', [(1, 64), (2, 128)])
@pytest.mark.parametrize('b,h,sq,sk,start', [(1, 2, 40, 300, 20), (70, 4, 40, 100, 20), (1, 2, 2, 100, 50), (1, 1, 300, 400, -100)])
def test_keys_ahead_of_every_query_are_not_read(b, h, sq, sk, start, maps, d, dtype):
    x = make(b, sq, sk, h, h, d, dtype, maps, 8, seed=18)
    last = start + sq
    y = dict(x)
    for n, bad in (('k', float('nan')), ('v', float('inf'))):
        y[n] = x[n].clone()
        y[n][:, last:] = bad
    kw = dict(max_distance=20, bidirectional=False, causal=True, query_start=start)
    got, want = [], []
    for z, out in ((x, want), (y, got)):
        leaves = [z[n].requires_grad_(True) for n in ('q', 'k', 'v', 'bias', 'lam') if z[n] is not None]
        o = call(z, maps, **kw)
        out += [o.detach(), *torch.autograd.grad(o, leaves, x['do'])]
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    assert torch.equal(got[2][:, last:], torch.zeros_like(got[2][:, last:])) and torch.equal(got[3][:, last:], torch.zeros_like(got[3][:, last:]))


def run_and_check_padded(x, maps, lens, start):
    from copy import copy
    y = copy(x)
    y['k'], y['v'] = x['k'].nan_to_num(0.0, 0.0, 0.0), x['v'].nan_to_num(0.0, 0.0, 0.0)
    t = lambda a: torch.tensor(a, dtype=torch.int32, device='cuda')                       # noqa: E731
    leaves = [x[n].requires_grad_(True) for n in ('q', 'k', 'v')]
    out = call(x, maps, causal=True, bidirectional=False, kv_len=t(lens), query_start=t(start))
    grads = torch.autograd.grad(out, leaves, x['do'])
    d = x['q'].shape[-1] // maps
    val, err = reference(y['q'], y['k'], y['v'], y['do'], maps, d ** -0.5, y['bias'], y['lam'], 128, False, True, lens, start)
    inside(out, val['out'], err['out'], 'out')
    for n, g in zip(('dq', 'dk', 'dv'), grads):
        inside(g, val[n], err[n], n)


@pytest.mark.parametrize('maps,d', [(1, 64), (1, 128), (2, 128)])
@pytest.mark.parametrize('causal', [False, True])
def test_key_gradients_joined_from_parts(maps, d, causal):
    """Few key heads: the queries of one key block are walked by several thread blocks."""
    x = make(1, 333, 210, 6, 1, d, BF, maps, 16, seed=14)
    run_and_check(x, maps, 40, not causal, causal, start=-100 if causal else None)


@pytest.mark.parametrize('maps', [1, 2])
def test_parameters_in_fp32_beside_bf16_tokens(maps):
    run_and_check(make(2, 50, 50, 2, 2, 64, BF, maps, 32, param=FP), maps)


@pytest.mark.parametrize('buckets,max_distance,two_sided', [(2, 2, False), (4, 2, True), (128, 1024, True), (127, 1000, False), (64, 34, True)])
def test_bucket_tables(buckets, max_distance, two_sided):
    from eo_vae_amd import token_ops as T
    side = buckets // 2 if two_sided else buckets
    e, borders = side // 2, T.bucket_borders(side, max_distance)
    assert len(borders) == side - e - 1 and list(borders) == sorted(borders)
    for n in range(0, max_distance + 3):
        want = reference_bucket(-n, buckets, max_distance, two_sided)
        assert want == (n if n < e else e + sum(n >= x for x in borders))
    x = make(1, 90, 150, 2, 1, 32, FP, 1, buckets, seed=3)
    run_and_check(x, 1, max_distance, two_sided)


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps', [1, 2])
def test_the_longest_reach_at_the_widest_heads(maps, dtype):
    x = make(1, 140, 900, 2, 2, 128, dtype, maps, 128, seed=13)
    run_and_check(x, maps, 1024, True, start=300)
    x = make(1, 1, 900, 4, 1, 128, dtype, maps, 128, seed=13)
    run_and_check(x, maps, 1024, False, True, kv_len=[870], start=869)


def test_lengths_outside_the_cache_and_starts_far_away():
    from eo_vae_amd import token_ops as T
    x = make(4, 3, 70, 2, 1, 64, BF, 1, 32, seed=15)
    t = lambda a: torch.tensor(a, dtype=torch.int32, device='cuda')                       # noqa: E731
    clamped = T.rel_pos_attention(x['q'], x['k'], x['v'], x['bias'], kv_len=t([70, 70, 0, 0]), query_start=t([67] * 4))
    assert torch.equal(T.rel_pos_attention(x['q'], x['k'], x['v'], x['bias'], kv_len=t([71, 2 ** 31 - 1, -1, -2 ** 31]), query_start=t([67] * 4)), clamped)
    assert torch.equal(clamped[2:], torch.zeros_like(clamped[2:]))
    # positions beyond any distance: the last buckets' constant, which a softmax does not see
    plain = T.rel_pos_attention(x['q'], x['k'], x['v'])
    for far in (2 ** 31 - 1, -2 ** 31, 2 ** 30, -2 ** 30):
        got = T.rel_pos_attention(x['q'], x['k'], x['v'], x['bias'], query_start=t([far] * 4))
        assert (got.float() - plain.float()).abs().max() <= 2.0 ** -7 * plain.float().abs().max()


@pytest.mark.parametrize('low', [float('-inf'), -3.0e38])
@pytest.mark.parametrize('sq,sk', [(1, 400), (150, 400), (300, 2100)])
def test_buckets_that_shut_keys_out(low, sq, sk):
    """A bias of -infinity, or of nearly the type's lowest value, for every key at and behind distance 64 leaves the others alone."""
    from eo_vae_amd import token_ops as T
    x = make(1, sq, sk, 2, 2, 64, FP, 1, 2, seed=16)
    for n in ('q', 'k', 'v'):
        x[n].requires_grad_(True)
    shut = torch.tensor([[0.0, 0.0], [low, low]], device='cuda')
    wide = torch.zeros(64, 2, device='cuda')
    wide[32:] = low                                    # 64 buckets, one-sided: 32 distances of their own, then up to 33
    out = T.rel_pos_attention(x['q'], x['k'], x['v'], wide, max_distance=33, bidirectional=False, causal=True)
    rel = torch.arange(sk)[None] - (sk - sq + torch.arange(sq))[:, None]
    seen = ((rel <= 0) & (rel > -32)).cuda()
    q, k, v = (x[n].detach().double() for n in ('q', 'k', 'v'))
    s = torch.einsum('bqhd,bkhd->bhqk', q, k) / 8
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    want = torch.einsum('bhqk,bkhd->bqhd', p, v)
    assert (out.double() - want).abs().max() < 1e-4 * want.abs().max()
    dk, dv = torch.autograd.grad(out, [x['k'], x['v']], x['do'])
    assert torch.isfinite(dk).all() and torch.isfinite(dv).all()
    hidden = ~seen.any(0)
    assert dk[:, hidden].abs().max() <= 1e-30 if hidden.any() else True
    # nothing but shut keys: -infinity leaves no key, the lowest value leaves the scores alone
    only = T.rel_pos_attention(x['q'], x['k'], x['v'], shut, max_distance=2, bidirectional=False, causal=True, query_start=sk + 5)
    assert torch.equal(only, torch.zeros_like(only)) if low == -math.inf else torch.isfinite(only).all() and only.abs().max() > 0


def test_a_far_long_range_reaches_the_last_buckets():
    x = make(1, 300, 1500, 1, 1, 32, FP, 1, 32, seed=9)
    run_and_check(x, 1, 128, True, start=600)


@pytest.mark.parametrize('dtype', [FP, BF])
def test_views_are_read_as_they_lie(dtype):
    from eo_vae_amd import token_ops as T
    g = torch.Generator().manual_seed(2)
    b, s, h, d = 2, 75, 4, 64
    packed = torch.randn(b, s, 3, h, d, generator=g).to(dtype).cuda()
    q, k, v = packed.unbind(2)
    want = T.rel_pos_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(T.rel_pos_attention(q, k, v), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(T.rel_pos_attention(*heads_first), want)
    flat = torch.empty(b * s * h * d + 8, dtype=dtype, device='cuda')
    odd = flat[1:1 + b * s * h * d].view(b, s, h, d).copy_(q)                # not on 16 bytes
    assert torch.equal(T.rel_pos_attention(odd, k, v), want)
    wide = torch.randn(b, s, h, d + 3, generator=g).to(dtype).cuda()
    wide[..., :d] = q
    assert torch.equal(T.rel_pos_attention(wide[..., :d], k, v), want)
    # one key sequence broadcast over the batch: its gradient is the sum
    k1 = k[:1].contiguous().requires_grad_(True)
    out = T.rel_pos_attention(q, k1.expand(b, s, h, d), v)
    do = torch.randn(b, s, h, d, generator=g).to(dtype).cuda()
    (got,) = torch.autograd.grad(out, [k1], do)
    kk = k[:1].repeat(b, 1, 1, 1).requires_grad_(True)
    (each,) = torch.autograd.grad(T.rel_pos_attention(q, kk, v), [kk], do)
    assert torch.equal(got, each.sum(0, keepdim=True))


@pytest.mark.parametrize('sq', [1, 40])
def test_offsets_beyond_32_bits(sq):
    """Key rows 2^27 elements apart: the last lies 5 * 10^9 elements behind the first."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip('needs 12 GiB')
    gap, n, d = 1 << 27, 40, 64
    x = make(1, sq, n, 2, 1, d, BF, 1, seed=4)
    far = torch.empty(gap * (n - 1) + d, dtype=BF, device='cuda')
    k = far.as_strided((1, n, 1, d), (0, gap, d, 1))
    k.copy_(x['k'])
    want = call(x, 1)
    y = dict(x)
    y['k'] = k
    assert torch.equal(call(y, 1), want)


@pytest.mark.parametrize('maps,causal', [(1, False), (2, True)])
def test_gradients_against_differences(maps, causal):
    x = make(1, 37, 45, 2, 1, 64, FP, maps, 16, seed=11)
    names = [n for n in ('q', 'k', 'v', 'bias', 'lam') if x[n] is not None]
    leaves = [x[n].requires_grad_(True) for n in names]
    kw = dict(max_distance=30, causal=causal, bidirectional=not causal)
    grads = torch.autograd.grad(call(x, maps, **kw), leaves, x['do'])
    g = torch.Generator().manual_seed(1)
    for n, grad in zip(names, grads):
        step = torch.randn(x[n].shape, generator=g).cuda()
        eps = 2.0 ** -7
        f = []
        for sign in (1, -1):
            y = dict(x)
            y[n] = (x[n] + sign * eps * step).detach()
            f.append((call({m: (t.detach() if t is not None else None) for m, t in y.items()}, maps, **kw).double() * x['do'].double()).sum())
        slope, want = float(f[0] - f[1]) / (2 * eps), float((grad.double() * step.double()).sum())
        # central difference: third derivatives of a softmax are of the order of the slope's scale times eps^2 (6e-5); fp32 values
        # of ~37 * 64 * 2 terms off by 2^-22 each, over 2 eps
        size = float((grad.double() * step.double()).abs().sum())
        assert abs(slope - want) < 2e-3 * size + 37 * 128 * 2.0 ** -22 / (2 * eps) * 0.1, (n, slope, want)


@pytest.mark.parametrize('maps', [1, 2])
def test_same_bits_every_time_and_on_another_stream(maps):
    x = make(2, 150, 260, 4, 2, 64, BF, maps, 32, seed=6)
    leaves = [x[n].requires_grad_(True) for n in ('q', 'k', 'v', 'bias', 'lam') if x[n] is not None]

    def once():
        out = call(x, maps)
        return (out.detach(),) + torch.autograd.grad(out, leaves, x['do'])
    first = once()
    for a, b in zip(first, once()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_two_captured_graphs_replay_in_turn():
    from eo_vae_amd import token_ops as T
    cases = [make(2, 1, 900, 8, 2, 64, BF, 1, 32, seed=7), make(2, 1, 900, 8, 2, 64, BF, 2, 32, seed=8)]
    lens = torch.tensor([900, 411], dtype=torch.int32, device='cuda')
    kw = dict(causal=True, bidirectional=False, kv_len=lens, query_start=lens - 1)
    for x in cases:
        call(x, 1 if x['lam'] is None else 2, **kw)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = call(x, 1 if x['lam'] is None else 2, **kw)
            y, z = T.gated_norm_residual(o, x['q'], torch.ones(64, dtype=BF, device='cuda'), pre_weight=torch.ones(64, dtype=BF, device='cuda'))
        graphs.append(g)
        outs.append((o, y, z))
    for turn in range(3):
        for x in cases:
            x['q'].copy_(torch.randn(x['q'].shape, generator=torch.Generator().manual_seed(turn)).to(BF))
        graphs[0].replay()
        graphs[1].replay()
        for x, (o, y, z) in zip(cases, outs):
            want = call(x, 1 if x['lam'] is None else 2, **kw)
            assert torch.equal(o, want)
            one = torch.ones(64, dtype=BF, device='cuda')
            wy, wz = T.gated_norm_residual(want, x['q'], one, pre_weight=one)
            assert torch.equal(y, wy) and torch.equal(z, wz)
        torch.cuda.synchronize()


def test_a_captured_training_step():
    from eo_vae_amd import token_ops as T
    x = make(2, 100, 100, 4, 2, 64, BF, 2, 32, seed=12)
    w = torch.ones(64, dtype=BF, device='cuda')

    def step(t):
        leaves = [t[n] for n in ('q', 'k', 'v', 'bias', 'lam')]
        y, z = T.gated_norm_residual(call(t, 2), t['q'], w, pre_weight=w)
        return torch.autograd.grad([y, z], leaves, [t['do'], t['do']])

    def fresh(t):        # leaves of their own: an eager graph and a captured one never share them
        return {n: a.detach().clone().requires_grad_(n != 'do') for n, a in t.items()}
    step(fresh(x))
    torch.cuda.synchronize()
    held = fresh(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(held)
    for turn in range(3):
        x['q'] = torch.randn(x['q'].shape, generator=torch.Generator().manual_seed(turn + 40)).to(BF).cuda()
        with torch.no_grad():
            held['q'].copy_(x['q'])
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(fresh(x))):
            assert torch.equal(a, b)


# ---- the residual step ----

def norm_reference(x, layer, alpha, eps, gate_rows):
    """(values, bounds) in fp64; rows [rows, c].  A row's statistics are off by (c + 8) f relative (sums of c positive terms), a
    mean by c f times the mean magnitude; everything else is a handful of fp32 operations."""
    t, pt = x['h'].dtype, x['w1'].dtype
    h_, ph = HALF[t], HALF[pt]
    d = {n: (None if a is None else a.detach().cpu().double()) for n, a in x.items()}
    c = d['h'].shape[-1]
    flat = lambda a: None if a is None else a.reshape(-1, c)                               # noqa: E731
    h, xs, dy, dz = flat(d['h']), flat(d['x']), flat(d['dy']), flat(d['dz'])
    rows = h.shape[0]
    per = rows // gate_rows
    g = d['gate'].reshape(gate_rows, c).repeat_interleave(per, 0) if d['gate'] is not None else torch.ones(rows, c, dtype=torch.float64)
    zero = torch.zeros(c, dtype=torch.float64)
    w1, w2 = d['w1'], d['w2']
    b1 = d['b1'] if d['b1'] is not None else zero
    b2 = d['b2'] if d['b2'] is not None else zero
    k = (c + 16) * F

    def unit(a, ea):
        m = a.mean(1, keepdim=True) if layer else 0 * a[:, :1]
        em = (c * F * a.abs() + ea).mean(1, keepdim=True) if layer else 0 * a[:, :1]
        v = (a - m).square().mean(1, keepdim=True)
        s = (v + eps).sqrt()
        ed = ea + em + F * (a.abs() + m.abs())
        es = ((a - m).abs() * ed).mean(1, keepdim=True) / s + k * s
        u = (a - m) / s
        return u, s, ed / s + u.abs() * (es / s + 4 * F), es / s

    u, s1, eu, rs1 = unit(h, 0 * h)
    n = u * w1 + b1
    en = eu * w1.abs() + 3 * F * ((u * w1).abs() + b1.abs())
    y = alpha * xs + g * n
    ey = g.abs() * en + 4 * F * ((alpha * xs).abs() + (g * n).abs())
    val, err = {'y': y}, {'y': ey + h_ * y.abs()}
    D, eD = dy, 0 * dy
    if w2 is not None:
        q, s2, eq, rs2 = unit(y, ey)
        z = q * w2 + b2
        val['z'], err['z'] = z, eq * w2.abs() + 3 * F * ((q * w2).abs() + b2.abs()) + h_ * z.abs()

        def back(a, ea, un, eun, s, rs):
            mean = (lambda r: r.mean(1, keepdim=True))
            m = mean(a) if layer else 0
            em = mean(ea + c * F * a.abs()) if layer else 0
            t_ = mean(a * un)
            et = mean(ea * un.abs() + a.abs() * eun + (c + 4) * F * (a * un).abs())
            r = (a - m - un * t_) / s
            size = a.abs() + (abs(m) if layer else 0) + (un * t_).abs()
            e = (ea + em + un.abs() * et + eun * t_.abs() + 4 * F * size) / s + r.abs() * (rs + 4 * F)
            return r, e
        a = dz * w2
        r, e = back(a, 2 * F * a.abs(), q, eq, s2, rs2)
        D, eD = dy + r, e + 2 * F * (dy.abs() + r.abs())
        val['dw2'] = (dz * q).sum(0)
        err['dw2'] = (dz.abs() * eq).sum(0) + (rows + 4) * F * (dz * q).abs().sum(0)
        val['db2'], err['db2'] = dz.sum(0), (rows + 4) * F * dz.abs().sum(0)
    else:
        def back(a, ea, un, eun, s, rs):
            m = a.mean(1, keepdim=True) if layer else 0
            em = (ea + c * F * a.abs()).mean(1, keepdim=True) if layer else 0
            t_ = (a * un).mean(1, keepdim=True)
            et = (ea * un.abs() + a.abs() * eun + (c + 4) * F * (a * un).abs()).mean(1, keepdim=True)
            r = (a - m - un * t_) / s
            size = a.abs() + (abs(m) if layer else 0) + (un * t_).abs()
            return r, (ea + em + un.abs() * et + eun * t_.abs() + 4 * F * size) / s + r.abs() * (rs + 4 * F)
    val['dx'], err['dx'] = alpha * D, abs(alpha) * eD + (h_ + 2 * F) * (alpha * D).abs()
    cc = D * g * w1
    r, e = back(cc, eD * (g * w1).abs() + 3 * F * cc.abs(), u, eu, s1, rs1)
    val['dh'], err['dh'] = r, e + h_ * r.abs()
    many = (rows + 8) * F
    val['dw1'] = (D * g * u).sum(0)
    err['dw1'] = (g.abs() * (eD * u.abs() + D.abs() * eu)).sum(0) + many * (D * g * u).abs().sum(0)
    val['db1'] = (D * g).sum(0)
    err['db1'] = (eD * g.abs()).sum(0) + many * (D * g).abs().sum(0)
    group = lambda a: a.reshape(gate_rows, per, c).sum(1)                                  # noqa: E731
    val['dgate'] = group(D * n)
    # w1 * sum(D u) + b1 * sum(D): the two sums are rounded apart
    err['dgate'] = group(eD * (u * w1).abs() + (D * w1).abs() * eu + eD * b1.abs()) + many * group((D * u * w1).abs() + (D * b1).abs())
    for name in ('dw1', 'db1', 'dw2', 'db2', 'dgate'):
        if name in val:
            err[name] = err[name] + ph * val[name].abs()
    return val, err


def make_norm(lead, c, dtype, layer, gate=None, second=True, param=None, seed=0):
    g = torch.Generator().manual_seed(seed + c)
    r = lambda *s: torch.randn(*s, generator=g)                                            # noqa: E731
    p = param or dtype
    x = {n: r(*lead, c).to(dtype).cuda() for n in ('h', 'x', 'dy', 'dz')}
    x['x'] = (2 * x['x'])
    x['w1'] = (1 + 0.2 * r(c)).to(p).cuda()
    x['w2'] = (1 + 0.2 * r(c)).to(p).cuda() if second else None
    x['b1'] = (0.3 * r(c)).to(p).cuda() if layer else None
    x['b2'] = (0.3 * r(c)).to(p).cuda() if layer and second else None
    x['gate'] = (0.5 + r(*gate, c)).to(p).cuda() if gate is not None else None
    if not second:
        x['dz'] = None
    return x


def run_norm(x, layer, alpha=1.0, eps=1e-6):
    from eo_vae_amd import token_ops as T
    names = [n for n in ('h', 'x', 'w1', 'b1', 'w2', 'b2', 'gate') if x[n] is not None]
    leaves = [x[n].requires_grad_(True) for n in names]
    y, z = T.gated_norm_residual(x['h'], x['x'], x['w1'], x['gate'], x['w2'], post_bias=x['b1'], pre_bias=x['b2'],
                                 norm='layer' if layer else 'rms', residual_scale=alpha, eps=eps)
    outs = [y] if z is None else [y, z]
    grads = torch.autograd.grad(outs, leaves, [x['dy']] if z is None else [x['dy'], x['dz']])
    return y, z, dict(zip(names, grads))


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('layer', [False, True])
@pytest.mark.parametrize('lead,c,gate', [
    ((1,), 1, None), ((3,), 8, ()), ((2, 7), 33, (2, 1)), ((5, 3), 257, (5, 3)), ((141,), 256, ()), ((2, 70), 512, (2, 1)), ((9,), 520, ()),
    ((4, 33), 1024, (4, 1)), ((3, 11), 1031, None), ((2, 20), 2048, (2, 20)), ((17,), 2050, ()), ((6, 5), 4096, (6, 1)), ((7,), 4100, ()),
    ((2, 3, 4), 8192, (2, 1, 1)), ((3,), 8191, (3,)), ((1600, 2), 24, (1600, 1)), ((3, 700), 40, (3, 1))])
def test_residual_step(lead, c, gate, layer, dtype):
    x = make_norm(lead, c, dtype, layer, gate)
    rows = math.prod(lead)
    y, z, grads = run_norm(x, layer, 0.75)
    val, err = norm_reference(x, layer, 0.75, 1e-6, math.prod(gate) if gate is not None else 1)
    inside(y.reshape(rows, c), val['y'], err['y'], 'y')
    inside(z.reshape(rows, c), val['z'], err['z'], 'z')
    for n, g in grads.items():
        assert g.shape == x[n].shape and g.dtype == x[n].dtype
        inside(g.reshape(val['d' + n].shape), val['d' + n], err['d' + n], 'd' + n)


@pytest.mark.parametrize('layer', [False, True])
def test_residual_step_gradients_against_differences(layer):
    x = make_norm((3, 3), 40, FP, layer, (3, 1), seed=2)
    y, z, grads = run_norm(x, layer, 0.75)
    g = torch.Generator().manual_seed(1)
    eps = 2.0 ** -7
    for n, grad in grads.items():
        step = torch.randn(x[n].shape, generator=g).cuda()
        f = []
        for sign in (1, -1):
            t = {m: (None if a is None else a.detach().clone()) for m, a in x.items()}
            t[n] = t[n] + sign * eps * step
            y, z, _ = run_norm(t, layer, 0.75)
            f.append((y.double() * x['dy'].double()).sum() + (z.double() * x['dz'].double()).sum())
        slope, want = float((f[0] - f[1]).detach()) / (2 * eps), float((grad.double() * step.double()).sum())
        # central difference: the next term is of the order of eps^2 (6e-5) of the slope's parts; 720 values off by some 2^-22 over 2 eps
        size = float((grad.double() * step.double()).abs().sum())
        assert abs(slope - want) < 2e-3 * size + 720 * 2.0 ** -22 / (2 * eps), (n, slope, want)


@pytest.mark.parametrize('layer', [False, True])
def test_residual_step_without_a_second_norm_and_with_fp32_weights(layer):
    x = make_norm((3, 50), 320, BF, layer, (3, 1), second=False, param=FP)
    y, z, grads = run_norm(x, layer)
    assert z is None
    val, err = norm_reference(x, layer, 1.0, 1e-6, 3)
    inside(y.reshape(-1, 320), val['y'], err['y'], 'y')
    for n, g in grads.items():
        inside(g.reshape(val['d' + n].shape), val['d' + n], err['d' + n], 'd' + n)


def test_residual_step_where_one_output_has_no_gradient():
    from eo_vae_amd import token_ops as T
    x = make_norm((40,), 96, FP, True, ())
    names = ['h', 'x', 'w1', 'b1', 'w2', 'b2', 'gate']
    leaves = [x[n].requires_grad_(True) for n in names]

    def outs():
        return T.gated_norm_residual(x['h'], x['x'], x['w1'], x['gate'], x['w2'], post_bias=x['b1'], pre_bias=x['b2'], norm='layer')
    zero = torch.zeros_like(x['dy'])
    y, z = outs()
    only_y = torch.autograd.grad(y, leaves, x['dy'], allow_unused=True)
    y, z = outs()
    for n, a, b in zip(names, only_y, torch.autograd.grad([y, z], leaves, [x['dy'], zero])):
        assert torch.equal(a, b), n
    y, z = outs()
    only_z = torch.autograd.grad(z, leaves, x['dz'], allow_unused=True)
    y, z = outs()
    for n, a, b in zip(names, only_z, torch.autograd.grad([y, z], leaves, [zero, x['dz']])):
        assert torch.equal(a, b), n


def test_residual_step_on_constant_rows_and_views():
    from eo_vae_amd import token_ops as T
    c = 264
    w = torch.ones(c, device='cuda')
    h = torch.full((5, c), 3.0, device='cuda')
    y, z = T.gated_norm_residual(h, torch.zeros_like(h), w, pre_weight=w, norm='layer')     # no spread: eps keeps it finite
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(z, torch.zeros_like(z))
    g = torch.Generator().manual_seed(0)
    big = torch.randn(5, 2 * c, generator=g).cuda()
    a, b = T.gated_norm_residual(big[:, 1:c + 1], big[:, c:], w, pre_weight=w)
    a2, b2 = T.gated_norm_residual(big[:, 1:c + 1].contiguous(), big[:, c:].contiguous(), w, pre_weight=w)
    assert torch.equal(a, a2) and torch.equal(b, b2)
    flat = torch.empty(5 * c + 1, device='cuda')
    odd = flat[1:].view(5, c).copy_(big[:, c:])
    assert torch.equal(T.gated_norm_residual(odd, odd, w, pre_weight=w)[1],
                       T.gated_norm_residual(odd.clone(), odd.clone(), w, pre_weight=w)[1])


def test_empty_tensors():
    from eo_vae_amd import token_ops as T
    q = torch.randn(2, 3, 2, 64, device='cuda', requires_grad=True)
    k = torch.randn(2, 0, 2, 64, device='cuda', requires_grad=True)
    out = T.rel_pos_attention(q, k, k)
    assert torch.equal(out, torch.zeros_like(q))
    out.sum().backward()
    assert torch.equal(q.grad, torch.zeros_like(q)) and k.grad.shape == k.shape
    assert T.diff_attention(q[:, :0], q, q, torch.ones(2, device='cuda')).shape == (2, 0, 2, 64)
    h = torch.randn(0, 64, device='cuda')
    y, z = T.gated_norm_residual(h, h, torch.ones(64, device='cuda'), pre_weight=torch.ones(64, device='cuda'))
    assert y.shape == z.shape == (0, 64)


@pytest.mark.parametrize('dtype', [FP, BF])
def test_a_block_of_all_three(dtype):
    """norm -> q k v -> differential attention with position bias -> projection -> gated, normed residual, trained for one step,
    against the same block in 64 bits.  Linear layers and glue are torch's; a block of five roundings per value stays within
    sixteen half steps of its largest value, its gradients (a second pass over all of it) within forty-eight."""
    from eo_vae_amd import token_ops as T
    g = torch.Generator().manual_seed(21)
    b, s, h, d = 2, 48, 2, 64
    c = h * d
    r = lambda *a, std=1.0: (std * torch.randn(*a, generator=g)).to(dtype)                 # noqa: E731
    P = {'x': r(b, s, c), 'w0': 1 + r(c, std=0.1), 'wq': r(c, c, std=c ** -0.5), 'wk': r(c, c, std=c ** -0.5), 'wv': r(c, c, std=c ** -0.5),
         'wo': r(c, c, std=c ** -0.5), 'bias': r(32, h, std=0.5), 'lam': 0.5 + r(h, std=0.1), 'w1': 1 + r(c, std=0.1), 'w2': 1 + r(c, std=0.1),
         'gate': 0.5 + r(b, 1, c, std=0.2)}
    dy, dz = r(b, s, c), r(b, s, c)

    def block(p, mine):
        def norm(a, w):
            a32 = a.float() if a.dtype == BF else a
            return ((a32 / (a32.square().mean(-1, keepdim=True) + 1e-6).sqrt()) * w).to(a.dtype)
        a = norm(p['x'], p['w0'])
        q, k, v = ((a @ p[n].T).view(b, s, h, d) for n in ('wq', 'wk', 'wv'))
        if mine:
            o = T.diff_attention(q, k, v, p['lam'], p['bias'])
            return T.gated_norm_residual(o.reshape(b, s, c) @ p['wo'].T, p['x'], p['w1'], p['gate'], p['w2'])
        rel = torch.arange(s)[None] - torch.arange(s)[:, None]
        bucket = torch.tensor([[reference_bucket(int(e), 32, 128, True) for e in row] for row in rel])
        add = p['bias'][bucket].permute(2, 0, 1)
        maps = [torch.softmax((d // 2) ** -0.5 * q[..., i:i + 32].transpose(1, 2) @ k[..., i:i + 32].permute(0, 2, 3, 1) + add, -1) for i in (0, 32)]
        o = ((maps[0] - p['lam'][:, None, None] * maps[1]) @ v.transpose(1, 2)).transpose(1, 2).reshape(b, s, c)
        y = p['x'] + p['gate'] * norm(o @ p['wo'].T, p['w1'])
        return y, norm(y, p['w2'])
    mine = {n: t.cuda().requires_grad_(True) for n, t in P.items()}
    want = {n: t.double().requires_grad_(True) for n, t in P.items()}
    out, ref = block(mine, True), block(want, False)
    got = torch.autograd.grad(out, list(mine.values()), [dy.cuda(), dz.cuda()])
    exp = torch.autograd.grad(ref, list(want.values()), [dy.double(), dz.double()])
    half = HALF[dtype]
    for name, a, e, steps in [('y', out[0], ref[0], 16), ('z', out[1], ref[1], 16)] + [(n, a, e, 48) for n, a, e in zip(P, got, exp)]:
        e = e.detach()
        off = float((a.detach().double().cpu() - e).abs().max() / e.abs().max())
        assert off < steps * half, (name, off / half)
