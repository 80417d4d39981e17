"""Token operators (eo_vae_amd.token_ops) at their edges, against their definitions in 64 bits (bounds as in test_gpu_token_ops)."""
import pytest
import torch

from eo_vae_amd import token_ops as T

from test_gpu_token_ops import BF, FP, call, inside, make, reference, run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('maps,d', [(1, 32), (1, 64), (1, 128), (2, 64), (2, 128)])
@pytest.mark.parametrize('b,sq,sk,h,hk,buckets,max_distance,two_sided,causal,start', [
    (1, 141, 141, 4, 4, 32, 128, True, False, None),
    (2, 577, 577, 4, 4, 32, 128, True, False, None),
    (1, 70, 900, 2, 1, 128, 1024, True, False, 300),      # the widest table
    (1, 40, 700, 2, 2, 8, 20, False, True, 650)])         # most tiles behind the last border: they read the table first of all
def test_small_fp32_backward_repeats_its_bits(b, sq, sk, h, hk, buckets, max_distance, two_sided, causal, start, maps, d):
    x = make(b, sq, sk, h, hk, d, FP, maps, buckets, seed=31)
    out, grads = run_and_check(x, maps, max_distance, two_sided, causal, start=start)
    leaves = [x[n] for n in ('q', 'k', 'v', 'bias', 'lam') if x[n] is not None]
    for _ in range(4):
        again = call(x, maps, max_distance=max_distance, bidirectional=two_sided, causal=causal, query_start=start)
        assert torch.equal(again, out)
        for a, e in zip(torch.autograd.grad(again, leaves, x['do']), grads):
            assert torch.equal(a, e)


@pytest.mark.parametrize('dtype', [FP, BF])
def test_other_bucket_tables_between_a_forward_and_its_backward(dtype):
    x = make(1, 90, 150, 2, 2, 64, dtype, 1, 32, seed=32)
    leaves = [x[n].requires_grad_(True) for n in ('q', 'k', 'v', 'bias')]
    want = torch.autograd.grad(call(x, 1, max_distance=97), leaves, x['do'])
    out = call(x, 1, max_distance=97)
    with torch.no_grad():
        for i in range(100):
            call(x, 1, max_distance=100 + i)
    for a, e in zip(torch.autograd.grad(out, leaves, x['do']), want):
        assert torch.equal(a, e)


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad
    x = make(1, 20, 30, 2, 2, 64, FP, 2, 8, seed=33)
    w = torch.ones(64, device='cuda')
    with forward_ad.dual_level():
        for n in ('q', 'k', 'v', 'bias', 'lam'):
            y = dict(x)
            y[n] = forward_ad.make_dual(x[n], torch.ones_like(x[n]))
            with torch.no_grad(), pytest.raises(NotImplementedError, match='jvp'):
                call(y, 2)
        for n in range(3):
            args = [x['q'], x['do'], w]
            args[n] = forward_ad.make_dual(args[n], torch.ones_like(args[n]))
            with pytest.raises(NotImplementedError, match='jvp'):
                T.gated_norm_residual(*args)


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps', [1, 2])
def test_no_keys_at_all_as_with_lengths_of_zero(maps, dtype):
    x = make(2, 3, 5, 2, 2, 64, dtype, maps, 8, seed=34)
    x['bias'][2:] = float('-inf')
    x['q'][0, 1] = float('inf')
    none = torch.zeros(2, dtype=torch.int32, device='cuda')
    want = call(x, maps, max_distance=20, kv_len=none, query_start=0)
    empty = dict(x, k=x['k'][:, :0], v=x['v'][:, :0])
    got = call(empty, maps, max_distance=20, query_start=0)
    assert torch.equal(got, want) and torch.equal(got, torch.zeros_like(got))
    leaves = [x[n].requires_grad_(True) for n in ('q', 'k', 'v', 'bias', 'lam') if x[n] is not None]
    for keys in (5, 0):
        y = dict(x, k=x['k'][:, :keys], v=x['v'][:, :keys])
        out = call(y, maps, max_distance=20, kv_len=none, query_start=0)
        for g in torch.autograd.grad(out, leaves, x['do']):
            assert torch.equal(g, torch.zeros_like(g))


# A query whose visible keys all carry one very low (or high) finite bias has the softmax of its bare scores: the definition does not
# change when a constant is added to all biases of a row.  So a table with an entry of -1e9 has to act as one whose entry lies
# 200 below the others (e^-200 is 0 beside them, and 64 bits hold scores next to it).
LEVELS = [(m, d, -1e9, -200.0) for m, d in [(1, 32), (1, 64), (1, 128), (2, 64), (2, 128)]] \
    + [(m, d, a, e) for m, d in [(1, 64), (2, 128)] for a, e in [(-100.0, -100.0), (-3.0e38, -200.0), (torch.finfo(FP).min, -200.0), (3.0e38, 200.0)]]


def level_check(x, maps, table, equal, max_distance, two_sided, causal=False, kv_len=None, start=None, scale=None):
    x = dict(x, bias=table.to(x['q'].device))
    leaves = {n: x[n].requires_grad_(True) for n in ('q', 'k', 'v', 'bias', 'lam') if x[n] is not None}
    dev = lambda t: t if t is None or isinstance(t, int) else torch.tensor(t, dtype=torch.int32, device='cuda')   # noqa: E731
    kw = dict(max_distance=max_distance, bidirectional=two_sided, causal=causal, kv_len=dev(kv_len), query_start=dev(start), scale=scale)
    out = call(x, maps, **kw)
    with torch.no_grad():
        assert torch.equal(out, call(x, maps, **kw))
    grads = torch.autograd.grad(out, list(leaves.values()), x['do'])
    w = x['q'].shape[-1] // maps
    val, err = reference(x['q'], x['k'], x['v'], x['do'], maps, w ** -0.5 if scale is None else scale, equal, x['lam'], max_distance, two_sided,
                         causal, kv_len, start)
    inside(out, val['out'], err['out'], 'out')
    for n, g in zip(leaves, grads):
        inside(g, val['d' + n], err['d' + n], 'd' + n)


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('shape', [
    dict(b=1, sq=70, sk=90, h=4, hk=2, two_sided=True),                                            # few blocks: step form, split backward
    dict(b=64, sq=37, sk=75, h=4, hk=4, two_sided=True),                                           # the chip full: row form
    dict(b=1, sq=90, sk=400, h=2, hk=1, two_sided=False, causal=True, start=330),                  # tiles of one bias value, causal
    dict(b=40, sq=131, sk=300, h=4, hk=2, two_sided=False, causal=True, start=250, kv_len=[300, 40, 0, 129] * 10),
    dict(b=3, sq=1, sk=1500, h=8, hk=2, two_sided=False, causal=True, kv_len=[1500, 1, 600], start=[1499, 300, 599]),
    dict(b=1, sq=2, sk=3000, h=4, hk=1, two_sided=True)])
@pytest.mark.parametrize('maps,d,low,near', LEVELS)
def test_rows_whose_keys_all_carry_one_extreme_bias(maps, d, low, near, shape, dtype):
    s = dict(shape)
    x = make(s.pop('b'), s.pop('sq'), s.pop('sk'), h := s.pop('h'), s.pop('hk'), d, dtype, maps, seed=41)
    level_check(x, maps, torch.full((8, h), max(low, torch.finfo(dtype).min), dtype=dtype), torch.zeros(8, h), 60, **s)


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('shape', [
    dict(b=1, sq=140, sk=200, h=4, hk=2, start=100),                      # the first 60 rows see distance 0, the last 40 start 40 behind the keys
    dict(b=64, sq=40, sk=64, h=4, hk=4, start=30),
    dict(b=40, sq=131, sk=300, h=4, hk=2, start=0, kv_len=[300, 40, 0, 90] * 10),     # padded: rows far behind their sequence's end
    dict(b=3, sq=1, sk=1500, h=8, hk=2, kv_len=[1500, 700, 600], start=[1499, 900, 640]),
    dict(b=2, sq=3, sk=3000, h=4, hk=1, kv_len=[2900, 3000], start=[2905, 2997])])
@pytest.mark.parametrize('two_sided', [False, True])
@pytest.mark.parametrize('maps,d,low,near', LEVELS)
def test_rows_that_see_an_extreme_bias_beside_others_or_alone(maps, d, low, near, two_sided, shape, dtype):
    """One-sided and causal, or both sides: keys at distance 8 and more (8 buckets a side, up to 60) carry the extreme."""
    s = dict(shape)
    x = make(s.pop('b'), s.pop('sq'), s.pop('sk'), h := s.pop('h'), s.pop('hk'), d, dtype, maps, seed=42)
    table = torch.randn(16 if two_sided else 8, h, generator=torch.Generator().manual_seed(3))
    equal = table.clone()
    for side in range(0, table.shape[0], 8):                       # in every head but the first
        table[side + 5:side + 8, 1:], equal[side + 5:side + 8, 1:] = low, near
    level_check(x, maps, table, equal, 60, two_sided, causal=not two_sided, **s)


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps', [1, 2])
@pytest.mark.parametrize('high,low', [(-1e9, -2e9), (-3.0e38, torch.finfo(FP).min), (-1000.0, -2000.0), (3.0e38, -3.0e38)])
def test_the_larger_of_two_extremes_wins(high, low, maps, dtype):
    """Distances from 8 on at one level, from 31 on at a lower one; most rows see nothing nearer."""
    for b, sq, sk in ((1, 100, 90), (70, 40, 90)):
        x = make(b, sq, sk, 4, 2, 64, dtype, maps, seed=43)
        table, equal = torch.zeros(8, 4), torch.zeros(8, 4)
        table[5:7], equal[5:7] = high, 200.0 if high > 0 else -200.0
        table[7], equal[7] = low, -400.0
        level_check(x, maps, table, equal, 60, False, True, start=sk + 4)


@pytest.mark.parametrize('dtype', [FP, BF])
def test_a_nan_in_the_table_reaches_the_rows_that_see_it(dtype):
    x = make(1, 60, 80, 2, 2, 64, dtype, 1, 8, seed=44)
    x['bias'] = torch.zeros(8, 2, device='cuda')
    x['bias'][7, 1] = float('nan')                                        # distances of 31 and more
    for start in (20, 200):
        out = call(x, 1, max_distance=60, bidirectional=False, causal=True, query_start=start)
        sees = start + torch.arange(60) >= 200 if start == 200 else start + torch.arange(60) >= T.bucket_borders(8, 60)[-1]
        assert torch.isnan(out[0, :, 1]).all(-1).cpu().equal(sees) and not torch.isnan(out[0, :, 0]).any()


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps,d', [(1, 32), (1, 64), (1, 128), (2, 64), (2, 128)])
@pytest.mark.parametrize('b,sq,sk,h,hk,causal,start,lens', [
    (1, 40, 90, 2, 2, False, 0, [70]), (1, 40, 90, 2, 1, True, 20, None), (1, 333, 210, 6, 1, False, 0, [150]),
    (64, 37, 75, 4, 4, False, 0, [75, 0, 40, 64] * 16)])
def test_keys_that_no_query_sees_take_no_gradient_of_a_nan(b, sq, sk, h, hk, causal, start, lens, maps, d, dtype):
    x = make(b, sq, sk, h, hk, d, dtype, maps, 8, seed=45)
    x['do'][:, sq // 2, 0, 3] = float('nan')
    x['q'][:, sq - 1] = float('inf')
    leaves = [x[n].requires_grad_(True) for n in ('k', 'v')]
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device='cuda')
    out = call(x, maps, max_distance=20, causal=causal, bidirectional=not causal, query_start=start, kv_len=n)
    for g in torch.autograd.grad(out, leaves, x['do']):
        for i in range(b):
            last = start + sq if causal else lens[i]
            assert torch.equal(g[i, last:], torch.zeros_like(g[i, last:]))
            assert last == 0 or torch.isnan(g[i, :last]).any()


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps,d', [(1, 32), (1, 64), (1, 128), (2, 64), (2, 128)])
@pytest.mark.parametrize('b,h,sq,sk', [(1, 2, 30, 40), (64, 4, 40, 50), (2, 4, 6, 2000)])
def test_queries_that_see_no_key_stay_zero_beside_keys_that_hold_nan(b, h, sq, sk, maps, d, dtype):
    """Causal, the first query five positions before the first key: five rows see nothing, the sixth sees a NaN."""
    x = make(b, sq, sk, h, h, d, dtype, maps, 8, seed=46)
    x['k'][:, 0], x['v'][:, 0] = float('nan'), float('inf')
    q = x['q'].requires_grad_(True)
    out = call(x, maps, max_distance=20, causal=True, bidirectional=False, query_start=-5)
    (dq,) = torch.autograd.grad(out, [q], x['do'])
    for t in (out, dq):
        assert torch.equal(t[:, :5], torch.zeros_like(t[:, :5])) and torch.isnan(t[:, 5:]).any(-1).all()


def rms_off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


@pytest.mark.parametrize('sk', [4096, 16000])
def test_two_maps_over_a_long_cache_round_like_one(sk):
    """bf16, lambda 0.8: a rounding to 8 bits is off by 1.66e-3 rms of values whose mantissas are spread evenly over a binade's logarithm.
    Weights and output rounded once: sqrt(2) times that, 2.35e-3.  Weights of two maps rounded apart, the second's counting 0.8 and
    both positive where the difference is not: 2.53e-3 and more.  A wave's first tile of at least four is still apart, so at most
    sqrt((3 * 2.35^2 + 2.65^2) / 4) = 2.43e-3."""
    x = make(4, 1, sk, 16, 8, 128, BF, 2, seed=47)
    x['lam'] = torch.full((16,), 0.8, device='cuda')
    out = call(x, 2)
    val, _ = reference(x['q'], x['k'], x['v'], x['do'], 2, 64 ** -0.5, None, x['lam'])
    assert rms_off(out, val['out']) < 2.43e-3


@pytest.mark.parametrize('maps,d', [(1, 64), (1, 128), (2, 64), (2, 128)])
def test_key_gradients_are_rounded_twice_and_no_more(maps, d):
    """bf16, rows of some hundred keys with a bias gradient: the score gradient's rounding into its product and dK's own, 1.66e-3 rms
    each (mantissas spread evenly over a binade's logarithm), are 2.35e-3; a delta from outputs in bf16 would add about 1.2e-3 to
    that square, 2.64e-3.  The bound lies between, 3 % above the first for the mantissas of a sample."""
    x = make(2, 300, 300, 8, 8, d, BF, maps, 32, seed=48)
    leaves = [x[n].requires_grad_(True) for n in ('k', 'bias')]
    dk, _ = torch.autograd.grad(call(x, maps), leaves, x['do'])
    w = d // maps
    val, _ = reference(x['q'], x['k'], x['v'], x['do'], maps, w ** -0.5, x['bias'], x['lam'])
    assert rms_off(dk, val['dk']) < 2.42e-3


@pytest.mark.parametrize('dtype', [FP, BF])
@pytest.mark.parametrize('maps', [1, 2])
@pytest.mark.parametrize('b,sq,sk', [(1, 40, 60), (64, 40, 60)])
def test_a_nan_key_reaches_all_gradients_of_the_rows_that_see_it(b, sq, sk, maps, dtype):
    """Its softmax has no value, whether or not the call also asks for the parameters' gradients."""
    x = make(b, sq, sk, 4, 4, 64, dtype, maps, 8, seed=49)
    x['k'][:, 7] = float('nan')
    for names in (('q', 'k', 'v'), ('q', 'k', 'v', 'bias') + (('lam',) if maps == 2 else ())):
        y = {n: None if t is None else t.detach().clone() for n, t in x.items()}
        leaves = [y[n].requires_grad_(True) for n in names]
        out = call(y, maps, max_distance=20)
        assert torch.isnan(out).all()
        dq, dk = torch.autograd.grad(out, leaves, y['do'])[:2]
        assert torch.isnan(dq).all() and torch.isnan(dk).all()
