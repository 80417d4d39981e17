"""Token operators (eo_vae_amd.token_ops) at their edges, against their definitions in 64 bits (bounds as in test_gpu_token_ops)."""
import pytest
import torch

from eo_vae_amd import token_ops as T

from test_gpu_token_ops import BF, FP, call, make, run_and_check

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
