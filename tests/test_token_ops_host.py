"""CPU: refusals and host logic of the token operators (eo_vae_amd.token_ops)."""
import ctypes as C

import pytest
import torch

from eo_vae_amd import lib as L
from eo_vae_amd import token_ops as T


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_bucket_borders_are_exact():
    assert T.bucket_borders(16, 128) == (12, 16, 23, 32, 46, 64, 91)      # 8 * 16^(t / 8): 11.3, 16, 22.6, 32, ...
    assert T.bucket_borders(2, 5) == ()
    assert T.bucket_borders(4, 1024) == (46,)                             # sqrt(2 * 1024) = 45.25
    for side in (3, 8, 31, 64, 128):
        b = T.bucket_borders(side, 1024)
        assert len(b) == side - side // 2 - 1 and list(b) == sorted(b) and all(side // 2 <= n <= 1024 for n in b)


@pytest.mark.parametrize('kw,text', [
    (dict(q=t(2, 3, 64)), 'wants \\[batch'),
    (dict(q=t(2, 3, 4, 64, dtype=torch.float16)), 'float32 or bfloat16'),
    (dict(q=t(2, 3, 4, 64, dtype=torch.bfloat16)), 'q, k, v are'),
    (dict(v=t(2, 6, 2, 64)), 'differ'),
    (dict(q=t(1, 3, 4, 64)), 'disagree'),
    (dict(q=t(2, 3, 4, 32)), 'disagree'),
    (dict(q=t(2, 3, 3, 64)), 'heads over'),
    (dict(q=t(2, 3, 4, 48), k=t(2, 5, 2, 48), v=t(2, 5, 2, 48)), 'width 48'),
    (dict(bias_table=t(32, 2)), 'bias_table'),
    (dict(bias_table=t(32)), 'bias_table'),
    (dict(bias_table=t(32, 4, dtype=torch.float64)), 'bias_table is'),
    (dict(bias_table=t(31, 4)), 'buckets'),
    (dict(bias_table=t(2, 4)), 'buckets'),
    (dict(bias_table=t(130, 4)), 'buckets'),
    (dict(bias_table=t(32, 4), max_distance=8), 'max_distance'),
    (dict(bias_table=t(32, 4), max_distance=1025), 'max_distance'),
    (dict(bias_table=t(32, 4), max_distance=64.0), 'max_distance'),
    (dict(scale=float('nan')), 'scale'),
    (dict(scale=float('inf')), 'scale'),
    (dict(kv_len=torch.zeros(2, dtype=torch.int64)), 'kv_len'),
    (dict(kv_len=torch.zeros(3, dtype=torch.int32)), 'kv_len'),
    (dict(kv_len=torch.zeros(2, dtype=torch.int32), causal=True), 'needs query_start'),
    (dict(kv_len=torch.zeros(2, dtype=torch.int32), bias_table=t(32, 4)), 'needs query_start'),
    (dict(query_start=torch.zeros(2)), 'query_start'),
    (dict(query_start=1.0), 'query_start'),
    (dict(query_start=1 << 31), 'query_start'),
])
def test_attention_refuses(kw, text):
    a = dict(q=t(2, 3, 4, 64), k=t(2, 5, 2, 64), v=t(2, 5, 2, 64))
    a.update(kw)
    with pytest.raises(ValueError, match=text):
        T.rel_pos_attention(a.pop('q'), a.pop('k'), a.pop('v'), **a)


@pytest.mark.parametrize('lam,text', [(None, 'lam'), (t(3), 'lam has shape'), (t(4, dtype=torch.float64), 'lam is')])
def test_differential_attention_refuses(lam, text):
    with pytest.raises(ValueError, match=text):
        T.diff_attention(t(2, 3, 4, 64), t(2, 5, 2, 64), t(2, 5, 2, 64), lam)
    with pytest.raises(ValueError, match='width 32'):
        T.diff_attention(t(2, 3, 4, 32), t(2, 5, 2, 32), t(2, 5, 2, 32), t(4))


@pytest.mark.parametrize('kw,text', [
    (dict(h=t(2, 3, 16, dtype=torch.float16)), 'float32 or bfloat16'),
    (dict(x=t(2, 4, 16)), 'differ'),
    (dict(x=t(2, 3, 16, dtype=torch.bfloat16)), 'differ'),
    (dict(h=t(1, 8200), x=t(1, 8200), post_weight=t(8200)), 'channels'),
    (dict(norm='batch'), 'norm'),
    (dict(post_bias=t(16)), 'no bias'),
    (dict(post_weight=t(15)), 'post_weight'),
    (dict(post_weight=t(16, dtype=torch.bfloat16)), 'post_weight'),
    (dict(norm='layer', pre_bias=t(16)), 'without pre_weight'),
    (dict(pre_weight=t(16, dtype=torch.float64)), 'pre_weight'),
    (dict(gate=t(2, 16)), 'gate'),
    (dict(gate=t(1, 3, 16)), 'gate'),
    (dict(gate=t(2, 1, 15)), 'gate'),
    (dict(gate=t(16, dtype=torch.bfloat16)), 'gate'),
    (dict(eps=0.0), 'eps'),
    (dict(eps=float('nan')), 'eps'),
    (dict(residual_scale=float('inf')), 'residual_scale'),
])
def test_residual_step_refuses(kw, text):
    a = dict(h=t(2, 3, 16), x=t(2, 3, 16), post_weight=t(16))
    a.update(kw)
    with pytest.raises(ValueError, match=text):
        T.gated_norm_residual(a.pop('h'), a.pop('x'), a.pop('post_weight'), **a)


def test_tensors_on_the_cpu_are_refused_loudly():
    with pytest.raises(L.EovaeError, match='no CPU fallback'):
        T.rel_pos_attention(t(2, 3, 4, 64), t(2, 5, 2, 64), t(2, 5, 2, 64))
    with pytest.raises(L.EovaeError, match='no CPU fallback'):
        T.gated_norm_residual(t(3, 16), t(3, 16), t(16))


def attention_descriptor(**kw):
    d = L.TokenAttention()
    fake = 1 << 20
    for n in ('q', 'k', 'v', 'out', 'lse', 'd_out', 'dq', 'dk', 'dv'):
        setattr(d, n, fake)
    d.batch, d.sq, d.sk, d.heads, d.kv_heads, d.dim, d.maps, d.scale = 2, 40, 50, 4, 2, 64, 1, 0.125
    for s in (d.q_strides, d.k_strides, d.v_strides):
        s[0], s[1], s[2] = 64 * 200, 256, 64
    for n, v in kw.items():
        if n.endswith('strides'):
            for i in range(3):
                getattr(d, n)[i] = v[i]
        else:
            setattr(d, n, v)
    return d


@pytest.mark.parametrize('kw,text', [
    (dict(q=None), b'null q'), (dict(dtype=2), b'dtype'), (dict(maps=3), b'maps'), (dict(dim=96), b'width'), (dict(dim=32, maps=2), b'width'),
    (dict(heads=5), b'heads'), (dict(batch=0), b'out of range'), (dict(sq=0), b'out of range'), (dict(k_strides=(8, 4, 1)), b'stride'),
    (dict(v_strides=(-64, 64, 64)), b'stride'), (dict(k=(1 << 20) + 4), b'aligned'), (dict(maps=2), b'lambda'), (dict(scale=float('nan')), b'scale'),
    (dict(bias=1 << 20, buckets=300), b'buckets'), (dict(bias=1 << 20, buckets=32), b'borders'),
    (dict(bias=1 << 20, buckets=32, borders=None), b'borders')])
def test_the_library_refuses_descriptors(kw, text):
    lib = L.load()
    d = attention_descriptor(**kw)
    assert lib.eovae_token_attention_fwd(C.byref(d), None) == -1 and text in lib.eovae_last_error()
    assert lib.eovae_token_attention_bwd(C.byref(d), None) == -1 and text in lib.eovae_last_error()
    assert lib.eovae_token_attention_workspace(C.byref(d), 0) == 0


def test_the_library_refuses_bad_borders_and_small_workspaces():
    lib = L.load()
    bad = (C.c_int * 15)(*range(40, 25, -1))
    d = attention_descriptor(bias=1 << 20, buckets=32, borders=C.cast(bad, C.c_void_p).value)
    assert lib.eovae_token_attention_fwd(C.byref(d), None) == -1 and b'border' in lib.eovae_last_error()
    far = (C.c_int * 15)(*range(1020, 1035))
    d = attention_descriptor(bias=1 << 20, buckets=32, borders=C.cast(far, C.c_void_p).value)
    assert lib.eovae_token_attention_fwd(C.byref(d), None) == -1 and b'border' in lib.eovae_last_error()
    d = attention_descriptor(sq=1, sk=5000)
    need = lib.eovae_token_attention_workspace(C.byref(d), 0)
    assert need > 0
    d.ws, d.ws_bytes = 1 << 20, need - 1
    assert lib.eovae_token_attention_fwd(C.byref(d), None) == -1 and b'workspace' in lib.eovae_last_error()
    d = attention_descriptor()
    need = lib.eovae_token_attention_workspace(C.byref(d), 1)
    assert need >= 4 * 2 * 4 * 40
    assert lib.eovae_token_attention_bwd(C.byref(d), None) == -1 and b'workspace' in lib.eovae_last_error()
    assert lib.eovae_token_attention_fwd(None, None) == -1 and b'null descriptor' in lib.eovae_last_error()


def norm_descriptor(**kw):
    d = L.TokenNorm()
    for n in ('h', 'x', 'y', 'w1', 'dy', 'dh', 'dx', 'stats'):
        setattr(d, n, 1 << 20)
    d.rows, d.channels, d.alpha, d.eps = 12, 64, 1.0, 1e-6
    for n, v in kw.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize('kw,text', [
    (dict(rows=0), b'rows'), (dict(channels=8193), b'channels'), (dict(dtype=3), b'dtype'), (dict(param_dtype=-1), b'param'), (dict(gates=3), b'gate'),
    (dict(gates=5, gate=1 << 20), b'gate'), (dict(h=None), b'null h'), (dict(b1=1 << 20), b'bias'), (dict(eps=0.0), b'eps'),
    (dict(alpha=float('inf')), b'alpha')])
def test_the_library_refuses_norm_descriptors(kw, text):
    lib = L.load()
    d = norm_descriptor(**kw)
    assert lib.eovae_token_norm_fwd(C.byref(d), None) == -1 and text in lib.eovae_last_error()
    assert lib.eovae_token_norm_bwd(C.byref(d), None) == -1 and text in lib.eovae_last_error()
    if {'rows', 'channels', 'dtype', 'param_dtype'} & set(kw):
        assert lib.eovae_token_norm_workspace(C.byref(d)) == 0


def test_norm_workspace_is_checked():
    lib = L.load()
    d = norm_descriptor()
    need = lib.eovae_token_norm_workspace(C.byref(d))
    assert need > 0
    d.ws, d.ws_bytes = 1 << 20, need - 4
    assert lib.eovae_token_norm_bwd(C.byref(d), None) == -1 and b'workspace' in lib.eovae_last_error()
    assert lib.eovae_token_norm_fwd(C.byref(norm_descriptor(z=1 << 20)), None) == -1 and b'without w2' in lib.eovae_last_error()
