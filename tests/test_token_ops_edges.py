"""CPU: what the token operators (eo_vae_amd.token_ops) keep, refuse and compile to."""
import ctypes as C
import gc
import os
import re
import shutil
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from eo_vae_amd import build as B
from eo_vae_amd import lib as L
from eo_vae_amd import token_ops as T


def listing(name):
    """The compiler's gfx950 output for one kernel source, as {kernel: [instruction, ...]}."""
    hipcc = shutil.which('hipcc') or '/opt/rocm/bin/hipcc'
    if not os.path.exists(hipcc):
        pytest.skip('hipcc not available')
    run = subprocess.run([hipcc, *B.NO_PACKED_FP32, f'--offload-arch={B.ARCH}', '-O3', '-std=c++17', '--offload-device-only', '-S',
                          os.path.join(B.CSRC, name), '-o', '-'], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]
    out, now = {}, None
    for line in run.stdout.split('\n'):
        m = re.match(r'(_Z\w+):', line)
        if m:
            now = out.setdefault(m.group(1), [])
        elif line.startswith('.Lfunc_end'):
            now = None
        elif now is not None and line.startswith('\t') and line[1:2] not in '.;':
            now.append(line.split()[0])
    return out


def test_the_shared_bias_table_is_complete_before_a_wave_reads_it():
    """fp32 dQ of few rows reads keys from memory, so no tile's arrival stands between the block's filling of its bias table and
    the first scores: a barrier of its own has to.  (Instructions up to the key loop's first product lie in program order.)"""
    found = 0
    for name, code in listing('token_attn_bwd.hip').items():
        if 'attn_dq_kernelIf' not in name or 'ELb1E' not in name:
            continue
        found += 1
        before = code[:next(i for i, op in enumerate(code) if op.startswith('v_mfma'))]
        fill = max(i for i, op in enumerate(before) if op.startswith('ds_write'))
        assert 's_barrier' in before[fill:], name
    assert found == 5                                        # widths 32, 64, 128 of one map, 64, 128 of two


def test_a_backward_still_has_its_borders_when_the_cache_has_let_go_of_them(monkeypatch):
    kept = []
    monkeypatch.setattr(T, '_check_gpu', lambda *a: None)
    monkeypatch.setattr(T, '_attention_forward', lambda *a: kept.append(a) or (a[0], None, None))
    q, bias = torch.zeros(1, 4, 2, 64), torch.zeros(32, 2)
    T.rel_pos_attention(q, q, q, bias, max_distance=97)
    *args, keep, rest = kept[0]
    for i in range(100):
        T.rel_pos_attention(q, q, q, bias, max_distance=100 + i)
    kept.clear()
    gc.collect()
    other = [(C.c_int * 7)(*[-1] * 7) for _ in range(4096)]           # what a freed array's memory would be used for
    q, k, v, bias, lam, kv_len, query_start = args
    d = T._describe(q, k, v, q, None, None, bias, lam, kv_len, query_start, rest)
    assert tuple((C.c_int * 7).from_address(d.borders)) == T.bucket_borders(16, 97)
    assert other[0][0] == -1


@pytest.mark.parametrize('mode', ['grad mode', 'no grad mode', 'functional'])
def test_forward_mode_tangents_are_refused(mode, monkeypatch):
    monkeypatch.setattr(T, '_check_gpu', lambda *a: None)
    monkeypatch.setattr(T, '_attention_forward', lambda q, *a: (q.clone(), None, None))
    monkeypatch.setattr(T, '_norm_forward', lambda h, *a: (h.clone(), None, None))
    q, lam, w = torch.randn(1, 4, 2, 64), torch.ones(2), torch.ones(64)
    calls = {'q': lambda a: T.rel_pos_attention(a(q), q, q), 'v': lambda a: T.rel_pos_attention(q, q, a(q)),
             'lam': lambda a: T.diff_attention(q, q, q, a(lam)), 'h': lambda a: T.gated_norm_residual(a(q), q, w)[0],
             'weight': lambda a: T.gated_norm_residual(q, q, a(w))[0]}
    for name, f in calls.items():
        assert not f(lambda t: t).requires_grad
        if mode == 'functional':
            with pytest.raises(RuntimeError, match='functorch|data pointer'):
                x = lam if name == 'lam' else w if name == 'weight' else q
                torch.func.jvp(lambda t: f(lambda _: t), (x,), (x,))
            continue
        with forward_ad.dual_level(), torch.set_grad_enabled(mode == 'grad mode'), pytest.raises(NotImplementedError, match='jvp'):
            f(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
    with forward_ad.dual_level():                             # nothing to refuse where no input has a tangent
        assert torch.equal(calls['q'](lambda t: t), q)


@pytest.mark.parametrize('maps', [1, 2])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_no_keys_give_zeros_whatever_the_inputs_hold(maps, dtype, monkeypatch):
    monkeypatch.setattr(T, '_check_gpu', lambda *a: None)
    q = torch.randn(2, 3, 2, 64).to(dtype)
    q[0, 0], q[1, 2] = float('nan'), float('-inf')
    k = torch.zeros(2, 0, 2, 64, dtype=dtype)
    bias = torch.full((8, 2), float('-inf'))
    lam = torch.tensor([float('inf'), 1.0])
    leaves = [t.requires_grad_(True) for t in ((q, k, bias) if maps == 1 else (q, k, bias, lam))]
    out = T.rel_pos_attention(q, k, k, bias) if maps == 1 else T.diff_attention(q, k, k, lam, bias)
    assert out.dtype == dtype and torch.equal(out, torch.zeros_like(q)) and not torch.signbit(out).any()
    for t, g in zip(leaves, torch.autograd.grad(out, leaves, torch.full_like(out, float('nan')))):
        assert g.dtype == t.dtype and torch.equal(g, torch.zeros_like(t))
    with torch.no_grad():
        assert torch.equal(T.rel_pos_attention(q, k, k, bias), torch.zeros_like(q))
    # no queries: zero gradients for the keys' side
    keys = torch.full((2, 5, 2, 64), float('inf')).to(dtype).requires_grad_(True)
    out = T.rel_pos_attention(q[:, :0], keys, keys, bias)
    assert out.shape == (2, 0, 2, 64)
    for t, g in zip((keys, bias), torch.autograd.grad(out, (keys, bias), torch.zeros_like(out))):
        assert torch.equal(g, torch.zeros_like(t))


def test_a_library_that_lacks_an_entry_is_refused_by_name(monkeypatch):
    monkeypatch.setattr(L, '_lib', None)
    monkeypatch.setitem(L.SIGNATURES, 'eovae_of_a_later_day', (C.c_int, []))
    with pytest.raises(L.EovaeError, match='lacks eovae_of_a_later_day.*rebuild'):
        L.load()
    assert L._lib is None


@pytest.mark.parametrize('newer,rebuilt', [
    (None, 0), ('pkg/csrc/a.hip', 1), ('pkg/csrc/common.h', 2), ('include/abi.h', 2), ('pkg/build.py', 2)])
def test_what_makes_a_built_library_stale(newer, rebuilt, tmp_path, monkeypatch):
    for n in ('pkg/csrc/a.hip', 'pkg/csrc/b.hip', 'pkg/csrc/common.h', 'include/abi.h', 'pkg/build.py', 'pkg/build/a.hip.o', 'pkg/build/b.hip.o',
              'pkg/lib.so'):
        f = tmp_path / n
        f.parent.mkdir(parents=True, exist_ok=True)
        f.write_text('')
        os.utime(f, (1000, 1000 + (f.suffix in ('.o', '.so')) + 2 * (n == newer)))
    for name, path in (('HERE', 'pkg'), ('CSRC', 'pkg/csrc'), ('LIB', 'pkg/lib.so'), ('__file__', 'pkg/build.py')):
        monkeypatch.setattr(B, name, str(tmp_path / path))
    ran = []

    class Compiler:
        returncode = 0

        def __init__(self, cmd, **kw):
            ran.append(cmd)

        def communicate(self):
            return b'', None
    monkeypatch.setattr(B.subprocess, 'Popen', Compiler)
    monkeypatch.setattr(B.subprocess, 'run', lambda cmd, **kw: None)
    monkeypatch.setattr(B.shutil, 'which', lambda n: str(tmp_path / 'pkg/lib.so'))          # any file that is there
    assert B.needs_build() == (newer is not None)
    B.build(verbose=False)
    assert len(ran) == rebuilt


def test_arguments_that_the_kernels_cannot_take_are_value_errors():
    z = torch.zeros
    with pytest.raises(ValueError, match='batch'):
        T.rel_pos_attention(*[z(1, 1, 1, 32).expand((1 << 20) + 1, 1, 1, 32)] * 3)
    with pytest.raises(ValueError, match='heads'):
        T.rel_pos_attention(*[z(1, 1, 1, 32).expand(1, 1, (1 << 16) + 1, 32)] * 3)
    for kw, text in ((dict(eps=1e-60), 'eps'), (dict(eps=1e60), 'eps'), (dict(residual_scale=-1e60), 'residual_scale')):
        with pytest.raises(ValueError, match=text):
            T.gated_norm_residual(z(3, 16), z(3, 16), z(16), **kw)


@pytest.mark.parametrize('kw,text', [(dict(bias=1 << 20, bias_dtype=2), b'bias dtype'), (dict(maps=2, lam=1 << 20, lam_dtype=-1), b'lambda dtype')])
def test_the_library_refuses_types_of_parameters(kw, text):
    from test_token_ops_host import attention_descriptor
    d = attention_descriptor(**kw)
    for call in (L.load().eovae_token_attention_fwd, L.load().eovae_token_attention_bwd):
        assert call(C.byref(d), None) == -1 and text in L.load().eovae_last_error()
