"""Operators over token rows (csrc/token_attn_fwd.hip, token_attn_bwd.hip, token_norm.hip): what a block of a token model needs
next to `ops.attention` and the generators' LayerNorm.

    rel_pos_attention    softmax(scale q k^T + bias[bucket(key - query)]) v, the bias learned by buckets of distance
    diff_attention       the difference of two softmax maps over the same values, weighted by a learned lambda per head
    gated_norm_residual  y = alpha x + gate * norm(h),  z = norm(y): a block's output normed, gated and added, and the
                         next block's normed input, in one pass

float32 and bfloat16; statistics and sums are fp32 in either.  With bfloat16 tensors what enters a product is bfloat16 too:
probabilities and score gradients are rounded once each, so outputs and gradients of attention are off by the rounding of one such
factor and of the result (2.3e-3 to 2.7e-3 rms, relative, where the result's own rounding is 1.7e-3).  Every operator runs on the tensors' device and its current
stream, allocates through torch (so calls of two streams or two captured graphs share nothing) and is differentiable;
gradients are bit-reproducible.  Forward-mode tangents and functional transforms are refused.  Wrong arguments raise ValueError,
tensors that are not on the GPU EovaeError."""
from __future__ import annotations

import ctypes as C
import functools
import math

import torch
from torch.autograd import forward_ad

from . import lib as L

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
MAX_BUCKETS, MAX_REACH, MAX_CHANNELS = 128, 1024, 8192


@functools.lru_cache(maxsize=64)
def bucket_borders(side, max_distance):
    """First distance of every bucket behind the exact half of one side's `side` buckets: with e = side // 2 exact buckets and
    m = side - e logarithmic ones, bucket e + t begins at the smallest n with n / e >= (max_distance / e)^(t / m), found in
    whole numbers (n^m >= e^(m - t) max_distance^t), so no logarithm decides a border."""
    e = side // 2
    m = side - e
    out = []
    for t in range(1, m):
        lo, hi, want = e, max_distance, e ** (m - t) * max_distance ** t
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid ** m >= want else (mid + 1, hi)
        out.append(lo)
    return tuple(out)


@functools.lru_cache(maxsize=64)
def _borders(side, max_distance):
    """`bucket_borders` as the C array a descriptor points to.  Whoever keeps its address for later (a backward) keeps the array:
    the cache lets go of it."""
    edge = bucket_borders(side, max_distance)
    return (C.c_int * max(1, len(edge)))(*edge)


def _check_gpu(what, t, *others):
    if not t.is_cuda:
        raise L.EovaeError(f'{what}: tensor is on {t.device}; eo_vae_amd kernels only run on an AMD GPU (no CPU fallback) -- '
                           'move the model and inputs to "cuda"')
    dev = t.device
    for o in others:
        if o is not None and o.device != dev:
            raise L.EovaeError(f'{what}: tensors on {dev} and {o.device}')


def _rows16(t):
    """`t` itself where the kernels can read it as it lies (last axis contiguous, rows and address on 16 bytes), else a copy."""
    es = t.element_size()
    st = t.stride()
    if t.data_ptr() % 16 == 0 and st[3] == 1 and st[0] * es % 16 == 0 and st[1] * es % 16 == 0 and st[2] * es % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _flat16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _tracked(*tensors):
    """Whether the call goes through its autograd function: a gradient may be asked for, or an input carries a forward-mode tangent
    (which needs no grad mode, and which the function refuses rather than drops)."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(t):
    return t.new_empty(t.shape)


class _on:
    """The tensor's device for the calls inside (no switch where it is the current one); yields its current stream."""

    def __init__(self, t):
        i = t.device.index
        self.guard = None if i == torch.cuda.current_device() else torch.cuda.device(i)
        self.index = i

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------


def _launch_attention(fn, backward, device, stream, d):
    lib = L.load()
    ref = C.byref(d)
    n = lib.eovae_token_attention_workspace(ref, backward)
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=device)
        d.ws, d.ws_bytes = ws.data_ptr(), n
    L.check(fn(ref, stream), 'token_attention_bwd' if backward else 'token_attention_fwd')


def _describe(q, k, v, out, out2, lse, bias, lam, kv_len, query_start, rest, d_out=None, dq=None, dk=None, dv=None, dbias=None, dlam=None):
    maps, two_sided, borders, causal, scale, start = rest
    b, sq, h, dim = q.shape
    return L.TokenAttention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(out2), _ptr(lse), _ptr(d_out), _ptr(dq), _ptr(dk), _ptr(dv),
        _ptr(dbias), _ptr(dlam), _ptr(bias), _ptr(lam), _ptr(kv_len), _ptr(query_start), None if borders is None else C.addressof(borders), None, 0,
        q.stride()[:3], k.stride()[:3], v.stride()[:3], _DTYPES[q.dtype], 0 if bias is None else _DTYPES[bias.dtype], 0 if lam is None else _DTYPES[lam.dtype], maps,
        b, sq, k.shape[1], h, k.shape[2], dim, start, causal, 0 if bias is None else bias.shape[0], two_sided, scale)


def _attention_forward(q, k, v, bias, lam, kv_len, query_start, keep, rest):
    out = _like(q)
    lse = out2 = None
    if keep:
        b, sq, h, _ = q.shape
        lse = torch.empty((b, h, rest[0], sq), dtype=torch.float32, device=q.device)
        if lam is not None:
            out2 = _like(q)
    with _on(q) as stream:
        d = _describe(q, k, v, out, out2, lse, bias, lam, kv_len, query_start, rest)
        _launch_attention(L.load().eovae_token_attention_fwd, 0, q.device, stream, d)
    return out, out2, lse


class TokenAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, lam, kv_len, query_start, rest):
        out, out2, lse = _attention_forward(q, k, v, bias, lam, kv_len, query_start, True, rest)
        ctx.save_for_backward(q, k, v, bias, lam, kv_len, query_start, out, out2, lse)
        ctx.rest = rest
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        q, k, v, bias, lam, kv_len, query_start, out, out2, lse = ctx.saved_tensors
        d_out = _flat16(d_out)
        dq, dk, dv = _like(q), _like(k), _like(v)
        dbias = _like(bias) if bias is not None and ctx.needs_input_grad[3] else None
        dlam = _like(lam) if lam is not None and ctx.needs_input_grad[4] else None
        with _on(q) as stream:
            d = _describe(_rows16(q), _rows16(k), _rows16(v), out, out2, lse, bias, lam, kv_len, query_start, ctx.rest, d_out, dq, dk, dv,
                          dbias, dlam)
            _launch_attention(L.load().eovae_token_attention_bwd, 1, q.device, stream, d)
        return dq, dk, dv, dbias, dlam, None, None, None


class NoKeysFn(torch.autograd.Function):
    """Attention without keys (or queries): zeros and zero gradients whatever the inputs hold."""

    @staticmethod
    def forward(ctx, *inputs):
        ctx.like = [t if t is None else (t.shape, t.dtype, t.device) for t in inputs]
        return inputs[0].new_zeros(inputs[0].shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        return tuple(torch.zeros(t[0], dtype=t[1], device=t[2]) if need else None for t, need in zip(ctx.like, ctx.needs_input_grad))


def _attention(what, maps, q, k, v, lam, bias_table, max_distance, bidirectional, causal, scale, kv_len, query_start):
    for n, t in (('q', q), ('k', k), ('v', v)):
        if not (t.dim() == 4):
            raise ValueError(f'{what}: {n} has shape {tuple(t.shape)}, wants [batch, tokens, heads, width]')
        if not (t.dtype in _DTYPES):
            raise ValueError(f'{what}: {n} is {t.dtype} (float32 or bfloat16)')
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f'{what}: q, k, v are {q.dtype}, {k.dtype}, {v.dtype}')
    b, sq, h, dim = q.shape
    if not (k.shape == v.shape):
        raise ValueError(f'{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ')
    sk, hk = k.shape[1], k.shape[2]
    if not (k.shape[0] == b and k.shape[3] == dim):
        raise ValueError(f'{what}: q {tuple(q.shape)} and k {tuple(k.shape)} disagree in batch or width')
    if not (hk > 0 and h % hk == 0):
        raise ValueError(f'{what}: {h} heads over {hk} key heads')
    widths = (32, 64, 128) if maps == 1 else (64, 128)
    if not (dim in widths):
        raise ValueError(f'{what}: head width {dim}, wants one of {widths}')
    if not (max(sq, sk) <= 1 << 28 and b <= 1 << 20 and h <= 1 << 16):
        raise ValueError(f'{what}: {sq} queries, {sk} keys (at most 2^28), batch {b} (2^20), {h} heads (2^16)')
    two_sided, borders = False, None
    if bias_table is not None:
        if not (bias_table.dim() == 2 and bias_table.shape[1] == h):
            raise ValueError(f'{what}: bias_table {tuple(bias_table.shape)}, wants [buckets, {h}]')
        if not (bias_table.dtype in _DTYPES):
            raise ValueError(f'{what}: bias_table is {bias_table.dtype} (float32 or bfloat16)')
        two_sided = bool(bidirectional)
        n = bias_table.shape[0]
        side = n // 2 if two_sided else n
        if not (side >= 2 and n <= MAX_BUCKETS and not (two_sided and n % 2)):
            raise ValueError(f'{what}: {n} buckets; wants 2 .. {MAX_BUCKETS}, bidirectional an even number of at least 4')
        if not (isinstance(max_distance, int) and side // 2 < max_distance <= MAX_REACH):
            raise ValueError(f'{what}: max_distance {max_distance}, wants {side // 2} < max_distance <= {MAX_REACH}')
        borders = _borders(side, max_distance)
        bias_table = bias_table.contiguous()
    if lam is not None:
        if not (lam.shape == (h,)):
            raise ValueError(f'{what}: lam has shape {tuple(lam.shape)}, wants [{h}]')
        if not (lam.dtype in _DTYPES):
            raise ValueError(f'{what}: lam is {lam.dtype} (float32 or bfloat16)')
    start = sk - sq
    if isinstance(query_start, int) and not isinstance(query_start, bool):
        if not (abs(query_start) <= 1 << 30):
            raise ValueError(f'{what}: query_start {query_start} (at most 2^30 either way)')
        start, query_start = query_start, None
    elif query_start is None:
        if not (kv_len is None or not (causal or bias_table is not None)):
            raise ValueError(f'{what}: kv_len with causal or a bias needs query_start (the position of the first query among the keys)')
    for n, t in (('kv_len', kv_len), ('query_start', query_start)):
        if t is not None:
            if not (torch.is_tensor(t) and t.dtype == torch.int32 and t.shape == (b,) and t.is_contiguous()):
                raise ValueError(f'{what}: {n} wants a contiguous int32 tensor [{b}]' + (' or an int' if n == 'query_start' else ''))
    scale = float(dim // maps) ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 1e30:
        raise ValueError(f'{what}: scale {scale}')
    _check_gpu(what, q, k, v, lam, bias_table, kv_len, query_start)
    if q.numel() == 0 or sk == 0:      # nothing to attend to
        return NoKeysFn.apply(q, k, v, bias_table, lam)
    args = (_rows16(q), _rows16(k), _rows16(v), bias_table, None if lam is None else lam.contiguous(), kv_len, query_start)
    rest = (maps, two_sided, borders, bool(causal), scale, start)
    if _tracked(q, k, v, bias_table, lam):
        return TokenAttentionFn.apply(*args, rest)
    return _attention_forward(*args, False, rest)[0]


def rel_pos_attention(q, k, v, bias_table=None, *, max_distance=128, bidirectional=True, causal=False, scale=None, kv_len=None,
                      query_start=None):
    """softmax(scale q k^T + bias_table[bucket(key position - query position)]) v -> [batch, queries, heads, width].

    q [batch, queries, heads, width], k and v [batch, keys, key heads, width], any strides; width 32, 64 or 128; heads a
    multiple of the key heads (head h reads key head h // (heads // key heads)).  scale: width^-0.5.
    bias_table [buckets, heads] (None: no bias): of a side's n buckets the first n // 2 hold one distance each, the others grow
    by equal ratios up to max_distance; bidirectional: half of the table for keys behind and at the query, half for keys
    ahead; otherwise keys ahead count as distance 0.  A bias of -infinity shuts keys out; a finite one never does (a query whose
    keys all carry the type's lowest value has the softmax of its scores).
    kv_len (int32 [batch], taken as 0 .. keys): keys at and behind it are not read.  causal: a query sees the keys up to its own position.
    query_start (int, or int32 [batch]): position of the first query among the keys; by default the queries are the last of
    the keys.  With kv_len it has to be given where positions count: 0 for a padded batch, kv_len - queries for a cache that
    the newest tokens have been written to.  A query that sees no key gives zeros and takes no gradient.  Keys that no query
    sees are not read; a NaN or an infinity in the values of a key reaches the queries that see it, and with causal it may reach
    up to 127 queries before them (none that see no key).

    Few queries per key head (at most 32, heads that share it included) run split over the keys, so single tokens against
    a long cache fill the chip; other calls walk the keys once per 128 queries.  The [queries, keys] map is never stored."""
    return _attention('rel_pos_attention', 1, q, k, v, None, bias_table, max_distance, bidirectional, causal, scale, kv_len, query_start)


def diff_attention(q, k, v, lam, bias_table=None, *, max_distance=128, bidirectional=True, causal=False, scale=None, kv_len=None,
                   query_start=None):
    """(softmax(scale q0 k0^T + bias) - lam softmax(scale q1 k1^T + bias)) v: differential attention.

    q0, q1 (k0, k1) are the halves of the last axis of q (k): width 64 or 128, maps of 32 or 64 columns over values of the
    whole width; scale: (width / 2)^-0.5.  lam [heads], learned; everything else as in `rel_pos_attention`."""
    if not (torch.is_tensor(lam)):
        raise ValueError('diff_attention: lam wants a tensor [heads]')
    return _attention('diff_attention', 2, q, k, v, lam, bias_table, max_distance, bidirectional, causal, scale, kv_len, query_start)


# ------------------------------------------------------------------------------------------
# the residual step
# ------------------------------------------------------------------------------------------


def _describe_norm(h, x, w1, b1, w2, b2, gate, stats, rest, y=None, z=None, dy=None, dz=None, dh=None, dx=None, grads=(None,) * 5):
    layer, alpha, eps = rest
    c = h.shape[-1]
    dw1, db1, dw2, db2, dgate = grads
    return L.TokenNorm(
        h.data_ptr(), x.data_ptr(), _ptr(dy), _ptr(dz), _ptr(y), _ptr(z), _ptr(dh), _ptr(dx), w1.data_ptr(), _ptr(b1), _ptr(w2), _ptr(b2),
        _ptr(gate), _ptr(dw1), _ptr(db1), _ptr(dw2), _ptr(db2), _ptr(dgate), _ptr(stats), None, 0, h.numel() // c,
        0 if gate is None else gate.numel() // c, c, layer, _DTYPES[h.dtype], _DTYPES[w1.dtype], alpha, eps)


def _norm_forward(h, x, w1, b1, w2, b2, gate, keep, rest):
    y = _like(h)
    z = _like(h) if w2 is not None else None
    stats = torch.empty((h.numel() // h.shape[-1], 4), dtype=torch.float32, device=h.device) if keep else None
    with _on(h) as stream:
        d = _describe_norm(h, x, w1, b1, w2, b2, gate, stats, rest, y, z)
        L.check(L.load().eovae_token_norm_fwd(C.byref(d), stream), 'token_norm_fwd')
    return y, z, stats


class GatedNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, x, w1, b1, w2, b2, gate, rest):
        y, z, stats = _norm_forward(h, x, w1, b1, w2, b2, gate, True, rest)
        ctx.save_for_backward(h, x, w1, b1, w2, b2, gate, stats)
        ctx.rest = rest
        ctx.set_materialize_grads(False)
        return (y, z) if z is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz=None):
        if dy is None and dz is None:
            return (None,) * 8
        h, x, w1, b1, w2, b2, gate, stats = ctx.saved_tensors
        dy = torch.zeros_like(h) if dy is None else dy.contiguous()
        dz = None if dz is None else dz.contiguous()
        dh, dx = _like(h), _like(x)
        have = [t is not None for t in (w1, b1, w2, b2)]
        rows = iter(w1.new_empty((sum(have), w1.shape[0])).unbind(0))          # one allocation for the [channels] gradients
        grads = [next(rows) if t else None for t in have] + [None if gate is None else _like(gate)]
        with _on(h) as stream:
            d = _describe_norm(h, x, w1, b1, w2, b2, gate, stats, ctx.rest, None, None, dy, dz, dh, dx, grads)
            lib, ref = L.load(), C.byref(d)
            n = lib.eovae_token_norm_workspace(ref)
            ws = torch.empty(n, dtype=torch.uint8, device=h.device)
            d.ws, d.ws_bytes = ws.data_ptr(), n
            L.check(lib.eovae_token_norm_bwd(ref, stream), 'token_norm_bwd')
        return (dh, dx, *grads, None)


def gated_norm_residual(h, x, post_weight, gate=None, pre_weight=None, *, post_bias=None, pre_bias=None, norm='rms', residual_scale=1.0,
                        eps=1e-6):
    """y = residual_scale * x + gate * (norm(h) * post_weight + post_bias);  z = norm(y) * pre_weight + pre_bias  -> (y, z).

    h (a block's output) and x (the residual stream) [..., channels], up to 8192 channels; norm 'rms', or 'layer', which takes
    the biases; pre_weight None: no second norm, z is None.  gate: None, [channels], the shape of h, or the shape of h with
    ones behind its leading axes ([batch, 1, channels]: a gate per sample).  Weights, biases and gate share one type, float32
    or that of h.  z is formed from the unrounded y."""
    what = 'gated_norm_residual'
    if not (h.dtype in _DTYPES):
        raise ValueError(f'{what}: h is {h.dtype} (float32 or bfloat16)')
    if not (h.dim() >= 1 and x.shape == h.shape and x.dtype == h.dtype):
        raise ValueError(f'{what}: h {tuple(h.shape)} {h.dtype} and x {tuple(x.shape)} {x.dtype} differ')
    c = h.shape[-1]
    if not (1 <= c <= MAX_CHANNELS):
        raise ValueError(f'{what}: {c} channels (1 .. {MAX_CHANNELS})')
    if not (norm in ('rms', 'layer')):
        raise ValueError(f"{what}: norm {norm!r} ('rms' or 'layer')")
    if not (norm == 'layer' or (post_bias is None and pre_bias is None)):
        raise ValueError(f'{what}: a root-mean-square norm has no bias')
    if not (pre_weight is not None or pre_bias is None):
        raise ValueError(f'{what}: pre_bias without pre_weight')
    if not (post_weight.dtype in (torch.float32, h.dtype)):
        raise ValueError(f'{what}: post_weight is {post_weight.dtype} (float32 or {h.dtype})')
    for n, t in (('post_weight', post_weight), ('post_bias', post_bias), ('pre_weight', pre_weight), ('pre_bias', pre_bias)):
        if not (t is None or (t.shape == (c,) and t.dtype == post_weight.dtype)):
            raise ValueError(f'{what}: {n} wants {post_weight.dtype} [{c}]')
    if gate is not None:
        lead = tuple(gate.shape[:-1])
        k = len(lead)
        while k and lead[k - 1] == 1:
            k -= 1
        if not (gate.dtype == post_weight.dtype):
            raise ValueError(f'{what}: gate is {gate.dtype}, the weights {post_weight.dtype}')
        if not (gate.dim() >= 1 and gate.shape[-1] == c and (gate.dim() == 1 or gate.dim() == h.dim()) and lead[:k] == tuple(h.shape[:k])):
            raise ValueError(f'{what}: gate {tuple(gate.shape)} for h {tuple(h.shape)}: [channels], or the shape of h with ones behind its leading axes')
    if not 0 < C.c_float(eps).value < math.inf:                     # as the kernels take it
        raise ValueError(f'{what}: eps {eps}')
    if not math.isfinite(C.c_float(residual_scale).value):
        raise ValueError(f'{what}: residual_scale {residual_scale}')
    _check_gpu(what, h, x, post_weight, post_bias, pre_weight, pre_bias, gate)
    if h.numel() == 0:
        tie = sum(t.sum() * 0 for t in (post_weight, post_bias, pre_weight, pre_bias, gate) if t is not None)
        y = residual_scale * x + h * 0 + tie.to(h.dtype)
        return y, (None if pre_weight is None else y * 1)
    args = [None if t is None else t.contiguous() for t in (h, x, post_weight, post_bias, pre_weight, pre_bias, gate)]
    rest = (norm == 'layer', float(residual_scale), float(eps))
    if not _tracked(*args):
        return _norm_forward(*args, False, rest)[:2]
    got = GatedNormFn.apply(*args, rest)
    return got if pre_weight is not None else (got, None)
