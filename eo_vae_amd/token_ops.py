"""Operators over token rows (csrc/token_attn_fwd.hip, token_attn_bwd.hip, token_norm.hip): what a block of a token model needs
next to `ops.attention` and the generators' LayerNorm.

    rel_pos_attention    softmax(scale q k^T + bias[bucket(key - query)]) v, the bias learned by buckets of distance
    diff_attention       the difference of two softmax maps over the same values, weighted by a learned lambda per head
    gated_norm_residual  y = alpha x + gate * norm(h),  z = norm(y): a block's output normed, gated and added, and the
                         next block's normed input, in one pass

float32 and bfloat16; statistics and sums are fp32 in either.  Every operator runs on the tensors' device and its current
stream, allocates through torch (so calls of two streams or two captured graphs share nothing) and is differentiable;
gradients are bit-reproducible.  Wrong arguments raise ValueError, tensors that are not on the GPU EovaeError."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import lib as L

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
MAX_BUCKETS, MAX_REACH, MAX_CHANNELS = 128, 1024, 8192


def _need(cond, text):
    if not cond:
        raise ValueError(text)


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


def _check_gpu(what, t, *others):
    if not t.is_cuda:
        raise L.EovaeError(f'{what}: tensor is on {t.device}; eo_vae_amd kernels only run on an AMD GPU (no CPU fallback) -- '
                           'move the model and inputs to "cuda"')
    for o in others:
        if o is not None and o.device != t.device:
            raise L.EovaeError(f'{what}: tensors on {t.device} and {o.device}')


def _rows16(t):
    """`t` itself where the kernels can read it as it lies (last axis contiguous, rows and address on 16 bytes), else a copy."""
    es = t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s * es % 16 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    return (C.c_longlong * 3)(*(t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)))


def _tracked(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _stream(t):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------


def _describe(q, k, v, bias, lam, kv_len, query_start, maps, two_sided, borders, causal, scale, start):
    """The descriptor of a call; `borders` is a ctypes array that outlives it."""
    d = L.TokenAttention()
    d.q, d.k, d.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    d.q_strides, d.k_strides, d.v_strides = _strides(q), _strides(k), _strides(v)
    d.batch, d.sq, d.heads, d.dim = q.shape
    d.sk, d.kv_heads = k.shape[1], k.shape[2]
    d.dtype, d.maps, d.causal, d.scale, d.start = _DTYPES[q.dtype], maps, int(causal), scale, start
    if bias is not None:
        d.bias, d.bias_dtype, d.buckets, d.two_sided = bias.data_ptr(), _DTYPES[bias.dtype], bias.shape[0], int(two_sided)
        d.borders = C.cast(borders, C.c_void_p).value
    if lam is not None:
        d.lam, d.lam_dtype = lam.data_ptr(), _DTYPES[lam.dtype]
    if kv_len is not None:
        d.kv_len = kv_len.data_ptr()
    if query_start is not None:
        d.query_start = query_start.data_ptr()
    return d


def _call(fn, d, backward, t):
    lib = L.load()
    n = lib.eovae_token_attention_workspace(C.byref(d), backward)
    ws = torch.empty(n, dtype=torch.uint8, device=t.device) if n else None
    if n:
        d.ws, d.ws_bytes = ws.data_ptr(), n
    L.check(getattr(lib, fn)(C.byref(d), _stream(t)), fn)


class TokenAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, lam, kv_len, query_start, keep, maps, two_sided, borders, causal, scale, start):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        bias = None if bias is None else bias.contiguous()
        lam = None if lam is None else lam.contiguous()
        b, sq, h, dim = q.shape
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        rest = (maps, two_sided, borders, causal, scale, start)
        with torch.cuda.device(q.device):
            d = _describe(q, k, v, bias, lam, kv_len, query_start, *rest)
            d.out = out.data_ptr()
            lse = out2 = None
            if keep:
                lse = torch.empty(b, h, maps, sq, dtype=torch.float32, device=q.device)
                d.lse = lse.data_ptr()
                if maps == 2:
                    out2 = torch.empty_like(out)
                    d.out2 = out2.data_ptr()
            _call('eovae_token_attention_fwd', d, 0, q)
        if keep:
            ctx.save_for_backward(q, k, v, bias, lam, kv_len, query_start, out, out2, lse)
            ctx.rest = rest
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        q, k, v, bias, lam, kv_len, query_start, out, out2, lse = ctx.saved_tensors
        d_out = d_out.contiguous()
        if d_out.data_ptr() % 16:
            d_out = d_out.clone()
        empty = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)   # noqa: E731
        dq, dk, dv = empty(q), empty(k), empty(v)
        dbias = empty(bias) if bias is not None and ctx.needs_input_grad[3] else None
        dlam = empty(lam) if lam is not None and ctx.needs_input_grad[4] else None
        with torch.cuda.device(q.device):
            d = _describe(q, k, v, bias, lam, kv_len, query_start, *ctx.rest)
            d.out, d.lse, d.d_out = out.data_ptr(), lse.data_ptr(), d_out.data_ptr()
            d.dq, d.dk, d.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
            if out2 is not None:
                d.out2 = out2.data_ptr()
            if dbias is not None:
                d.dbias = dbias.data_ptr()
            if dlam is not None:
                d.dlam = dlam.data_ptr()
            _call('eovae_token_attention_bwd', d, 1, q)
        return (dq, dk, dv, dbias, dlam) + (None,) * 9


def _attention(what, maps, q, k, v, lam, bias_table, max_distance, bidirectional, causal, scale, kv_len, query_start):
    for n, t in (('q', q), ('k', k), ('v', v)):
        _need(t.dim() == 4, f'{what}: {n} has shape {tuple(t.shape)}, wants [batch, tokens, heads, width]')
        _need(t.dtype in _DTYPES, f'{what}: {n} is {t.dtype} (float32 or bfloat16)')
    _need(q.dtype == k.dtype == v.dtype, f'{what}: q, k, v are {q.dtype}, {k.dtype}, {v.dtype}')
    b, sq, h, dim = q.shape
    _need(k.shape == v.shape, f'{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ')
    sk, hk = k.shape[1], k.shape[2]
    _need(k.shape[0] == b and k.shape[3] == dim, f'{what}: q {tuple(q.shape)} and k {tuple(k.shape)} disagree in batch or width')
    _need(hk > 0 and h % hk == 0, f'{what}: {h} heads over {hk} key heads')
    widths = (32, 64, 128) if maps == 1 else (64, 128)
    _need(dim in widths, f'{what}: head width {dim}, wants one of {widths}')
    _need(max(sq, sk) <= 1 << 28, f'{what}: {sq} queries, {sk} keys (at most 2^28)')
    two_sided, borders = False, None
    if bias_table is not None:
        _need(bias_table.dim() == 2 and bias_table.shape[1] == h, f'{what}: bias_table {tuple(bias_table.shape)}, wants [buckets, {h}]')
        _need(bias_table.dtype in _DTYPES, f'{what}: bias_table is {bias_table.dtype} (float32 or bfloat16)')
        two_sided = bool(bidirectional)
        n = bias_table.shape[0]
        side = n // 2 if two_sided else n
        _need(side >= 2 and n <= MAX_BUCKETS and not (two_sided and n % 2),
              f'{what}: {n} buckets; wants 2 .. {MAX_BUCKETS}, bidirectional an even number of at least 4')
        _need(side // 2 < max_distance <= MAX_REACH, f'{what}: max_distance {max_distance}, wants {side // 2} < max_distance <= {MAX_REACH}')
        edge = bucket_borders(side, int(max_distance))
        borders = (C.c_int * max(1, len(edge)))(*edge)
    if lam is not None:
        _need(lam.shape == (h,), f'{what}: lam has shape {tuple(lam.shape)}, wants [{h}]')
        _need(lam.dtype in _DTYPES, f'{what}: lam is {lam.dtype} (float32 or bfloat16)')
    start = sk - sq
    if isinstance(query_start, int) and not isinstance(query_start, bool):
        _need(abs(query_start) <= 1 << 30, f'{what}: query_start {query_start} (at most 2^30 either way)')
        start, query_start = query_start, None
    elif query_start is None:
        _need(kv_len is None or not (causal or bias_table is not None),
              f'{what}: kv_len with causal or a bias needs query_start (the position of the first query among the keys)')
    for n, t in (('kv_len', kv_len), ('query_start', query_start)):
        if t is not None:
            _need(torch.is_tensor(t) and t.dtype == torch.int32 and t.shape == (b,) and t.is_contiguous(),
                  f'{what}: {n} wants a contiguous int32 tensor [{b}]' + (' or an int' if n == 'query_start' else ''))
    _check_gpu(what, q, k, v, lam, bias_table, kv_len, query_start)
    if scale is None:
        scale = float(dim // maps) ** -0.5
    if q.numel() == 0 or sk == 0:      # nothing to attend to: zeros, tied to the inputs so that gradients are zeros too
        zero = v.sum() * 0 + (0 if lam is None else lam.sum() * 0) + (0 if bias_table is None else bias_table.sum() * 0) + k.sum() * 0
        return q * 0 + zero.to(q.dtype)
    return TokenAttentionFn.apply(q, k, v, bias_table, lam, kv_len, query_start, _tracked(q, k, v, bias_table, lam), maps, two_sided, borders,
                                  bool(causal), float(scale), start)


def rel_pos_attention(q, k, v, bias_table=None, *, max_distance=128, bidirectional=True, causal=False, scale=None, kv_len=None,
                      query_start=None):
    """softmax(scale q k^T + bias_table[bucket(key position - query position)]) v -> [batch, queries, heads, width].

    q [batch, queries, heads, width], k and v [batch, keys, key heads, width], any strides; width 32, 64 or 128; heads a
    multiple of the key heads (head h reads key head h // (heads // key heads)).  scale: width^-0.5.
    bias_table [buckets, heads] (None: no bias): of a side's n buckets the first n // 2 hold one distance each, the others grow
    by equal ratios up to max_distance; bidirectional: half of the table for keys behind and at the query, half for keys
    ahead; otherwise keys ahead count as distance 0.
    kv_len (int32 [batch]): keys at and behind it are not read.  causal: a query sees the keys up to its own position.
    query_start (int, or int32 [batch]): position of the first query among the keys; by default the queries are the last of
    the keys.  With kv_len it has to be given where positions count: 0 for a padded batch, kv_len - queries for a cache that
    the newest tokens have been written to.  A query that sees no key gives zeros and takes no gradient.

    Few queries per key head (at most 32, heads that share it included) run split over the keys, so single tokens against
    a long cache fill the chip; other calls walk the keys once per 128 queries.  The [queries, keys] map is never stored."""
    return _attention('rel_pos_attention', 1, q, k, v, None, bias_table, max_distance, bidirectional, causal, scale, kv_len, query_start)


def diff_attention(q, k, v, lam, bias_table=None, *, max_distance=128, bidirectional=True, causal=False, scale=None, kv_len=None,
                   query_start=None):
    """(softmax(scale q0 k0^T + bias) - lam softmax(scale q1 k1^T + bias)) v: differential attention.

    q0, q1 (k0, k1) are the halves of the last axis of q (k): width 64 or 128, maps of 32 or 64 columns over values of the
    whole width; scale: (width / 2)^-0.5.  lam [heads], learned; everything else as in `rel_pos_attention`."""
    _need(torch.is_tensor(lam), 'diff_attention: lam wants a tensor [heads]')
    return _attention('diff_attention', 2, q, k, v, lam, bias_table, max_distance, bidirectional, causal, scale, kv_len, query_start)


# ------------------------------------------------------------------------------------------
# the residual step
# ------------------------------------------------------------------------------------------


def _norm_desc(h, x, w1, b1, w2, b2, gate, layer, alpha, eps):
    d = L.TokenNorm()
    for n, t in (('h', h), ('x', x), ('w1', w1), ('b1', b1), ('w2', w2), ('b2', b2), ('gate', gate)):
        if t is not None:
            setattr(d, n, t.data_ptr())
    d.channels = h.shape[-1]
    d.rows = h.numel() // d.channels
    d.gates = 0 if gate is None else gate.numel() // d.channels
    d.layer, d.dtype, d.param_dtype, d.alpha, d.eps = int(layer), _DTYPES[h.dtype], _DTYPES[w1.dtype], alpha, eps
    return d


class GatedNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, x, w1, b1, w2, b2, gate, keep, layer, alpha, eps):
        h, x = h.contiguous(), x.contiguous()
        w1, b1, w2, b2, gate = (None if t is None else t.contiguous() for t in (w1, b1, w2, b2, gate))
        y = torch.empty_like(h)
        z = torch.empty_like(h) if w2 is not None else None
        with torch.cuda.device(h.device):
            d = _norm_desc(h, x, w1, b1, w2, b2, gate, layer, alpha, eps)
            d.y = y.data_ptr()
            if z is not None:
                d.z = z.data_ptr()
            stats = None
            if keep:
                stats = torch.empty(d.rows, 4, dtype=torch.float32, device=h.device)
                d.stats = stats.data_ptr()
            L.check(L.load().eovae_token_norm_fwd(C.byref(d), _stream(h)), 'eovae_token_norm_fwd')
        if keep:
            ctx.save_for_backward(h, x, w1, b1, w2, b2, gate, stats)
            ctx.rest = (layer, alpha, eps)
        ctx.set_materialize_grads(False)
        return (y, z) if z is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz=None):
        if dy is None and dz is None:
            return (None,) * 11
        h, x, w1, b1, w2, b2, gate, stats = ctx.saved_tensors
        dy = torch.zeros_like(h) if dy is None else dy.contiguous()
        dz = None if dz is None else dz.contiguous()
        dh, dx = torch.empty_like(h), torch.empty_like(x)
        grads = [None if t is None else torch.empty_like(t) for t in (w1, b1, w2, b2, gate)]
        with torch.cuda.device(h.device):
            d = _norm_desc(h, x, w1, b1, w2, b2, gate, *ctx.rest)
            d.dy, d.dh, d.dx, d.stats = dy.data_ptr(), dh.data_ptr(), dx.data_ptr(), stats.data_ptr()
            if dz is not None:
                d.dz = dz.data_ptr()
            for n, t in zip(('dw1', 'db1', 'dw2', 'db2', 'dgate'), grads):
                if t is not None:
                    setattr(d, n, t.data_ptr())
            lib = L.load()
            n = lib.eovae_token_norm_workspace(C.byref(d))
            ws = torch.empty(n, dtype=torch.uint8, device=h.device)
            d.ws, d.ws_bytes = ws.data_ptr(), n
            L.check(lib.eovae_token_norm_bwd(C.byref(d), _stream(h)), 'eovae_token_norm_bwd')
        return (dh, dx, *grads, None, None, None, None)


def gated_norm_residual(h, x, post_weight, gate=None, pre_weight=None, *, post_bias=None, pre_bias=None, norm='rms', residual_scale=1.0,
                        eps=1e-6):
    """y = residual_scale * x + gate * (norm(h) * post_weight + post_bias);  z = norm(y) * pre_weight + pre_bias  -> (y, z).

    h (a block's output) and x (the residual stream) [..., channels], up to 8192 channels; norm 'rms', or 'layer', which takes
    the biases; pre_weight None: no second norm, z is None.  gate: None, [channels], the shape of h, or the shape of h with
    ones behind its leading axes ([batch, 1, channels]: a gate per sample).  Weights, biases and gate share one type, float32
    or that of h.  z is formed from the unrounded y."""
    what = 'gated_norm_residual'
    _need(h.dtype in _DTYPES, f'{what}: h is {h.dtype} (float32 or bfloat16)')
    _need(h.dim() >= 1 and x.shape == h.shape and x.dtype == h.dtype, f'{what}: h {tuple(h.shape)} {h.dtype} and x {tuple(x.shape)} {x.dtype} differ')
    c = h.shape[-1]
    _need(1 <= c <= MAX_CHANNELS, f'{what}: {c} channels (1 .. {MAX_CHANNELS})')
    _need(norm in ('rms', 'layer'), f"{what}: norm {norm!r} ('rms' or 'layer')")
    _need(norm == 'layer' or (post_bias is None and pre_bias is None), f'{what}: a root-mean-square norm has no bias')
    _need(pre_weight is not None or pre_bias is None, f'{what}: pre_bias without pre_weight')
    _need(post_weight.dtype in (torch.float32, h.dtype), f'{what}: post_weight is {post_weight.dtype} (float32 or {h.dtype})')
    for n, t in (('post_weight', post_weight), ('post_bias', post_bias), ('pre_weight', pre_weight), ('pre_bias', pre_bias)):
        _need(t is None or (t.shape == (c,) and t.dtype == post_weight.dtype), f'{what}: {n} wants {post_weight.dtype} [{c}]')
    if gate is not None:
        lead = tuple(gate.shape[:-1])
        k = len(lead)
        while k and lead[k - 1] == 1:
            k -= 1
        _need(gate.dtype == post_weight.dtype, f'{what}: gate is {gate.dtype}, the weights {post_weight.dtype}')
        _need(gate.dim() >= 1 and gate.shape[-1] == c and (gate.dim() == 1 or gate.dim() == h.dim()) and lead[:k] == tuple(h.shape[:k]),
              f'{what}: gate {tuple(gate.shape)} for h {tuple(h.shape)}: [channels], or the shape of h with ones behind its leading axes')
    _need(float(eps) > 0, f'{what}: eps {eps}')
    _check_gpu(what, h, x, post_weight, post_bias, pre_weight, pre_bias, gate)
    if h.numel() == 0:
        tie = sum(t.sum() * 0 for t in (post_weight, post_bias, pre_weight, pre_bias, gate) if t is not None)
        y = residual_scale * x + h * 0 + tie.to(h.dtype)
        return y, (None if pre_weight is None else y * 1)
    got = GatedNormFn.apply(h, x, post_weight, post_bias, pre_weight, pre_bias, gate,
                            _tracked(h, x, post_weight, post_bias, pre_weight, pre_bias, gate), norm == 'layer', float(residual_scale),
                            float(eps))
    return got if pre_weight is not None else (got, None)
