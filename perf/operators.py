"""Timed cases of the token operators: attention with a bucketed relative position bias, differential attention, and the
normed, gated residual step.  `own` chooses between their plain form (elementary torch operations in 32 bits) and the calls
of `eo_vae_amd.token_ops`."""
import math

import torch

own = False

_T = {'fp32': torch.float32, 'bf16': torch.bfloat16}
BUCKETS, MAX_DISTANCE = 32, 128


def _attn(name, op, mode, dtype, batch, sq, sk, heads, kv_heads, dim, causal, bias, ragged):
    return {'name': name, 'op': op, 'mode': mode, 'dtype': dtype, 'batch': batch, 'sq': sq, 'sk': sk, 'heads': heads,
            'kv_heads': kv_heads, 'dim': dim, 'causal': causal, 'bias': bias, 'ragged': ragged}


def _norm(name, mode, dtype, groups, rows, channels, norm, scale):
    return {'name': name, 'op': 'norm', 'mode': mode, 'dtype': dtype, 'groups': groups, 'rows': rows, 'channels': channels,
            'norm': norm, 'scale': scale}


def listed():
    return [
        # one sequence of 128 weight tokens, 12 wavelengths and a bias token, 4 heads of 64: a weight generator's layer
        _attn('rel_generator_fp32_train', 'rel', 'train', 'fp32', 1, 141, 141, 4, 4, 64, False, True, False),
        # a batch of 32 x 32 latent grids as token rows, trained
        _attn('rel_latents_bf16_train', 'rel', 'train', 'bf16', 16, 1024, 1024, 8, 8, 64, False, True, False),
        # a long prompt with shared key heads, one token short of a round size
        _attn('rel_prompt_bf16_forward', 'rel', 'forward', 'bf16', 1, 8191, 8191, 16, 4, 128, True, True, False),
        # single tokens against a cache that is filled to a different length for each sequence
        _attn('rel_cache_bf16_step', 'rel', 'step', 'bf16', 32, 1, 4096, 16, 4, 128, True, True, True),
        # a causal sequence model over latents, trained
        _attn('diff_causal_bf16_train', 'diff', 'train', 'bf16', 4, 2048, 2048, 8, 8, 128, True, False, False),
        # a small fp32 model over an odd number of tokens, with position bias, trained
        _attn('diff_odd_fp32_train', 'diff', 'train', 'fp32', 2, 577, 577, 4, 4, 64, False, True, False),
        # a batch padded to its longest sequence, inference
        _attn('diff_padded_bf16_forward', 'diff', 'forward', 'bf16', 16, 1000, 1000, 8, 8, 128, False, False, True),
        # few sequences with a very long cache: single tokens
        _attn('diff_cache_bf16_step', 'diff', 'step', 'bf16', 4, 1, 32768, 16, 8, 128, True, False, True),
        # the residual step of 16 sequences' single tokens
        _norm('norm_step_bf16_forward', 'forward', 'bf16', 1, 16, 2048, 'rms', 1.0),
        # the fp32 layer norms of a weight generator's 141 tokens of 256 channels, trained
        _norm('norm_generator_fp32_train', 'train', 'fp32', 1, 141, 256, 'layer', 1.0),
        # 16 latent grids of 1024 tokens, a gate per sample, trained
        _norm('norm_latents_bf16_train', 'train', 'bf16', 16, 1024, 1024, 'rms', 1.0),
        # a wide model's long batch, trained, with a scaled residual stream
        _norm('norm_wide_bf16_train', 'train', 'bf16', 1, 32768, 4096, 'rms', 1.25),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    top = {}
    for c in listed():
        key = 'norm' if c['op'] == 'norm' else 'attn'
        top[key] = max(top.get(key, 0.0), work(c)['flops'])
    while True:
        case = _draw(rng)
        cap = top['norm' if case['op'] == 'norm' else 'attn']
        if case['op'] != 'norm':
            cap /= {'train': 4.0, 'forward': 2.0, 'step': 1.0}[case['mode']]
            if case['dtype'] == 'fp32':
                cap /= 16.0
            if case['batch'] * case['heads'] * case['sq'] * case['sk'] > 400_000_000:
                continue
        if work(case)['flops'] <= cap:
            return case


def _draw(rng):
    op = rng.choice(['rel', 'rel', 'diff', 'diff', 'norm'])
    dtype = rng.choice(['bf16', 'bf16', 'fp32'])
    if op == 'norm':
        return _norm(None, rng.choice(['train', 'forward']), dtype, rng.choice([1, 1, 2, 5, 16]), _log_int(rng, 1, 8192),
                     _log_int(rng, 32, 6000), rng.choice(['rms', 'layer']), rng.choice([1.0, 0.5, 1.25]))
    dim = rng.choice([32, 64, 128] if op == 'rel' else [64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    bias = op == 'rel' or rng.random() < 0.4
    mode = rng.choice(['train', 'train', 'forward', 'step'])
    if mode == 'step':
        return _attn(None, op, mode, dtype, _log_int(rng, 1, 48), rng.choice([1, 1, 1, 2, 4]), _log_int(rng, 33, 32768), heads, kv_heads,
                     dim, True, bias, True)
    s = _log_int(rng, 17, 6000)
    sk = s if rng.random() < 0.7 else _log_int(rng, max(17, s // 4), 4 * s)
    causal = rng.random() < 0.5 and sk >= s
    return _attn(None, op, mode, dtype, _log_int(rng, 1, 24), s, sk, heads, kv_heads, dim, causal, bias,
                 (not causal or s == sk) and rng.random() < 0.3)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    t = _T[case['dtype']]

    def normal(*shape, std=1.0, mean=0.0):
        x = torch.randn(*shape, device='cuda', generator=g, dtype=torch.float32)
        return x.mul_(std).add_(mean).to(t)

    st = {'case': case}
    if case['op'] == 'norm':
        g_, r, c = case['groups'], case['rows'], case['channels']
        wide = 1.0 + 3.0 * (torch.rand(c, device='cuda', generator=g) < 0.02).float()      # a few loud channels
        st['h'] = (torch.randn(g_, r, c, device='cuda', generator=g) * wide).to(t)
        st['x'] = (torch.randn(g_, r, c, device='cuda', generator=g) * (2.0 * wide)).to(t)
        st['post_weight'], st['pre_weight'] = normal(c, std=0.1, mean=1.0), normal(c, std=0.1, mean=1.0)
        st['gate'] = normal(g_, 1, c, std=0.3, mean=0.5)
        layer = case['norm'] == 'layer'
        st['post_bias'] = normal(c, std=0.1) if layer else None
        st['pre_bias'] = normal(c, std=0.1) if layer else None
        st['leaves'] = [st[n] for n in ('h', 'x', 'post_weight', 'post_bias', 'gate', 'pre_weight', 'pre_bias') if st[n] is not None]
        if case['mode'] == 'train':
            st['dy'], st['dz'] = normal(g_, r, c), normal(g_, r, c)
    else:
        b, d = case['batch'], case['dim']
        st['q'] = normal(b, case['sq'], case['heads'], d)
        st['k'] = normal(b, case['sk'], case['kv_heads'], d)
        st['v'] = normal(b, case['sk'], case['kv_heads'], d)
        st['bias'] = normal(BUCKETS, case['heads'], std=0.7) if case['bias'] else None
        st['lam'] = normal(case['heads'], std=0.1, mean=0.5) if case['op'] == 'diff' else None
        st['kv_len'] = st['query_start'] = None
        if case['ragged']:
            low = max(case['sq'] if case['mode'] == 'step' else 1, case['sk'] // 4)
            n = torch.randint(low, case['sk'] + 1, (b,), device='cuda', generator=g)
            st['kv_len'] = n.to(torch.int32)
            if case['mode'] == 'step':
                st['query_start'] = (n - case['sq']).to(torch.int32)
            else:
                st['query_start'] = torch.zeros(b, dtype=torch.int32, device='cuda')
        st['leaves'] = [st[n] for n in ('q', 'k', 'v', 'bias', 'lam') if st[n] is not None]
        if case['mode'] == 'train':
            st['do'] = normal(b, case['sq'], case['heads'], d)
    for x in st['leaves'] if case['mode'] == 'train' else ():
        x.requires_grad_(True)
    return st


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_norm(state) if state['case']['op'] == 'norm' else _plain_attention(state)


def _run_own(st):
    from eo_vae_amd import token_ops
    case = st['case']
    if case['op'] == 'norm':
        outs = token_ops.gated_norm_residual(st['h'], st['x'], st['post_weight'], gate=st['gate'], pre_weight=st['pre_weight'],
                                             post_bias=st['post_bias'], pre_bias=st['pre_bias'], norm=case['norm'],
                                             residual_scale=case['scale'])
        upstream = (st.get('dy'), st.get('dz'))
    else:
        kw = dict(bias_table=st['bias'], max_distance=MAX_DISTANCE, bidirectional=not case['causal'], causal=case['causal'],
                  kv_len=st['kv_len'], query_start=st['query_start'])
        if case['op'] == 'diff':
            out = token_ops.diff_attention(st['q'], st['k'], st['v'], st['lam'], **kw)
        else:
            out = token_ops.rel_pos_attention(st['q'], st['k'], st['v'], **kw)
        outs, upstream = (out,), (st.get('do'),)
    if case['mode'] != 'train':
        return tuple(outs)
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, st['leaves'], upstream)


# ---- the plain form ----------------------------------------------------------------------------------------------------

def _borders(buckets, max_distance):
    """Smallest distance of each logarithmic bucket of one side: the n with n^m >= e^(m-t) * max_distance^t, in whole numbers."""
    e = buckets // 2
    m = buckets - e
    out, n = [], e
    for t in range(1, m):
        while n ** m < e ** (m - t) * max_distance ** t:
            n += 1
        out.append(n)
    return e, out


def _plain_bucket(rel, bidirectional):
    """Bucket of key position minus query position."""
    side = BUCKETS // 2 if bidirectional else BUCKETS
    base = (rel > 0).long() * side if bidirectional else torch.zeros_like(rel)
    n = rel.abs() if bidirectional else (-rel).clamp(min=0)
    e, borders = _borders(side, MAX_DISTANCE)
    far = torch.full_like(n, e)
    for b in borders:
        far = far + (n >= b).long()
    return base + torch.where(n < e, n, far)


def _positions(st):
    case = st['case']
    dev = st['q'].device
    start = st['query_start']
    start = torch.full((1,), case['sk'] - case['sq'], device=dev) if start is None else start.long()
    qp = start[:, None] + torch.arange(case['sq'], device=dev)[None]                      # [B or 1, Sq]
    kp = torch.arange(case['sk'], device=dev)
    rel = kp[None, None, :] - qp[:, :, None]                                              # [B or 1, Sq, Sk]
    seen = torch.ones_like(rel, dtype=torch.bool)
    if case['causal']:
        seen = rel <= 0
    if st['kv_len'] is not None:
        seen = seen & (kp[None, None, :] < st['kv_len'].long()[:, None, None])
    return rel, seen


def _plain_attention(st):
    case = st['case']
    t = st['q'].dtype
    share = case['heads'] // case['kv_heads']
    q = st['q'].float().transpose(1, 2)                                                   # [B, H, Sq, D]
    k = st['k'].float().transpose(1, 2).repeat_interleave(share, 1)
    v = st['v'].float().transpose(1, 2).repeat_interleave(share, 1)
    maps = 2 if case['op'] == 'diff' else 1
    d = case['dim'] // maps
    scale = d ** -0.5
    rel, seen = _positions(st)
    seen = seen[:, None]
    bias = None
    if st['bias'] is not None:
        bucket = _plain_bucket(rel, not case['causal'])
        bias = st['bias'].float()[bucket].permute(0, 3, 1, 2)                              # [B or 1, H, Sq, Sk]
    probs = []
    for i in range(maps):
        s = torch.matmul(q[..., i * d:(i + 1) * d], k[..., i * d:(i + 1) * d].transpose(-1, -2).contiguous()) * scale
        if bias is not None:
            s = s + bias
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        probs.append(p / torch.where(total == 0, torch.ones_like(total), total))
    weights = [1.0] if maps == 1 else [1.0, -st['lam'].float()[None, :, None, None]]
    mix = probs[0] if maps == 1 else probs[0] + weights[1] * probs[1]
    o = torch.matmul(mix, v)
    out = o.transpose(1, 2).to(t).contiguous()
    if case['mode'] != 'train':
        return (out,)
    do = st['do'].float().transpose(1, 2)
    dmix = torch.matmul(do, v.transpose(-1, -2).contiguous())
    fold = lambda x: x.unflatten(1, (case['kv_heads'], share)).sum(2)                     # noqa: E731
    dv = fold(torch.matmul(mix.transpose(-1, -2).contiguous(), do))
    dqs, dks, dlam, dscore = [], [], None, None
    for i, p in enumerate(probs):
        dp = dmix * weights[i]
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        dqs.append(torch.matmul(ds, k[..., i * d:(i + 1) * d]) * scale)
        dks.append(fold(torch.matmul(ds.transpose(-1, -2).contiguous(), q[..., i * d:(i + 1) * d])) * scale)
        dscore = ds if dscore is None else dscore + ds
        if i == 1:
            dlam = -(p * dmix).sum(-1).sum((0, 2), dtype=torch.float64)
    grads = [torch.cat(dqs, -1).transpose(1, 2), torch.cat(dks, -1).transpose(1, 2), dv.transpose(1, 2)]
    if bias is not None:
        dtable = torch.zeros(BUCKETS, case['heads'], dtype=torch.float64, device=out.device)
        shared = bucket.shape[0] == 1
        folded = dscore.sum(0, keepdim=True) if shared else dscore
        for j in range(BUCKETS):
            dtable[j] = torch.where((bucket == j)[:, None], folded, torch.zeros_like(folded)).sum((0, 2, 3), dtype=torch.float64)
        grads.append(dtable)
    if dlam is not None:
        grads.append(dlam)
    return (out,) + tuple(x.to(t).contiguous() for x in grads)


EPS = 1e-6


def _plain_norm(st):
    case = st['case']
    t = st['h'].dtype
    h, x = st['h'].float(), st['x'].float()
    pw, qw, gate = st['post_weight'].float(), st['pre_weight'].float(), st['gate'].float()
    layer = case['norm'] == 'layer'

    def unit(a):
        if layer:
            a = a - a.mean(-1, keepdim=True)
        r = torch.rsqrt((a * a).mean(-1, keepdim=True) + EPS)
        return a * r, r

    def unit_back(da, u, r):
        inner = da - u * (da * u).mean(-1, keepdim=True)
        if layer:
            inner = inner - da.mean(-1, keepdim=True)
        return inner * r

    u1, r1 = unit(h)
    n1 = u1 * pw
    if layer:
        n1 = n1 + st['post_bias'].float()
    y = case['scale'] * x + gate * n1
    u2, r2 = unit(y)
    z = u2 * qw
    if layer:
        z = z + st['pre_bias'].float()
    out = (y.to(t), z.to(t))
    if case['mode'] != 'train':
        return out
    dz = st['dz'].float()
    dy = st['dy'].float() + unit_back(dz * qw, u2, r2)
    dn = dy * gate
    rows = lambda a: a.sum((0, 1), dtype=torch.float64)                                   # noqa: E731
    grads = [unit_back(dn * pw, u1, r1), case['scale'] * dy, rows(dn * u1)]
    if layer:
        grads.append(rows(dn))
    grads += [(dy * n1).sum(1, keepdim=True, dtype=torch.float64), rows(dz * u2)]
    if layer:
        grads.append(rows(dz))
    return out + tuple(a.to(t) for a in grads)


# ---- what one pass has to read, write and compute ----------------------------------------------------------------------

def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'norm':
        n = case['groups'] * case['rows'] * case['channels']
        if case['mode'] == 'train':       # in: h, x, dy, dz; out: y, z, dh, dx
            return {'bytes': 8 * n * size, 'flops': 40 * n}
        return {'bytes': 4 * n * size, 'flops': 14 * n}
    b, sq, sk, d = case['batch'], case['sq'], case['sk'], case['dim']
    keys = 0.625 * sk if case['ragged'] else sk                # lengths lie between a quarter and the whole
    if case['causal'] and case['mode'] != 'step':
        pairs = sq * (sk - sq) + sq * (sq + 1) / 2 if sk >= sq else sk * (sk + 1) / 2
    else:
        pairs = sq * keys
    pairs *= b * case['heads']
    rows_q, rows_k = b * sq * case['heads'] * d, b * keys * case['kv_heads'] * d
    products = 2 if case['mode'] != 'train' else 6             # scores and values; their four gradients
    passes = 1 if case['mode'] != 'train' else 2
    # q and out, k and v (for training their gradients and the upstream one too)
    return {'bytes': size * (2 * rows_q + 2 * rows_k + (passes - 1) * (2 * rows_q + 2 * rows_k)),
            'flops': 2.0 * products * pairs * d}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case['op'] == 'norm':
            return _exact_norm(case, st)
        if case['batch'] * case['heads'] * case['sq'] * case['sk'] * (6 if case['mode'] == 'train' else 2) * case['dim'] > 6e12:
            return None
        return _exact_attention(case, st)


def _exact_table(case, st, head, lo, hi):
    """bucket of every distance lo .. hi (key minus query), and the head's bias there, distance by distance"""
    two_sided = not case['causal']
    side = BUCKETS // 2 if two_sided else BUCKETS
    e = side // 2
    m = side - e
    known = {}
    for n in range(0, MAX_DISTANCE + 1):
        if n < e:
            known[n] = n
        else:
            t = 0
            while t + 1 < m and n ** m >= e ** (m - t - 1) * MAX_DISTANCE ** (t + 1):
                t += 1
            known[n] = e + t
    ids = []
    for r in range(lo, hi + 1):
        n = abs(r) if two_sided else max(-r, 0)
        ids.append(known[min(n, MAX_DISTANCE)] + (side if two_sided and r > 0 else 0))
    return torch.tensor(ids, device='cuda')


def _exact_attention(case, st):
    train = case['mode'] == 'train'
    f = torch.float64
    b, sq, sk, h, d = case['batch'], case['sq'], case['sk'], case['heads'], case['dim']
    share = h // case['kv_heads']
    maps = 2 if case['op'] == 'diff' else 1
    w = d // maps
    out = torch.zeros(b, sq, h, d, dtype=f, device='cuda')
    dq, dk, dv = torch.zeros_like(out), torch.zeros(st['k'].shape, dtype=f, device='cuda'), torch.zeros(st['v'].shape, dtype=f, device='cuda')
    dtable = torch.zeros(BUCKETS, h, dtype=f, device='cuda')
    dlam = torch.zeros(h, dtype=f, device='cuda')
    starts = [sk - sq] * b if st['query_start'] is None else st['query_start'].tolist()
    lens = [sk] * b if st['kv_len'] is None else st['kv_len'].tolist()
    ids = _exact_table(case, st, 0, -(sq + max(starts)), sk - min(starts)) if case['bias'] else None
    for i in range(b):
        n = lens[i]
        if n == 0:
            continue
        rel = torch.arange(n, device='cuda')[None, :] - (starts[i] + torch.arange(sq, device='cuda'))[:, None]
        hidden = (rel > 0) if case['causal'] else torch.zeros_like(rel, dtype=torch.bool)
        blank = hidden.all(1, keepdim=True)
        bucket = ids[rel + sq + max(starts)] if ids is not None else None
        for j in range(h):
            kj, vj = st['k'][i, :n, j // share].to(f), st['v'][i, :n, j // share].to(f)
            qj = st['q'][i, :, j].to(f)
            part = []
            for m in range(maps):
                s = qj[:, m * w:(m + 1) * w] @ kj[:, m * w:(m + 1) * w].T.contiguous() / math.sqrt(w)
                if bucket is not None:
                    s += st['bias'][:, j].to(f)[bucket]
                s.masked_fill_(hidden, -1e300)
                a = torch.softmax(s, 1)
                part.append(a.masked_fill_(hidden | blank, 0.0))
            lam = st['lam'][j].to(f) if maps == 2 else None
            a = part[0] if maps == 1 else part[0] - lam * part[1]
            out[i, :, j] = a @ vj
            if not train:
                continue
            g = st['do'][i, :, j].to(f)
            da = g @ vj.T.contiguous()
            dv[i, :n, j // share] += a.T.contiguous() @ g
            for m in range(maps):
                dam = da if m == 0 else da * -lam
                ds = part[m] * (dam - (part[m] * dam).sum(1, keepdim=True))
                dq[i, :, j, m * w:(m + 1) * w] = ds @ kj[:, m * w:(m + 1) * w] / math.sqrt(w)
                dk[i, :n, j // share, m * w:(m + 1) * w] += ds.T.contiguous() @ qj[:, m * w:(m + 1) * w] / math.sqrt(w)
                if bucket is not None:
                    dtable[:, j] += torch.bincount(bucket.reshape(-1), weights=ds.reshape(-1), minlength=BUCKETS)
            if maps == 2:
                dlam[j] -= (da * part[1]).sum()
    if not train:
        return (out,)
    got = [out, dq, dk, dv]
    if case['bias']:
        got.append(dtable)
    if maps == 2:
        got.append(dlam)
    return tuple(got)


def _exact_norm(case, st):
    f = torch.float64
    layer = case['norm'] == 'layer'
    h, x, gate = st['h'].to(f), st['x'].to(f), st['gate'].to(f)
    pw, qw = st['post_weight'].to(f), st['pre_weight'].to(f)

    def stats(a):
        mean = a.mean(2, keepdim=True) if layer else torch.zeros_like(a[..., :1])
        return mean, ((a - mean).square().mean(2, keepdim=True) + EPS).sqrt()

    m1, s1 = stats(h)
    u1 = (h - m1) / s1
    n1 = u1 * pw + (st['post_bias'].to(f) if layer else 0.0)
    y = x * case['scale'] + n1 * gate
    m2, s2 = stats(y)
    u2 = (y - m2) / s2
    z = u2 * qw + (st['pre_bias'].to(f) if layer else 0.0)
    if case['mode'] != 'train':
        return y, z

    def back(g, u, s):
        g = g / s
        return g - u * (g * u).mean(2, keepdim=True) - (g.mean(2, keepdim=True) if layer else 0.0)

    dz = st['dz'].to(f)
    dy = st['dy'].to(f) + back(dz * qw, u2, s2)
    dn = dy * gate
    got = [y, z, back(dn * pw, u1, s1), dy * case['scale'], (dn * u1).sum((0, 1))]
    if layer:
        got.append(dn.sum((0, 1)))
    got += [(dy * n1).sum(1, keepdim=True), (dz * u2).sum((0, 1))]
    if layer:
        got.append(dz.sum((0, 1)))
    return tuple(got)
