"""Cases for the token operators of tcvom_amd.ops: the relative position bias by buckets, the attention that adds it inside, and the
norms before and after a block with its gate and residual scale.

A case is a dict of plain values.  `prepare` makes what a program holds before the call, `run` is one call (a training case: the call
and its gradients), `exact` the same outputs from the definition in 64 bits.  With `own` false `run` computes the operators from
elementary torch operations in 32 bits; with `own` true it calls tcvom_amd.ops.

Definitions
  bias       bias[h, i, j] = table[bucket(j - i - q_start), h].  Distances below `exact` have a bucket each, longer ones share buckets
             whose borders grow geometrically up to max_distance.
  attention  out[b, i, h] = sum_j softmax_j(scale <q[b, i, h], k[b, j, h']> + bias[h, i, j]) v[b, j, h'],  h' = h // (heads / kv_heads),
             over the keys j < k_lens[b] with key_mask[b, j] and, causal, j <= i + q_start[b]; a row without a key is zero.
  block norm x' = residual_scale x + branch_scale gate N(y; post),  h = N(x'; pre),  N = RMSNorm or LayerNorm over the channels.
"""
import math

import torch

own = False

DEV = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed():
    """The token counts are those of a 1088 x 1920 frame at output stride 16 (8160), of half and a quarter of it (4080, 2040), and of a
    512 x 512 crop at stride 16 (1024); 512 channels are the trunk's width."""
    return [
        # the materialised bias of one training step on 512 x 512 crops, and the gradient of its table
        dict(name='bias_train_512', op='bias', train=True, dtype='bf16', heads=8, q_len=1024, k_len=1024, buckets=32, max_distance=128,
             bidirectional=True, q_start=0),
        # a quarter of a frame's tokens against all of them (inference in strips)
        dict(name='bias_strip_1080p', op='bias', train=False, dtype='bf16', heads=8, q_len=2040, k_len=8160, buckets=32, max_distance=128,
             bidirectional=True, q_start=4080),
        # a long training sequence of odd length in 32 bits, one-sided buckets
        dict(name='bias_train_odd_fp32', op='bias', train=True, dtype='fp32', heads=12, q_len=2041, k_len=2041, buckets=64,
             max_distance=400, bidirectional=False, q_start=0),
        # all tokens of a frame at stride 16, inference: the largest forward
        _attn('attn_frame_1080p', 'bf16', False, 1, 8160, 8160, 8, 8, 64),
        # a training step on 512 x 512 crops
        _attn('attn_train_512', 'fp16', True, 4, 1024, 1024, 8, 8, 64),
        # a training step on padded causal sequences with shared key / value heads: the largest of all
        _attn('attn_train_causal_shared', 'bf16', True, 2, 4080, 4080, 16, 4, 128, causal=True, ragged=True),
        # a small window of odd length with holes in its key mask: the smallest prompt
        _attn('attn_small_masked', 'fp16', False, 3, 77, 93, 4, 2, 40, masked=True),
        # one new token against a short cache: latency
        _attn('attn_token_short', 'bf16', False, 1, 1, 197, 8, 8, 64, causal=True, decode=True),
        # one new token a sequence against long ragged caches: bandwidth
        _attn('attn_token_long', 'bf16', False, 8, 1, 32768, 16, 2, 128, causal=True, decode=True, ragged=True),
        # one token a sequence through the norms of a block: latency
        _norm('norm_token', 'bf16', 'bf16', False, 4, 1, 4096, 'rms', 'channel'),
        # the tokens of a frame, 512 channels, 32-bit residual stream, gate of each sample: training
        _norm('norm_train_frame', 'fp32', 'bf16', True, 2, 4080, 512, 'layer', 'sample'),
        # a wide training step, gate of each channel
        _norm('norm_train_wide', 'bf16', 'bf16', True, 4, 2048, 4096, 'rms', 'channel'),
    ]


def _attn(name, dtype, train, batch, q_len, k_len, heads, kv_heads, width, causal=False, ragged=False, masked=False, decode=False,
          buckets=32, max_distance=128):
    return dict(name=name, op='attention', dtype=dtype, train=train, batch=batch, q_len=q_len, k_len=k_len, heads=heads,
                kv_heads=kv_heads, width=width, causal=causal, ragged=ragged, masked=masked, decode=decode, buckets=buckets,
                max_distance=max_distance)


def _norm(name, x_dtype, dtype, train, batch, tokens, channels, kind, gate, residual_scale=1.0, branch_scale=1.0):
    return dict(name=name, op='norm', x_dtype=x_dtype, dtype=dtype, train=train, batch=batch, tokens=tokens, channels=channels, kind=kind,
                gate=gate, residual_scale=residual_scale, branch_scale=branch_scale)


def _cost(case):
    """Rough seconds of a pass at 5 TB/s and 500 TFLOP/s: keeps the drawn cases below the largest listed one."""
    w = work(case)
    return w['bytes'] / 5e12 + w['flops'] / 5e14


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(['bias', 'attention', 'attention', 'token', 'norm', 'norm'])
        half = rng.choice(['bf16', 'fp16'])
        buckets = rng.choice([16, 32, 32, 64, 128])
        reach = rng.choice([128, 128, 200, 512, 1000])
        if op == 'bias':
            case = dict(op='bias', train=rng.random() < 0.5, dtype=rng.choice([half, half, 'fp32']), heads=rng.randint(1, 24),
                        q_len=_log(rng, 1, 4096), k_len=_log(rng, 1, 8192), buckets=buckets, max_distance=reach,
                        bidirectional=rng.random() < 0.6, q_start=rng.choice([0, 0, 7, 500]))
        elif op == 'attention':
            kv = rng.choice([1, 2, 4, 8])
            n = _log(rng, 16, 8192)
            case = _attn(None, half, rng.random() < 0.6, _log(rng, 1, 16), n, n if rng.random() < 0.6 else _log(rng, 16, 8192),
                         kv * rng.choice([1, 1, 2, 4]), kv, rng.choice([32, 40, 64, 64, 96, 128, 128]), causal=rng.random() < 0.5,
                         ragged=rng.random() < 0.5, masked=rng.random() < 0.25, buckets=buckets, max_distance=reach)
        elif op == 'token':
            kv = rng.choice([1, 2, 4, 8])
            case = _attn(None, half, False, _log(rng, 1, 32), rng.choice([1, 1, 1, 2, 4]), _log(rng, 8, 65536),
                         kv * rng.choice([1, 2, 4, 8]), kv, rng.choice([64, 64, 128, 128, 80]), causal=True, decode=True,
                         ragged=rng.random() < 0.7, buckets=buckets, max_distance=reach)
        else:
            case = _norm(None, rng.choice(['fp32', half, half]), half, rng.random() < 0.5, _log(rng, 1, 16), _log(rng, 1, 8192),
                         rng.choice([_log(rng, 16, 8192), 8 * _log(rng, 2, 1024)]), rng.choice(['rms', 'layer']),
                         rng.choice(['none', 'channel', 'sample', 'token']), residual_scale=rng.choice([1.0, 1.0, 0.7]),
                         branch_scale=rng.choice([1.0, 1.0, 1.5]))
        case.pop('name', None)
        if _cost(case) <= top:
            return case


# --------------------------------------------------------------------------------------------- buckets
def _sides(case):
    """(buckets of one side, distances with a bucket of their own)."""
    n = case['buckets'] // 2 if _bidirectional(case) else case['buckets']
    return n, n // 2


def _bidirectional(case):
    return case['bidirectional'] if case['op'] == 'bias' else not case['causal']


def _buckets(case, rel):
    """Bucket of each relative position (an integer tensor): logarithms in 64 bits, nudged past the rounding of the borders that are
    whole numbers (two borders differ by far more)."""
    n, exact = _sides(case)
    d = rel.abs() if _bidirectional(case) else (-rel).clamp(min=0)
    far = torch.floor(torch.log(d.clamp(min=1).double() / exact) / math.log(case['max_distance'] / exact) * (n - exact) + 1e-9).long()
    b = torch.where(d < exact, d, (exact + far).clamp(max=n - 1))
    return b + n * (rel > 0).long() if _bidirectional(case) else b


# --------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {'bias': _prepare_bias, 'attention': _prepare_attention, 'norm': _prepare_norm}[case['op']](case, g)


def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * std


def _prepare_bias(case, g):
    dt = DTYPES[case['dtype']]
    table = _randn(g, case['buckets'], case['heads'])
    s = dict(case=case, table=table)
    if case['train']:
        table.requires_grad_(True)
        s['dout'] = _randn(g, case['heads'], case['q_len'], case['k_len'], std=0.02).to(dt)
    return s


def _prepare_attention(case, g):
    dt, B, D = DTYPES[case['dtype']], case['batch'], case['width']
    Nq, Nk = case['q_len'], case['k_len']
    s = dict(case=case, q=_randn(g, B, Nq, case['heads'], D).to(dt), k=_randn(g, B, Nk, case['kv_heads'], D).to(dt),
             v=_randn(g, B, Nk, case['kv_heads'], D).to(dt), table=_randn(g, case['buckets'], case['heads']), k_lens=None, key_mask=None,
             q_start=0)
    if case['ragged']:                   # lengths between half the padded one and all of it, the first sequence whole
        lens = torch.randint((Nk + 1) // 2, Nk + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        lens[0] = Nk
        s['k_lens'] = lens
    if case['decode']:                   # the queries are the last positions of each sequence
        s['q_start'] = s['k_lens'] - Nq if case['ragged'] else Nk - Nq
    if case['masked']:
        s['key_mask'] = torch.rand(B, Nk, generator=g, device=DEV) < 0.7
    if case['train']:
        for n in ('q', 'k', 'v', 'table'):
            s[n].requires_grad_(True)
        s['dout'] = _randn(g, B, Nq, case['heads'], D).to(dt)
    return s


def _prepare_norm(case, g):
    dt, xt, B, T, C = DTYPES[case['dtype']], DTYPES[case['x_dtype']], case['batch'], case['tokens'], case['channels']
    layer = case['kind'] == 'layer'
    s = dict(case=case, x=_randn(g, B, T, C, std=2.0).to(xt), y=_randn(g, B, T, C).to(dt), post_weight=1 + _randn(g, C, std=0.1),
             post_bias=_randn(g, C, std=0.1) if layer else None, pre_weight=1 + _randn(g, C, std=0.1),
             pre_bias=_randn(g, C, std=0.1) if layer else None)
    shape = {'none': None, 'channel': (C,), 'sample': (B, C), 'token': (B, T, C)}[case['gate']]
    s['gate'] = None if shape is None else 0.5 + _randn(g, *shape, std=0.3)
    if case['gate'] == 'token':          # a gate of every element comes out of the block itself, in its type
        s['gate'] = s['gate'].to(dt)
    if case['train']:
        for n in _NORM_INPUTS:
            if s[n] is not None:
                s[n].requires_grad_(True)
        s['dx'], s['dh'] = _randn(g, B, T, C).to(xt), _randn(g, B, T, C).to(dt)
    return s


_NORM_INPUTS = ('x', 'y', 'post_weight', 'post_bias', 'gate', 'pre_weight', 'pre_bias')
EPS = 1e-6


# --------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state['case']
    if not case['train']:
        with torch.no_grad():
            return _forward(state)
    out = _forward(state)
    names, douts = _differentiated(state)
    outs = out if isinstance(out, tuple) else (out,)
    grads = torch.autograd.grad(outs, [state[n] for n in names], douts)
    return dict([('out%d' % i, o.detach()) for i, o in enumerate(outs)] + [('d_' + n, g) for n, g in zip(names, grads)])


def _differentiated(state):
    op = state['case']['op']
    if op == 'bias':
        return ['table'], [state['dout']]
    if op == 'attention':
        return ['q', 'k', 'v', 'table'], [state['dout']]
    return [n for n in _NORM_INPUTS if state[n] is not None], [state['dx'], state['dh']]


def _forward(s):
    case = s['case']
    if not own:
        return {'bias': _plain_bias, 'attention': _plain_attention, 'norm': _plain_norm}[case['op']](s)
    from tcvom_amd import ops
    if case['op'] == 'bias':
        return ops.relative_position_bias(s['table'], case['q_len'], case['k_len'], max_distance=case['max_distance'],
                                          bidirectional=case['bidirectional'], q_start=case['q_start'], dtype=DTYPES[case['dtype']])
    if case['op'] == 'attention':
        return ops.biased_attention(s['q'], s['k'], s['v'], s['table'], max_distance=case['max_distance'], causal=case['causal'],
                                    k_lens=s['k_lens'], key_mask=s['key_mask'], q_start=s['q_start'])
    return ops.block_norm(s['x'], s['y'], post_weight=s['post_weight'], post_bias=s['post_bias'], gate=s['gate'],
                          branch_scale=case['branch_scale'], residual_scale=case['residual_scale'], pre_weight=s['pre_weight'],
                          pre_bias=s['pre_bias'], kind=case['kind'], eps=EPS)


def _relative(case, q_start, device):
    i = torch.arange(case['q_len'], device=device)[:, None] + q_start
    return torch.arange(case['k_len'], device=device)[None, :] - i


def _plain_bias(s):
    case = s['case']
    b = _buckets(case, _relative(case, case['q_start'], DEV))
    return s['table'].t()[:, b].to(DTYPES[case['dtype']])


def _visible(s):
    """(relative positions [B or 1, Nq, Nk], which keys each query sees [B or 1, Nq, Nk])."""
    case = s['case']
    start = s['q_start'].long()[:, None, None] if torch.is_tensor(s['q_start']) else s['q_start']
    rel = _relative(case, start, DEV)
    rel = rel if rel.dim() == 3 else rel[None]
    see = rel <= 0 if case['causal'] else torch.ones_like(rel, dtype=torch.bool)
    if s['k_lens'] is not None:
        see = see & (torch.arange(case['k_len'], device=DEV) < s['k_lens'][:, None, None])
    if s['key_mask'] is not None:
        see = see & s['key_mask'][:, None, :]
    return rel, see


def _plain_attention(s):
    case = s['case']
    B, Nq, H, D = s['q'].shape
    Nk, Hkv = s['k'].shape[1:3]
    G = H // Hkv
    rel, see = _visible(s)
    # heads that share keys are rows of one product: [B, Hkv, G Nq, D] x [B, Hkv, D, Nk]
    q = s['q'].float().reshape(B, Nq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Nq, D)
    k = s['k'].float().permute(0, 2, 3, 1).contiguous()
    v = s['v'].float().permute(0, 2, 1, 3).contiguous()
    logits = (torch.matmul(q, k) * D ** -0.5).reshape(B, H, Nq, Nk)
    bias = s['table'].t()[:, _buckets(case, rel)].transpose(0, 1)                 # [B or 1, H, Nq, Nk]
    logits = (logits + bias).masked_fill(~see[:, None], -math.inf)
    top = logits.detach().amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.reshape(B, Hkv, G * Nq, Nk), v)
    return out.reshape(B, Hkv, G, Nq, D).permute(0, 3, 1, 2, 4).reshape(B, Nq, H, D).to(s['q'].dtype)


def _plain_norm(s):
    case = s['case']

    def norm(t, w, b):
        if case['kind'] == 'layer':
            t = t - t.mean(-1, keepdim=True)
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) * w
        return t if b is None else t + b

    n = norm(s['y'].float(), s['post_weight'], s['post_bias'])
    if s['gate'] is not None:
        n = n * (s['gate'].float()[:, None, :] if case['gate'] == 'sample' else s['gate'].float())
    x = case['residual_scale'] * s['x'].float() + case['branch_scale'] * n
    return x.to(s['x'].dtype), norm(x, s['pre_weight'], s['pre_bias']).to(s['y'].dtype)


# --------------------------------------------------------------------------------------------- work
def work(case):
    size = {'bf16': 2, 'fp16': 2, 'fp32': 4}
    e = size[case['dtype']]
    if case['op'] == 'bias':
        cells = case['heads'] * case['q_len'] * case['k_len']
        return dict(bytes=(2 if case['train'] else 1) * cells * e, flops=cells if case['train'] else 0)
    if case['op'] == 'norm':
        n = case['batch'] * case['tokens'] * case['channels']
        xe = size[case['x_dtype']]
        gate = n * e if case['gate'] == 'token' else 0
        passes = 2 * (xe + e) * n + gate                                          # x, y in, x', h out
        if case['train']:                                                         # x, y, dx', dh in, dx, dy out
            passes += 3 * (xe + e) * n + 2 * gate
        return dict(bytes=passes, flops=(30 if case['train'] else 10) * n)
    B, H, Hkv, D, Nq, Nk = (case[n] for n in ('batch', 'heads', 'kv_heads', 'width', 'q_len', 'k_len'))
    keys = 0.75 * Nk if case['ragged'] and B > 1 else Nk                          # the mean of the drawn lengths, about
    seen = keys if case['decode'] or not case['causal'] else keys * (1 - 0.5 * min(1.0, keys / Nq)) if keys < Nq else Nq / 2
    pairs = B * H * Nq * seen
    io = e * B * D * (2 * Nq * H + 2 * min(keys, Nq if case['causal'] and not case['decode'] else keys) * Hkv)
    if not case['train']:
        return dict(bytes=io, flops=4 * D * pairs)
    return dict(bytes=2.5 * io, flops=14 * D * pairs)


# --------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {'bias': _exact_bias, 'attention': _exact_attention, 'norm': _exact_norm}[case['op']](case, s)


def _exact_buckets(case, lo, hi):
    """Buckets of the relative positions lo..hi as a list, by integer arithmetic: bucket exact + k starts at the smallest distance d
    with (d / exact)^m >= (max_distance / exact)^k, m = buckets of the side - exact."""
    n, ex = _sides(case)
    m, top = n - ex, case['max_distance']
    starts, d = [], ex
    for k in range(m):
        while d ** m * ex ** k < top ** k * ex ** m:
            d += 1
        starts.append(d)

    def one(rel):
        dist = abs(rel) if _bidirectional(case) else max(-rel, 0)
        b = dist if dist < ex else ex + sum(1 for t in starts if t <= dist) - 1
        return b + n if _bidirectional(case) and rel > 0 else b

    edge = starts[-1]
    near = {r: one(r) for r in range(max(lo, -edge), min(hi, edge) + 1)}
    left, right = one(-edge), one(edge)              # every longer distance shares the last bucket of its side
    return [near[r] if r in near else left if r < 0 else right for r in range(lo, hi + 1)]


def _exact_index(case, starts):
    """Bucket of every (sequence, query, key) from a list over the relative positions: int64 [B, Nq, Nk]."""
    lo, hi = -(case['q_len'] - 1) - max(starts), case['k_len'] - 1 - min(starts)
    by_rel = torch.tensor(_exact_buckets(case, lo, hi), device=DEV)
    i = torch.arange(case['q_len'], device=DEV)[:, None]
    j = torch.arange(case['k_len'], device=DEV)[None, :]
    return torch.stack([by_rel[j - i - st - lo] for st in starts])


def _exact_bias(case, s):
    at = _exact_index(case, [case['q_start']])[0]
    table = s['table'].detach().double()
    out = torch.stack([table[:, h][at] for h in range(case['heads'])])
    if not case['train']:
        return out
    dt = torch.zeros_like(table)
    for h in range(case['heads']):
        dt[:, h].index_add_(0, at.flatten(), s['dout'][h].double().flatten())
    return dict(out0=out, d_table=dt)


def _exact_attention(case, s):
    B, Nq, H, D = s['q'].shape
    G = H // case['kv_heads']
    start = s['q_start'].tolist() if torch.is_tensor(s['q_start']) else [s['q_start']] * B
    lens = s['k_lens'].tolist() if s['k_lens'] is not None else [case['k_len']] * B
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device=DEV)
    table = s['table'].detach().double()
    grads = {n: torch.zeros(s[n].shape, dtype=torch.float64, device=DEV) for n in ('q', 'k', 'v', 'table')} if case['train'] else None
    i = torch.arange(Nq, device=DEV)[:, None]
    for b in range(B):
        at = _exact_index(case, [start[b]])[0]
        keys = torch.arange(case['k_len'], device=DEV)
        ok = (keys < lens[b])[None, :].expand(Nq, -1)
        if s['key_mask'] is not None:
            ok = ok & s['key_mask'][b]
        if case['causal']:
            ok = ok & (keys[None, :] <= i + start[b])
        for h in range(H):
            q, k, v = s['q'][b, :, h].detach().double(), s['k'][b, :, h // G].detach().double(), s['v'][b, :, h // G].detach().double()
            x = (q @ k.t()) / math.sqrt(D) + table[:, h][at]
            x = torch.where(ok, x, torch.full_like(x, -1e300))
            p = torch.where(ok, torch.exp(x - x.max(-1, keepdim=True).values), torch.zeros_like(x))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out[b, :, h] = p @ v
            if not case['train']:
                continue
            do = s['dout'][b, :, h].double()
            dp = do @ v.t()
            ds = p * (dp - (dp * p).sum(-1, keepdim=True))
            grads['v'][b, :, h // G] += p.t() @ do
            grads['q'][b, :, h] = ds @ k / math.sqrt(D)
            grads['k'][b, :, h // G] += ds.t() @ q / math.sqrt(D)
            grads['table'][:, h].index_add_(0, at.flatten(), ds.flatten())
    if not case['train']:
        return out
    return dict([('out0', out)] + [('d_' + n, g) for n, g in grads.items()])


def _exact_norm(case, s):
    f = {n: None if s[n] is None else s[n].detach().double() for n in _NORM_INPUTS}
    layer, rs, bs = case['kind'] == 'layer', case['residual_scale'], case['branch_scale']

    def centre(t):
        return t - t.mean(-1, keepdim=True) if layer else t

    def hat(t):
        c = centre(t)
        r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
        return c * r, r

    def back(da, xh, r):
        return r * (centre(da) - xh * (da * xh).mean(-1, keepdim=True))

    gate = torch.ones((), dtype=torch.float64, device=DEV) if f['gate'] is None else f['gate'][:, None] if case['gate'] == 'sample' else f['gate']
    yh, r1 = hat(f['y'])
    n = yh * f['post_weight'] + (f['post_bias'] if layer else 0)
    x1 = rs * f['x'] + bs * gate * n
    xh, r2 = hat(x1)
    h = xh * f['pre_weight'] + (f['pre_bias'] if layer else 0)
    if not case['train']:
        return x1, h
    dh = s['dh'].double()
    dx1 = s['dx'].double() + back(dh * f['pre_weight'], xh, r2)
    dn = bs * gate * dx1
    dg = bs * dx1 * n
    sums = {'channel': (0, 1), 'sample': (1,), 'token': None, 'none': None}[case['gate']]
    d = dict(x=rs * dx1, y=back(dn * f['post_weight'], yh, r1), post_weight=(dn * yh).sum((0, 1)), post_bias=dn.sum((0, 1)),
             gate=dg.sum(sums) if sums else dg, pre_weight=(dh * xh).sum((0, 1)), pre_bias=dh.sum((0, 1)))
    return dict([('out0', x1), ('out1', h)] + [('d_' + m, d[m]) for m in _NORM_INPUTS if s[m] is not None])
