"""GPU parity of the token operators (tcvom_amd/token_ops.py): relative position bias, attention with it, norms around a block, forward
and gradients against plain implementations in 64 bits on the CPU.

Tolerances, from the roundings alone.  u = eps / 2 of the 16-bit type: half a step.
  * bias matrix: one rounding, u |value|.  Table gradient: fp32 sums, 2^-24 a partial sum, far below 1e-6 of the sum of magnitudes.
  * norms: 32-bit arithmetic and one rounding at the end, u |value| plus a few 2^-24 of the terms' sizes, taken as 1e-6 of the largest.
  * attention: out = sum p v with p rounded to 16 bits, relative error u each: at most u sum |p| |v|, then the rounding of the result, u |out|;
    the same for gradients with the magnitudes of what is summed (`slack` below computes those sums).  The 32-bit part (scores of
    magnitude |x| <= 64 in base 2, hardware exponentials) adds 2^-24 |x| relative, taken as 2e-5.
"""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tcvom_amd import _lib as L
from tcvom_amd import ops
from tcvom_amd.token_ops import rel_buckets

pytestmark = pytest.mark.gpu
DEV = 'cuda'
HALF = [torch.bfloat16, torch.float16]
ids = lambda t: str(t).replace('torch.', '') if isinstance(t, torch.dtype) else None  # noqa: E731


def step(dt):
    return 2.0 ** -24 if dt == torch.float32 else torch.finfo(dt).eps / 2


def rnd(*shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64) * std


def bucket_matrix(n, max_distance, bidirectional, nq, nk, start):
    """Bucket of every (query, key) by the definition, one element at a time."""
    b = rel_buckets(n, max_distance, bidirectional)
    side = n // 2 if bidirectional else n

    def one(rel):
        d = abs(rel) if bidirectional else max(-rel, 0)
        k = d if d < b.exact else b.exact - 1 + sum(1 for s in b.starts[:b.n_starts] if s <= d)
        return k + (side if bidirectional and rel > 0 else 0)

    lo = -(nq - 1) - start
    line = torch.tensor([one(r) for r in range(lo, nk - start)] or [0])
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None, :]
    return line[(j - i - start) - lo]


def close(got, want, bound, what=''):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound).max().item() if want.numel() else 0.0
    assert over <= 0, '%s: %.3g over a bound of %.3g' % (what, over, float(torch.as_tensor(bound).max()))


# --------------------------------------------------------------------------------------------- bias matrix
BIAS = [
    # heads, q_len, k_len, buckets, max_distance, bidirectional, q_start
    (1, 1, 1, 32, 128, True, 0),
    (3, 7, 13, 8, 16, True, 0),
    (2, 65, 64, 32, 128, False, 0),
    (5, 130, 401, 32, 128, True, 37),
    (2, 1, 1000, 32, 128, False, 999),
    (4, 333, 517, 64, 200, True, -20),
    (2, 257, 1500, 128, 1000, True, 300),
    (1, 40, 33, 4, 3, True, 5),
    (2, 20, 30, 256, 1024, False, 5000),
    (1, 300, 3, 2, 2, False, -400),
]


@pytest.mark.parametrize('dt', HALF + [torch.float32], ids=ids)
@pytest.mark.parametrize('case', BIAS, ids=lambda c: 'x'.join(str(int(v)) for v in c))
def test_bias_matrix_and_its_gradient(case, dt):
    H, nq, nk, n, far, bidir, start = case
    table = rnd(n, H, seed=1).float()
    leaf = table.to(DEV).requires_grad_(True)
    out = ops.relative_position_bias(leaf, nq, nk, max_distance=far, bidirectional=bidir, q_start=start, dtype=dt)
    at = bucket_matrix(n, far, bidir, nq, nk, start)
    want = table.double().t()[:, at]
    assert out.dtype == dt
    close(out, want, step(dt) * want.abs(), 'bias')
    dout = rnd(H, nq, nk, seed=2).to(dt)
    g, = torch.autograd.grad(out, leaf, dout.to(DEV))
    wg, size = torch.zeros(n, H, dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)
    for h in range(H):
        wg[:, h].index_add_(0, at.flatten(), dout[h].double().flatten())
        size[:, h].index_add_(0, at.flatten(), dout[h].double().abs().flatten())
    close(g, wg, 1e-6 * size, 'table gradient')
    again, = torch.autograd.grad(ops.relative_position_bias(leaf, nq, nk, far, bidir, start, dt), leaf, dout.to(DEV))
    assert torch.equal(g, again)


def test_bias_matrix_of_no_rows_and_no_columns():
    leaf = rnd(32, 2).float().to(DEV).requires_grad_(True)
    for nq, nk in ((0, 5), (5, 0)):
        out = ops.relative_position_bias(leaf, nq, nk)
        assert out.shape == (2, nq, nk)
        g, = torch.autograd.grad(out, leaf, torch.zeros_like(out))
        assert not g.any()


# --------------------------------------------------------------------------------------------- norms
def norm64(x, y, w1, b1, gate, rows, bs, rs, w2, b2, layer, eps):
    def n(t, w, b):
        t = t - t.mean(-1, keepdim=True) if layer else t
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * w
        return t if b is None else t + b

    C = x.shape[-1]
    if y is None:
        return None, n(x, w2, b2)
    t = y if w1 is None else n(y, w1, b1)
    if gate is not None:
        t = gate.reshape(-1, 1, C).expand(-1, rows, C).reshape(x.shape) * t
    xo = rs * x + bs * t
    return xo, None if w2 is None else n(xo, w2, b2)


NORM_TYPES = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
              (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]
NORMS = [
    # shape, kind, post, gate, pre, branch_scale, residual_scale, offset (elements the tensors start off a 16-byte boundary)
    ((1, 1, 128), 'rms', True, 'channel', True, 1.0, 1.0, 0),
    ((2, 9, 64), 'layer', True, 'sample', True, 0.5, 1.0, 0),
    ((3, 33, 512), 'rms', True, 'token', True, 1.0, 0.7, 0),
    ((2, 70, 1000), 'layer', True, 'channel', True, 2.0, 1.3, 0),
    ((4, 5, 2048), 'rms', False, None, True, 1.0, 1.0, 0),
    ((2, 3, 4096), 'layer', True, 'sample', False, 1.0, 1.0, 0),
    ((1, 3, 8192), 'layer', True, 'token', True, 1.0, 1.0, 0),
    ((5, 7, 37), 'layer', True, 'sample', True, 1.0, 1.0, 0),
    ((3, 11, 1001), 'rms', True, 'channel', True, 1.0, 1.0, 0),
    ((1, 2, 5001), 'layer', True, 'channel', True, 1.0, 1.0, 0),
    ((130, 1, 96), 'rms', True, 'sample', True, 1.0, 1.0, 0),
    ((700, 40), 'rms', None, None, True, 1.0, 1.0, 0),
    ((2, 17, 256), 'rms', True, 'channel', True, 1.0, 1.0, 1),
    ((1500, 128), 'layer', True, 'channel', True, 1.0, 1.0, 0),
    ((3, 1), 'rms', True, 'channel', True, 1.0, 1.0, 0),
]


@pytest.mark.parametrize('types', NORM_TYPES, ids=lambda t: '%s-%s' % (ids(t[0]), ids(t[1])))
@pytest.mark.parametrize('case', NORMS, ids=lambda c: '%s-%s-%s' % ('x'.join(map(str, c[0])), c[1], c[3]))
def test_block_norm_and_its_gradients(case, types):
    shape, kind, post, gate, pre, bs, rs, off = case
    xt, yt = types
    C, layer, eps = shape[-1], kind == 'layer', 1e-6
    gshape = {None: None, 'channel': (C,), 'sample': (shape[0], C), 'token': shape}[gate]
    rows = {None: 1, 'channel': math.prod(shape[:-1]), 'sample': math.prod(shape[1:-1]), 'token': 1}[gate]
    host = dict(x=(rnd(*shape, seed=1, std=2.0) + 0.5).to(xt), y=None if post is None else (rnd(*shape, seed=2) - 0.3).to(yt),
                w1=1 + rnd(C, seed=3, std=0.2) if post else None, b1=rnd(C, seed=4, std=0.2) if post and layer else None,
                gate=None if gate is None else (0.5 + rnd(*gshape, seed=5, std=0.3)).to(yt if gate == 'token' else torch.float32),
                w2=1 + rnd(C, seed=6, std=0.2) if pre else None, b2=rnd(C, seed=7, std=0.2) if pre and layer else None)
    for n in ('w1', 'b1', 'w2', 'b2'):
        host[n] = None if host[n] is None else host[n].float()

    def on_gpu(t):
        if t is None:
            return None
        flat = torch.empty(t.numel() + off, dtype=t.dtype, device=DEV)
        flat[off:] = t.flatten().to(DEV)
        return flat[off:].view(t.shape).requires_grad_(True)

    dev = {n: on_gpu(t) for n, t in host.items()}
    ref = {n: None if t is None else t.double().requires_grad_(True) for n, t in host.items()}
    xo, h = ops.block_norm(dev['x'], dev['y'], dev['w1'], dev['b1'], dev['gate'], bs, rs, dev['w2'], dev['b2'], kind, eps)
    wxo, wh = norm64(ref['x'], ref['y'], ref['w1'], ref['b1'], ref['gate'], rows, bs, rs, ref['w2'], ref['b2'], layer, eps)
    outs, wants, douts = [], [], []
    if post is None:
        assert xo is dev['x']
    else:
        outs, wants, douts = [xo], [wxo], [rnd(*shape, seed=8).to(xt)]
    if pre:
        outs, wants, douts = outs + [h], wants + [wh], douts + [rnd(*shape, seed=9).to(yt)]
    else:
        assert h is None
    for o, w in zip(outs, wants):
        w = w.detach()
        assert o.dtype == (yt if o is h and post is not None else o.dtype)
        close(o, w, step(o.dtype) * w.abs() * (1 + 1e-3) + 2e-6 * (1 + w.abs().max()), 'output')
    names = [n for n in host if host[n] is not None]
    got = torch.autograd.grad(outs, [dev[n] for n in names], [d.to(DEV) for d in douts])
    want = torch.autograd.grad(wants, [ref[n] for n in names], [d.double() for d in douts])
    tokens = math.prod(shape[:-1])
    for n, g, w in zip(names, got, want):
        assert g.dtype == host[n].dtype and g.shape == host[n].shape
        # sums over the tokens of terms about as large as the largest entry of a token's: fp32 errors grow with sqrt(tokens) at most
        scale = w.abs().max() + (math.sqrt(tokens) if n in ('w1', 'b1', 'w2', 'b2', 'gate') else 1.0)
        extra = 16 if C == 1 else 1                     # one channel: 1 / |t| amplifies
        close(g, w, step(g.dtype) * w.abs() * (1 + 1e-3) + 4e-6 * extra * scale, n)
    again = torch.autograd.grad(ops.block_norm(dev['x'], dev['y'], dev['w1'], dev['b1'], dev['gate'], bs, rs, dev['w2'], dev['b2'], kind, eps)
                                [0 if post is not None else 1:2 if pre else 1], [dev[n] for n in names], [d.to(DEV) for d in douts])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize('types', NORM_TYPES, ids=lambda t: '%s-%s' % (ids(t[0]), ids(t[1])))
def test_block_norm_types(types):
    """x' has x's type and h has y's, or x's without y; each within the rounding of that type."""
    xt, yt = types
    x, y, w = rnd(6, 72, seed=1).to(xt), rnd(6, 72, seed=2).to(yt), 1 + rnd(72, seed=3, std=0.2).float()
    for grad in (False, True):
        dev = [t.to(DEV).requires_grad_(grad) for t in (x, y, w)]
        xo, h = ops.block_norm(dev[0], dev[1], post_weight=dev[2], pre_weight=dev[2])
        h0 = ops.block_norm(dev[0], None, pre_weight=dev[2])[1]
        wxo, wh = norm64(x.double(), y.double(), w.double(), None, None, 1, 1.0, 1.0, w.double(), None, False, 1e-6)
        wh0 = norm64(x.double(), None, None, None, None, 1, 1.0, 1.0, w.double(), None, False, 1e-6)[1]
        for got, want, t in ((xo, wxo, xt), (h, wh, yt), (h0, wh0, xt)):
            assert got.dtype == t
            close(got, want, step(t) * want.abs() * (1 + 1e-3) + 2e-6 * (1 + want.abs().max()))


def test_block_norm_passes_only_one_gradient():
    x, y, w = rnd(4, 6, 256, seed=1).float(), rnd(4, 6, 256, seed=2).float(), 1 + rnd(256, seed=3, std=0.1).float()
    for which in (0, 1):
        dev = [t.to(DEV).requires_grad_(True) for t in (x, y, w, w)]
        ref = [t.double().requires_grad_(True) for t in (x, y, w, w)]
        o = ops.block_norm(dev[0], dev[1], post_weight=dev[2], pre_weight=dev[3])[which]
        r = norm64(ref[0], ref[1], ref[2], None, None, 1, 1.0, 1.0, ref[3], None, False, 1e-6)[which]
        (o * o).sum().backward()
        (r * r).sum().backward()
        for d, t in zip(dev, ref):
            if t.grad is None:
                assert d.grad is None
            else:
                close(d.grad, t.grad, 1e-5 * (1 + t.grad.abs().max()), str(which))


def test_block_norm_keeps_nan_and_inf_in_their_rows():
    x, y, w = rnd(8, 128, seed=1).bfloat16(), rnd(8, 128, seed=2).bfloat16(), torch.ones(128)
    y[3, 5], y[6, 0] = float('nan'), float('inf')
    xo, h = ops.block_norm(x.to(DEV), y.to(DEV), post_weight=w.to(DEV), pre_weight=w.to(DEV))
    bad = ~torch.isfinite(h.float()).all(-1).cpu()
    assert bad.tolist() == [False] * 3 + [True] + [False] * 2 + [True] + [False]


# --------------------------------------------------------------------------------------------- attention
def attention64(q, k, v, table, at, see, scale):
    """Outputs, and for each what the 16-bit rounding of the probabilities can add: sum |p| |v|."""
    H, Hkv = q.shape[2], k.shape[2]
    k, v = (t.repeat_interleave(H // Hkv, 2) for t in (k, v))
    x = scale * torch.einsum('bihd,bjhd->bhij', q, k) + table.t()[:, at].transpose(0, 1)
    x = x.masked_fill(~see[:, None], -math.inf)
    top = x.amax(-1, keepdim=True) if x.shape[-1] else x.new_zeros(x.shape[:-1] + (1,))
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top).detach())
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.einsum('bhij,bjhd->bihd', p, torch.where(see.any(1)[:, :, None, None], v, torch.zeros_like(v))), p


ATTN = [
    # B, Nq, Nk, H, Hkv, D, causal, k_lens, mask, q_start, buckets, max_distance
    dict(B=1, Nq=1, Nk=1, H=1, Hkv=1, D=8),
    dict(B=2, Nq=33, Nk=65, H=2, Hkv=1, D=32),
    dict(B=2, Nq=64, Nk=64, H=4, Hkv=4, D=64, causal=True),
    dict(B=1, Nq=129, Nk=200, H=2, Hkv=2, D=40),
    dict(B=3, Nq=77, Nk=93, H=4, Hkv=2, D=40, mask=True),
    dict(B=2, Nq=300, Nk=300, H=4, Hkv=1, D=128, causal=True, lens=[300, 177]),
    dict(B=3, Nq=65, Nk=130, H=2, Hkv=2, D=64, lens=[0, 1, 130]),
    dict(B=2, Nq=257, Nk=190, H=2, Hkv=2, D=96, causal=True, start=-100),
    dict(B=2, Nq=40, Nk=517, H=6, Hkv=2, D=128, causal=True, start=[477, 100], lens=[517, 140]),
    dict(B=1, Nq=513, Nk=700, H=2, Hkv=2, D=64, buckets=64, far=700),
    dict(B=1, Nq=200, Nk=333, H=2, Hkv=2, D=16, buckets=4, far=3, mask=True, causal=True),
    dict(B=2, Nq=150, Nk=150, H=3, Hkv=3, D=64, causal=True, bidirectional=True),
    # few queries
    dict(B=1, Nq=1, Nk=197, H=8, Hkv=8, D=64, causal=True, start=196),
    dict(B=4, Nq=1, Nk=700, H=8, Hkv=2, D=128, causal=True, start=[699, 0, -1, 300], lens=[700, 1, 0, 301]),
    dict(B=2, Nq=5, Nk=3000, H=16, Hkv=2, D=64, causal=True, start=[2995, 1200], lens=[3000, 1205]),
    dict(B=2, Nq=3, Nk=900, H=4, Hkv=4, D=80, mask=True),
    dict(B=1, Nq=32, Nk=1100, H=4, Hkv=2, D=32, buckets=128, far=1000),
    dict(B=1, Nq=2, Nk=0, H=2, Hkv=2, D=64),
    dict(B=1, Nq=70, Nk=0, H=2, Hkv=2, D=64),
]


def attn_case(c, dt):
    B, Nq, Nk, H, Hkv, D = (c[n] for n in ('B', 'Nq', 'Nk', 'H', 'Hkv', 'D'))
    causal, n, far = c.get('causal', False), c.get('buckets', 32), c.get('far', 128)
    bidir = c.get('bidirectional', not causal)
    start = c.get('start', 0)
    starts = start if isinstance(start, list) else [start] * B
    lens = c.get('lens')
    mask = torch.rand(B, Nk, generator=torch.Generator().manual_seed(9)) < 0.6 if c.get('mask') else None
    host = dict(q=rnd(B, Nq, H, D, seed=1).to(dt), k=rnd(B, Nk, Hkv, D, seed=2).to(dt), v=rnd(B, Nk, Hkv, D, seed=3).to(dt),
                table=rnd(n, H, seed=4).float())
    at = torch.stack([bucket_matrix(n, far, bidir, Nq, Nk, s) for s in starts])
    i, j = torch.arange(Nq)[:, None], torch.arange(Nk)[None, :]
    see = torch.stack([(j < (lens[b] if lens else Nk)) & ((j <= i + starts[b]) if causal else (j >= 0)) for b in range(B)])
    if mask is not None:
        see = see & mask[:, None]
    kw = dict(max_distance=far, causal=causal, bidirectional=c.get('bidirectional'),
              k_lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV),
              key_mask=None if mask is None else mask.to(DEV),
              q_start=torch.tensor(start, dtype=torch.int32, device=DEV) if isinstance(start, list) else start)
    return host, at, see, kw


def attn_id(c):
    return '-'.join('%s%s' % (k, '_'.join(map(str, v)) if isinstance(v, list) else int(v)) for k, v in c.items())


@pytest.mark.parametrize('dt', HALF, ids=ids)
@pytest.mark.parametrize('case', ATTN, ids=attn_id)
def test_attention_and_its_gradients(case, dt):
    host, at, see, kw = attn_case(case, dt)
    D, u = case['D'], step(dt)
    G = case['H'] // case['Hkv']
    ref = {n: t.double().requires_grad_(True) for n, t in host.items()}
    want, p = attention64(ref['q'], ref['k'], ref['v'], ref['table'], at, see, D ** -0.5)
    v_abs = host['v'].double().abs().repeat_interleave(G, 2)
    spread = torch.einsum('bhij,bjhd->bihd', p.detach(), v_abs)
    want_d = want.detach()
    with torch.no_grad():                                   # inference: the few-query kernel where it applies
        out = ops.biased_attention(*(host[n].to(DEV) for n in ('q', 'k', 'v', 'table')), **kw)
    close(out, want_d, u * want_d.abs() * 1.01 + (u + 2e-5) * spread + 1e-7, 'out')
    # what is hidden from everybody may hold anything
    hidden = ~see.any(1)
    bad_k, bad_v = host['k'].clone(), host['v'].clone()
    bad_k[hidden], bad_v[hidden] = float('nan'), float('inf')
    if not (case.get('causal') and kw['k_lens'] is None and kw['key_mask'] is None) or case['Nk'] <= case['Nq']:
        with torch.no_grad():
            assert torch.equal(out, ops.biased_attention(host['q'].to(DEV), bad_k.to(DEV), bad_v.to(DEV), host['table'].to(DEV), **kw))
    # gradients
    leaf = {n: t.to(DEV).requires_grad_(True) for n, t in host.items()}
    out = ops.biased_attention(leaf['q'], leaf['k'], leaf['v'], leaf['table'], **kw)
    close(out, want_d, u * want_d.abs() * 1.01 + (u + 2e-5) * spread + 1e-7, 'training out')
    dout = rnd(*host['q'].shape, seed=5).to(dt)
    names = ['q', 'k', 'v', 'table']
    got = dict(zip(names, torch.autograd.grad(out, [leaf[n] for n in names], dout.to(DEV))))
    want_g = dict(zip(names, torch.autograd.grad(want, [ref[n] for n in names], dout.double())))
    # magnitudes of what the rounding of p and ds (u each) is summed over
    with torch.no_grad():
        do = dout.double()
        vv, kk = (host[n].double().repeat_interleave(G, 2) for n in ('v', 'k'))
        vv = torch.where(see.any(1)[:, :, None, None], vv, torch.zeros_like(vv))
        dp = torch.einsum('bihd,bjhd->bhij', do, vv)
        delta = (p * dp).sum(-1, keepdim=True)
        ds = (p * (dp - delta)).abs()
        size = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True))          # ds without its cancellation: 32-bit errors go by this
        kt, qt = kk.abs(), host['q'].double().abs()
        group = lambda t: t.reshape(t.shape[0], t.shape[1], case['Hkv'], G, D).sum(3)  # noqa: E731
        slack = dict(q=D ** -0.5 * torch.einsum('bhij,bjhd->bihd', u * ds + 2e-5 * size, kt),
                     k=group(D ** -0.5 * torch.einsum('bhij,bihd->bjhd', u * ds + 2e-5 * size, qt)),
                     v=group(torch.einsum('bhij,bihd->bjhd', (u + 2e-5) * p, do.abs())))
        st = torch.zeros_like(want_g['table'])
        for b in range(case['B']):
            for h in range(case['H']):
                st[:, h].index_add_(0, at[b].flatten(), size[b, h].flatten())
        slack['table'] = (2e-5 + u * u) * st
    for n in names:
        w = want_g[n]
        assert got[n].dtype == host[n].dtype
        # fp16: results and operands below 2^-14 step by 2^-24
        tiny = 0.0 if n == 'table' else 1e-6 if dt == torch.bfloat16 else 2.0 ** -25 * (2 + case['Nk'] + case['Nq'] * G)
        close(got[n], w, (u * 1.01 if n != 'table' else 1e-6) * w.abs() + slack[n] + tiny, 'd' + n)
    again = torch.autograd.grad(ops.biased_attention(leaf['q'], leaf['k'], leaf['v'], leaf['table'], **kw), [leaf[n] for n in names], dout.to(DEV))
    for n, a in zip(names, again):
        assert torch.equal(got[n], a), n


FROZEN = [
    dict(B=2, Nq=1, Nk=197, H=4, Hkv=2, D=64),
    dict(B=2, Nq=5, Nk=3000, H=8, Hkv=2, D=64, causal=True, start=[2995, 1200], lens=[3000, 1205]),
    dict(B=1, Nq=32, Nk=1100, H=4, Hkv=2, D=32, mask=True),
    dict(B=2, Nq=130, Nk=150, H=4, Hkv=4, D=128, causal=True, lens=[150, 0]),
    dict(B=3, Nq=77, Nk=93, H=2, Hkv=1, D=40),
]


@pytest.mark.parametrize('dt', HALF, ids=ids)
@pytest.mark.parametrize('case', FROZEN, ids=attn_id)
def test_gradients_with_a_frozen_table(case, dt):
    """Without the table's gradient the forward keeps its 16-bit output only: <dout, out> is off by the roundings of p and of out, u (|out| + sum
    p |v|) |dout| together, and ds by p times that."""
    host, at, see, kw = attn_case(case, dt)
    D, u, G = case['D'], step(dt), case['H'] // case['Hkv']
    ref = {n: t.double().requires_grad_(n != 'table') for n, t in host.items()}
    want, p = attention64(ref['q'], ref['k'], ref['v'], ref['table'], at, see, D ** -0.5)
    dout = rnd(*host['q'].shape, seed=5).to(dt)
    names = ['q', 'k', 'v']
    want_g = dict(zip(names, torch.autograd.grad(want, [ref[n] for n in names], dout.double())))
    leaf = {n: t.to(DEV).requires_grad_(n != 'table') for n, t in host.items()}
    out = ops.biased_attention(leaf['q'], leaf['k'], leaf['v'], leaf['table'], **kw)
    got = dict(zip(names, torch.autograd.grad(out, [leaf[n] for n in names], dout.to(DEV))))
    with torch.no_grad():
        do = dout.double()
        vv, kk = (host[n].double().repeat_interleave(G, 2) for n in ('v', 'k'))
        vv = torch.where(see.any(1)[:, :, None, None], vv, torch.zeros_like(vv))
        dp = torch.einsum('bihd,bjhd->bhij', do, vv)
        ds = (p * (dp - (p * dp).sum(-1, keepdim=True))).abs()
        size = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True))
        spread = torch.einsum('bhij,bjhd->bihd', p, vv.abs())
        off = 1.01 * u * (do.abs() * (want.abs() + spread)).sum(-1).permute(0, 2, 1)[..., None] * p
        group = lambda t: t.reshape(t.shape[0], t.shape[1], case['Hkv'], G, D).sum(3)  # noqa: E731
        e = u * (ds + off) + off + 2e-5 * size
        slack = dict(q=D ** -0.5 * torch.einsum('bhij,bjhd->bihd', e, kk.abs()),
                     k=group(D ** -0.5 * torch.einsum('bhij,bihd->bjhd', e, host['q'].double().abs())),
                     v=group(torch.einsum('bhij,bihd->bjhd', (u + 2e-5) * p, do.abs())))
    close(out, want.detach(), u * want.detach().abs() * 1.01 + (u + 2e-5) * spread + 1e-7, 'out')
    for n in names:
        tiny = 1e-6 if dt == torch.bfloat16 else 2.0 ** -25 * (2 + case['Nk'] + case['Nq'] * G)
        close(got[n], want_g[n], u * 1.01 * want_g[n].abs() + slack[n] + tiny, 'd' + n)
    # asked for one at a time, and together with the table's: v's gradient does not change (its p and dout are the same)
    for n in names:
        one = {m: t.to(DEV).requires_grad_(m == n) for m, t in host.items()}
        g, = torch.autograd.grad(ops.biased_attention(one['q'], one['k'], one['v'], one['table'], **kw), [one[n]], dout.to(DEV))
        assert torch.equal(g, got[n]), n


DOUTS = [
    dict(B=1, Nq=300, Nk=4000, H=2, Hkv=1, D=64),
    dict(B=2, Nq=300, Nk=300, H=4, Hkv=1, D=128, causal=True, lens=[300, 177]),
    dict(B=1, Nq=130, Nk=517, H=2, Hkv=2, D=32),
    dict(B=1, Nq=700, Nk=200, H=2, Hkv=2, D=40, mask=True),
]


@pytest.mark.parametrize('dt', HALF, ids=ids)
@pytest.mark.parametrize('std', [1e-4, 1.0, 4e3, 'rows'])
@pytest.mark.parametrize('which', ['q', 'k'])
@pytest.mark.parametrize('case', DOUTS, ids=attn_id)
def test_gradients_of_small_and_large_douts(case, which, std, dt):
    """dout of deviation 1e-4, 1, 4000 (with values of 16: score gradients up to 1e6) and 1e-3 .. 1e3 from row to row.  The other operand of the
    product is lifted or lowered by 2^6, so that the gradient itself is within fp16's range: what the score gradients lose would show.  Bound of an
    element: its own rounding (u |w|, or half of fp16's last step, 2^-24) and, as independent errors, those of the ds it sums, u |ds| each
    plus the 32-bit part.  Twice their deviation bounds the root mean square of error / bound by 1 (equally distributed roundings have half a step
    / sqrt 3)."""
    host, at, see, kw = attn_case(case, dt)
    other = 'k' if which == 'q' else 'q'
    lift = {1e-4: 64.0, 4e3: 1 / 64}.get(std, 1.0)
    host[other], host[which] = host[other] * lift, host[which] / lift
    if std == 4e3:
        host['v'] = host['v'] * 16
    D, u, G = case['D'], step(dt), case['H'] // case['Hkv']
    size = 10.0 ** torch.linspace(-3, 3, case['Nq'], dtype=torch.float64)[None, :, None, None] if std == 'rows' else std
    dout = (rnd(*host['q'].shape, seed=5) * size).to(dt)
    ref = {n: t.double().requires_grad_(n == which) for n, t in host.items()}
    want, p = attention64(ref['q'], ref['k'], ref['v'], ref['table'], at, see, D ** -0.5)
    w, = torch.autograd.grad(want, ref[which], dout.double())
    leaf = {n: t.to(DEV).requires_grad_(True) for n, t in host.items()}
    out = ops.biased_attention(leaf['q'], leaf['k'], leaf['v'], leaf['table'], **kw)
    g, = torch.autograd.grad(out, leaf[which], dout.to(DEV))
    assert torch.isfinite(g).all()
    with torch.no_grad():
        vv, kk = (host[n].double().repeat_interleave(G, 2) for n in ('v', 'k'))
        vv = torch.where(see.any(1)[:, :, None, None], vv, torch.zeros_like(vv))
        dp = torch.einsum('bihd,bjhd->bhij', dout.double(), vv)
        ds = (p * (dp - (p * dp).sum(-1, keepdim=True))).abs()
        terms = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True))
        e = (u * ds + 2e-5 * terms) ** 2 / D
        if which == 'q':
            var = torch.einsum('bhij,bjhd->bihd', e, kk ** 2)
        else:
            var = torch.einsum('bhij,bihd->bjhd', e, host['q'].double() ** 2)
            var = var.reshape(var.shape[0], var.shape[1], case['Hkv'], G, D).sum(3)
        bound = 2 * var.sqrt() + (u * w.abs()).clamp(min=2.0 ** -25 if dt == torch.float16 else 2.0 ** -134)
        rms = float((((g.double().cpu() - w) / bound) ** 2).mean().sqrt())
    assert rms < 1, rms


@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('c', [dict(B=260, Nq=20, Nk=33, Hkv=2), dict(B=260, Nq=33, Nk=20, Hkv=2, causal=True), dict(B=1025, Nq=9, Nk=17, Hkv=2, causal=True, start=8)],
                         ids=attn_id)
def test_heads_that_share_keys_in_one_workgroup(c, D):
    """So many sequences that dk and dv of a group of heads are summed by the workgroup that owns the keys; with fewer they meet in memory."""
    test_attention_and_its_gradients(dict(c, H=4, D=D), torch.float16 if D == 64 else torch.bfloat16)


@pytest.mark.parametrize('dt', HALF, ids=ids)
@pytest.mark.parametrize('case', FROZEN, ids=attn_id)
def test_gradient_of_v_with_and_without_the_tables(case, dt):
    """Another forward kernel and log-sum, the same dv within the rounding of p and of the result; and equal bits alone and with the others."""
    host, at, see, kw = attn_case(case, dt)
    u, G = step(dt), case['H'] // case['Hkv']
    ref = {n: t.double().requires_grad_(n == 'v') for n, t in host.items()}
    want, p = attention64(ref['q'], ref['k'], ref['v'], ref['table'], at, see, case['D'] ** -0.5)
    dout = rnd(*host['q'].shape, seed=5).to(dt)
    w, = torch.autograd.grad(want, ref['v'], dout.double())
    sums = torch.einsum('bhij,bihd->bjhd', p.detach(), dout.double().abs())
    sums = sums.reshape(sums.shape[0], sums.shape[1], case['Hkv'], G, case['D']).sum(3)
    tiny = 0.0 if dt == torch.bfloat16 else 2.0 ** -25
    got = {}
    for wanted in ('v', 'v table', 'q k v', 'q k v table'):
        leaf = {n: t.to(DEV).requires_grad_(n in wanted.split()) for n, t in host.items()}
        out = ops.biased_attention(leaf['q'], leaf['k'], leaf['v'], leaf['table'], **kw)
        got[wanted], = torch.autograd.grad(out, leaf['v'], dout.to(DEV))
        close(got[wanted], w, u * 1.01 * w.abs() + (u + 2e-5) * sums + tiny, wanted)
    assert torch.equal(got['v'], got['q k v']) and torch.equal(got['v table'], got['q k v table'])


UNUSED = [
    dict(B=1, Nq=200, Nk=200, H=2, Hkv=1, D=64, causal=True, bidirectional=True, buckets=16, far=20),
    dict(B=2, Nq=33, Nk=64, H=2, Hkv=2, D=32, far=200),
    dict(B=2, Nq=33, Nk=64, H=2, Hkv=2, D=128, far=200),
    dict(B=2, Nq=5, Nk=64, H=2, Hkv=2, D=64, causal=True, bidirectional=True, start=30),
    dict(B=1, Nq=130, Nk=300, H=2, Hkv=2, D=64, causal=True, start=-20, far=200),
    dict(B=2, Nq=150, Nk=400, H=2, Hkv=2, D=64, lens=[90, 0], buckets=64, far=300),
]


@pytest.mark.parametrize('dt', HALF, ids=ids)
@pytest.mark.parametrize('fill', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('case', UNUSED, ids=attn_id)
def test_table_entries_that_no_pair_uses(case, fill, dt):
    """Distances that no query sees (keys after it of a causal call, beyond the lengths, of rows that do not exist) may hold anything."""
    host, at, see, kw = attn_case(case, dt)
    used = torch.zeros(host['table'].shape[0], dtype=torch.bool)
    used[at[see.expand_as(at)].unique()] = True
    assert not used.all()
    dout = rnd(*host['q'].shape, seed=5).to(dt).to(DEV)
    results = []
    for f in (0.0, fill):
        table = host['table'].clone()
        table[~used] = f
        leaves = [t.to(DEV).requires_grad_(True) for t in (host['q'], host['k'], host['v'], table)]
        with torch.no_grad():
            plain = ops.biased_attention(*leaves, **kw)
        out = ops.biased_attention(*leaves, **kw)
        results.append([plain, out] + list(torch.autograd.grad(out, leaves, dout)))
    for name, a, b in zip(('inference', 'out', 'dq', 'dk', 'dv', 'dtable'), *results):
        assert torch.equal(a, b), name
    assert not results[1][-1][~used].any()


@pytest.mark.parametrize('C', [40, 203, 1024])
def test_norm_gradients_asked_for_one_at_a_time(C):
    """Each gradient alone equals, bit for bit, the one asked for with all others; gates of channels, samples and tokens."""
    B, N = 3, 37
    host = dict(x=rnd(B, N, C, seed=1), y=rnd(B, N, C, seed=2), post_weight=rnd(C, seed=3), post_bias=rnd(C, seed=4), pre_weight=rnd(C, seed=5),
                pre_bias=rnd(C, seed=6))
    dx, dh = rnd(B, N, C, seed=7).float().to(DEV), rnd(B, N, C, seed=8).float().to(DEV)
    for gate in ((C,), (B, C), (B, N, C)):
        host['gate'] = rnd(*gate, seed=9)

        def grads(wanted):
            leaf = {n: t.float().to(DEV).requires_grad_(n in wanted) for n, t in host.items()}
            out = ops.block_norm(**leaf, branch_scale=0.7, residual_scale=1.1, kind='layer')
            return dict(zip(wanted, torch.autograd.grad(out, [leaf[n] for n in wanted], (dx, dh))))

        every = grads(list(host))
        for n in host:
            assert torch.equal(grads([n])[n], every[n]), (gate, n)


def test_attention_with_the_longest_line_and_the_most_buckets():
    """The largest LDS footprints: width 128, reach 1024, 256 buckets, with the table's gradient; 64 and 128 heads on one key head."""
    for c in (dict(B=1, Nq=130, Nk=2300, H=2, Hkv=2, D=128, buckets=256, far=1024), dict(B=1, Nq=33, Nk=1500, H=2, Hkv=1, D=64, buckets=256, far=1024),
              dict(B=1, Nq=2, Nk=600, H=64, Hkv=1, D=128, buckets=256, far=1024), dict(B=1, Nq=1, Nk=300, H=128, Hkv=1, D=32)):
        test_attention_and_its_gradients(c, torch.bfloat16)


@pytest.mark.parametrize('nq', [1, 70])
def test_attention_reads_any_strides(nq):
    """Heads in front of tokens, slices of a fused projection, a cache shared by the batch (stride 0), rows that have to be copied."""
    B, Nk, H, D = 2, 150, 4, 64
    base = dict(B=B, Nq=nq, Nk=Nk, H=H, Hkv=H, D=D)
    host, at, see, kw = attn_case(base, torch.bfloat16)
    q, k, v, t = (host[n].to(DEV) for n in ('q', 'k', 'v', 'table'))
    want = ops.biased_attention(q, k, v, t)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert not heads_first[1].is_contiguous()
    assert torch.equal(want, ops.biased_attention(*heads_first, t))
    fused = torch.cat([k, v], -1)
    assert torch.equal(want, ops.biased_attention(q, fused[..., :D], fused[..., D:], t))
    odd = torch.empty(B, Nk, H, D + 3, dtype=k.dtype, device=DEV)
    odd[..., 1:D + 1] = k
    assert torch.equal(want, ops.biased_attention(q, odd[..., 1:D + 1], v, t))
    last = k.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)           # innermost stride not 1
    assert torch.equal(want, ops.biased_attention(q, last, v, t))
    one_k, one_v = k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1)
    assert torch.equal(ops.biased_attention(q, one_k.contiguous(), one_v.contiguous(), t), ops.biased_attention(q, one_k, one_v, t))
    # gradients of broadcast keys and of a transposed dout
    leaf = k[:1].clone().requires_grad_(True)
    full = k[:1].expand(B, -1, -1, -1).contiguous().requires_grad_(True)
    dout = rnd(B, H, nq, D, seed=6).to(q.dtype).to(DEV).transpose(1, 2)
    ga, = torch.autograd.grad(ops.biased_attention(q, leaf.expand(B, -1, -1, -1), v, t), leaf, dout)
    gb, = torch.autograd.grad(ops.biased_attention(q, full, v, t), full, dout.contiguous())
    close(ga, gb.double().cpu().sum(0, keepdim=True), step(q.dtype) * gb.double().cpu().sum(0, keepdim=True).abs() * 1.01 + 1e-7, 'broadcast keys')


@pytest.mark.parametrize('nq', [1, 40])
def test_attention_offsets_past_32_bits(nq):
    """Tokens 2^17 elements apart: the last key is 2.6e9 elements (5 GB) behind the first."""
    Nk, D, step_ = 20000, 64, 1 << 17
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip('needs 12 GB of device memory')
    store = torch.empty(Nk * step_, dtype=torch.bfloat16, device=DEV)
    k = store.as_strided((1, Nk, 1, D), (0, step_, D, 1))
    v = store.as_strided((1, Nk, 1, D), (0, step_, D, 1), D)
    k.copy_(rnd(1, Nk, 1, D, seed=1))
    v.copy_(rnd(1, Nk, 1, D, seed=2))
    q, t = rnd(1, nq, 2, D, seed=3).bfloat16().to(DEV), rnd(32, 2, seed=4).float().to(DEV)
    kc, vc = k.contiguous(), v.contiguous()
    assert torch.equal(ops.biased_attention(q, k, v, t, q_start=Nk - nq, causal=True), ops.biased_attention(q, kc, vc, t, q_start=Nk - nq, causal=True))
    dout = rnd(1, nq, 2, D, seed=5).bfloat16().to(DEV)
    grads = []
    for kk, vv in ((k, v), (kc, vc)):
        leaves = [x.detach().requires_grad_(True) for x in (q, kk, vv, t)]
        grads.append(torch.autograd.grad(ops.biased_attention(*leaves, q_start=Nk - nq, causal=True), leaves, dout))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_empty_rows_ignore_their_gradient():
    c = dict(B=3, Nq=65, Nk=130, H=2, Hkv=2, D=64, lens=[0, 1, 130], causal=True, start=[0, -30, -40])
    host, at, see, kw = attn_case(c, torch.bfloat16)
    dout = rnd(*host['q'].shape, seed=5).bfloat16()
    empty = ~see.any(2)
    assert empty.any() and not empty.all()
    grads = []
    for fill in (0.0, float('nan'), float('inf')):
        leaves = [host[n].to(DEV).requires_grad_(True) for n in ('q', 'k', 'v', 'table')]
        d = dout.clone()
        d[empty] = fill
        out = ops.biased_attention(*leaves, **kw)
        assert not out[empty.to(DEV)].any()
        grads.append(torch.autograd.grad(out, leaves, d.to(DEV)))
    for g in grads[1:]:
        assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(g, grads[0]))
    assert not grads[0][0][empty.to(DEV)].any()


@pytest.mark.parametrize('dt', HALF, ids=ids)
@pytest.mark.parametrize('D', [32, 64, 128])
def test_empty_rows_ignore_their_query(D, dt):
    """Rows in front of the first key of a causal call see nothing, whatever their q and dout hold, also beside rows that do."""
    B, Nq, Nk, H, dead = 1, 200, 150, 2, 41
    host = [rnd(B, n, H, D, seed=i).to(dt) for i, n in enumerate((Nq, Nk, Nk, Nq))]
    table = rnd(32, H, seed=4).float().to(DEV)
    results = []
    for fill in (0.0, float('nan'), float('inf')):
        q, k, v, dout = (t.clone() for t in host)
        q[:, :dead] = fill
        dout[:, :dead] = fill
        leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)] + [table.clone().requires_grad_(True)]
        out = ops.biased_attention(*leaves, causal=True, q_start=-dead)
        assert not out[:, :dead].any()
        results.append([out] + list(torch.autograd.grad(out, leaves, dout.to(DEV))))
    for r in results[1:]:
        assert not r[1][:, :dead].any()
        assert all(torch.isfinite(t).all() and torch.equal(t, w) for t, w in zip(r, results[0]))


@pytest.mark.parametrize('dt', HALF, ids=ids)
@pytest.mark.parametrize('nq', [5, 600])
@pytest.mark.parametrize('low', [-1e4, -1e9, -1e30, torch.finfo(torch.float32).min, -float('inf')])
def test_distances_masked_by_the_table(low, nq, dt):
    """A very low bias of the last bucket keeps rows to their neighbourhood; padded rows, beyond it, see keys with that bias only: the
    softmax of their scores (zeros for -inf).  Logits are rounded to half of 2^-6 around 2^17: three such roundings, of a logit, of the
    maximum and of a split's or tile's, are 1.7 % of a probability, and as much again of their sum."""
    B, Nk, H, D, far = 2, 700, 2, 64, 64
    starts, lens = [40, 690 - nq], [700, 100]
    q, k, v, dout = (rnd(B, n, H, D, seed=i).to(dt) for i, n in enumerate((nq, Nk, Nk, nq)))
    table = rnd(32, H, seed=4).float()
    table[15] = table[31] = low
    at = torch.stack([bucket_matrix(32, far, True, nq, Nk, s) for s in starts])
    see = torch.stack([(torch.arange(Nk) < n)[None].expand(nq, Nk) for n in lens])
    lonely = (see & ~((at == 15) | (at == 31))).sum(-1) == 0
    assert lonely.any() and not lonely.all()
    kw = dict(max_distance=far, k_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), q_start=torch.tensor(starts, dtype=torch.int32, device=DEV))
    limit = 2.0 ** 17 / math.log2(math.e)
    if low == -float('inf'):
        see, clamped = see & ~lonely[:, :, None], table.double()
    else:
        clamped = table.double().clamp(min=-limit)
    want, p = attention64(q.double(), k.double(), v.double(), clamped, at, see, D ** -0.5)
    want = torch.where(see.any(-1)[:, :, None, None], want, torch.zeros_like(want))
    spread = torch.einsum('bhij,bjhd->bihd', torch.nan_to_num(p), v.double().abs())
    u = step(dt)
    bound = u * want.abs() * 1.01 + (u + 2e-5) * spread + 1e-7 + torch.where(lonely[:, :, None, None], 0.034 * spread, torch.zeros_like(spread))
    with torch.no_grad():
        out = ops.biased_attention(q.to(DEV), k.to(DEV), v.to(DEV), table.to(DEV), **kw)
    close(out, want, bound, 'out')
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v, table)]
    out = ops.biased_attention(*leaves, **kw)
    close(out, want, bound, 'training out')
    # gradients: those of the limit itself, and rows beyond the length with a dout of zeros add nothing
    quiet = torch.where(lonely[:, :, None, None], torch.zeros_like(dout), dout)
    if low != -float('inf'):
        other = [t.to(DEV).requires_grad_(True) for t in (q, k, v, table.clamp(min=-90852.5))]
        out_ = ops.biased_attention(*other, **kw)
        assert torch.equal(out, out_) or low > -90852
    for g in (quiet, dout):
        grads = torch.autograd.grad(out, leaves, g.to(DEV), retain_graph=True)
        assert all(torch.isfinite(t).all() for t in grads)
        if low < -90852 and low != -float('inf'):
            assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(out_, other, g.to(DEV), retain_graph=True)))
        if g is quiet:
            assert not grads[0].cpu()[lonely].any()


@pytest.mark.parametrize('dt', HALF, ids=ids)
def test_one_token_at_a_time_equals_the_whole_sequence(dt):
    """A cache that grows by a token a call, against the causal call over all tokens: the same sums in other orders, each rounded as its
    own call rounds (probabilities and results: 2 u each side)."""
    N, H, Hkv, D = 300, 4, 2, 64
    q, k, v, t = rnd(2, N, H, D, seed=1).to(dt), rnd(2, N, Hkv, D, seed=2).to(dt), rnd(2, N, Hkv, D, seed=3).to(dt), rnd(32, H, seed=4).float()
    q, k, v, t = (x.to(DEV) for x in (q, k, v, t))
    whole = ops.biased_attention(q, k, v, t, causal=True).double().cpu()
    cache_k, cache_v = torch.full_like(k, float('nan')), torch.full_like(v, float('nan'))
    at, see = bucket_matrix(32, 128, False, N, N, 0)[None], (torch.arange(N)[None] <= torch.arange(N)[:, None])[None]
    p = attention64(q.double().cpu(), k.double().cpu(), v.double().cpu(), t.double().cpu(), at.expand(2, -1, -1), see.expand(2, -1, -1), D ** -0.5)[1]
    spread = torch.einsum('bhij,bjhd->bihd', p, v.double().cpu().abs().repeat_interleave(H // Hkv, 2))
    for i in range(N):
        cache_k[:, i], cache_v[:, i] = k[:, i], v[:, i]
        lens = torch.full((2,), i + 1, dtype=torch.int32, device=DEV)
        one = ops.biased_attention(q[:, i:i + 1], cache_k, cache_v, t, causal=True, k_lens=lens, q_start=lens - 1)
        u = step(dt)
        close(one[:, 0], whole[:, i], 2 * (u * whole[:, i].abs() * 1.01 + (u + 2e-5) * spread[:, i] + 1e-7), str(i))


# --------------------------------------------------------------------------------------------- together
def _block(p, x, h, table, **kw):
    """Attention block over tokens, as the operators are used together: h -> q, k, v -> attention -> projection -> norms."""
    B, N, Cc = h.shape
    H, D = table.shape[1], p['wq'].shape[1] // table.shape[1]
    q, k, v = ((h @ p[n]).view(B, N, -1, D) for n in ('wq', 'wk', 'wv'))
    y = ops.biased_attention(q, k, v, table, **kw).reshape(B, N, H * D) @ p['wo']
    return ops.block_norm(x, y, post_weight=p['post'], gate=p['gate'], pre_weight=p['pre'], residual_scale=0.9)


def test_two_blocks_together_against_64_bits():
    """bias -> attention -> norms, twice, on a 32-bit residual stream: outputs and every gradient against the same program in 64 bits.
    bf16 steps in the chain (h, q, k, v, attention, projection, twice; and their gradients): about 12 roundings of u = 2^-8 that add up as
    independent errors, sqrt(12) u = 1.4 % of a result's size, four times that asked of the relative 2-norm."""
    B, N, Cc, H, Hkv, D = 2, 150, 128, 4, 2, 32
    dt = torch.bfloat16
    names = dict(wq=(Cc, H * D), wk=(Cc, Hkv * D), wv=(Cc, Hkv * D), wo=(H * D, Cc))
    host = [dict({n: (rnd(*s, seed=10 * l + i) * s[0] ** -0.5).to(dt) for i, (n, s) in enumerate(names.items())},
                 post=1 + rnd(Cc, seed=10 * l + 5, std=0.1).float(), pre=1 + rnd(Cc, seed=10 * l + 6, std=0.1).float(),
                 gate=0.5 + rnd(B, Cc, seed=10 * l + 7, std=0.2).float()) for l in range(2)]
    tables = [rnd(32, H, seed=30 + l).float() for l in range(2)]
    x0, w0 = rnd(B, N, Cc, seed=40).float(), 1 + rnd(Cc, seed=41, std=0.1).float()
    lens = [N, 101]
    target = rnd(B, N, Cc, seed=42)
    dev = [{n: t.to(DEV).requires_grad_(True) for n, t in p.items()} for p in host]
    dtab = [t.to(DEV).requires_grad_(True) for t in tables]
    x, w = x0.to(DEV).requires_grad_(True), w0.to(DEV).requires_grad_(True)
    h = ops.block_norm(x, None, pre_weight=w)[1].to(dt)
    cur = x
    for p, t in zip(dev, dtab):
        cur, h = _block(p, cur, h, t, causal=True, k_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    ((cur * target.float().to(DEV)).sum() + (h.float() * target.float().to(DEV)).sum()).backward()

    ref = [{n: t.double().requires_grad_(True) for n, t in p.items()} for p in host]
    rtab = [t.double().requires_grad_(True) for t in tables]
    rx, rw = x0.double().requires_grad_(True), w0.double().requires_grad_(True)
    at = bucket_matrix(32, 128, False, N, N, 0)[None].expand(B, -1, -1)
    i, j = torch.arange(N)[:, None], torch.arange(N)[None]
    see = torch.stack([(j <= i) & (j < n) for n in lens])
    rh = norm64(rx, None, None, None, None, 1, 1.0, 1.0, rw, None, False, 1e-6)[1]
    rcur = rx
    for p, t in zip(ref, rtab):
        q, k, v = ((rh @ p[n]).view(B, N, -1, D) for n in ('wq', 'wk', 'wv'))
        y = attention64(q, k, v, t, at, see, D ** -0.5)[0].reshape(B, N, H * D) @ p['wo']
        rcur, rh = norm64(rcur, y, p['post'], None, p['gate'], N, 1.0, 0.9, p['pre'], None, False, 1e-6)
    ((rcur * target).sum() + (rh * target).sum()).backward()

    bound = 4 * math.sqrt(12) * 2.0 ** -8
    pairs = [('x', cur, rcur), ('h', h, rh), ('dx', x.grad, rx.grad), ('dw0', w.grad, rw.grad)]
    pairs += [('dtable%d' % l, dtab[l].grad, rtab[l].grad) for l in range(2)]
    pairs += [('d%s%d' % (n, l), dev[l][n].grad, ref[l][n].grad) for l in range(2) for n in host[l]]
    for name, g, r in pairs:
        r = r.detach()
        err = float((g.detach().double().cpu() - r).norm() / r.norm())
        assert err < bound, '%s: %.4f' % (name, err)


def test_norm_gradient_against_differences():
    """fp32, along random directions, on the GPU itself: central differences of step 1e-2 (error of third order, about 1e-4 of the value,
    and rounding 2^-24 x |loss| / 1e-2, about 1e-4)."""
    shape, Cc = (3, 7, 96), 96
    t = [rnd(*shape, seed=1), rnd(*shape, seed=2), 1 + rnd(Cc, seed=3, std=0.1), rnd(Cc, seed=4), 0.5 + rnd(3, Cc, seed=5, std=0.2), 1 + rnd(Cc, seed=6, std=0.1), rnd(Cc, seed=7)]
    t = [x.float().to(DEV).requires_grad_(True) for x in t]
    wa, wb = rnd(*shape, seed=8).to(DEV), rnd(*shape, seed=9).to(DEV)

    def loss(t):
        xo, h = ops.block_norm(t[0], t[1], t[2], t[3], t[4], 0.8, 1.1, t[5], t[6], 'layer')
        return (xo.double() * wa).sum() + (h.double() * wb).sum()

    grads = torch.autograd.grad(loss(t), t)
    for n, g in enumerate(grads):
        d = rnd(*t[n].shape, seed=20 + n).float().to(DEV)
        with torch.no_grad():
            e = 1e-2
            up, down = (loss([x + s * e * d if i == n else x for i, x in enumerate(t)]) for s in (1, -1))
        want, got = float((up - down) / (2 * e)), float((g.double() * d.double()).sum())
        size = float((g.double() * d.double()).abs().sum())
        assert abs(want - got) < 2e-3 * size + 1e-3, (n, want, got)


def test_bias_and_attention_agree_on_the_buckets():
    """The matrix of relative_position_bias added to plain logits gives what biased_attention gives."""
    B, N, H, D = 1, 200, 2, 64
    q, k, v, t = rnd(B, N, H, D, seed=1).half().to(DEV), rnd(B, N, H, D, seed=2).half().to(DEV), rnd(B, N, H, D, seed=3).half().to(DEV), rnd(32, H, seed=4).float().to(DEV)
    bias = ops.relative_position_bias(t, N, N).double().cpu()
    x = D ** -0.5 * torch.einsum('bihd,bjhd->bhij', q.double().cpu(), k.double().cpu()) + bias
    p = torch.softmax(x, -1)
    want = torch.einsum('bhij,bjhd->bihd', p, v.double().cpu())
    spread = torch.einsum('bhij,bjhd->bihd', p, v.double().cpu().abs())
    u = step(torch.float16)
    close(ops.biased_attention(q, k, v, t), want, u * want.abs() * 1.01 + (u + 2e-5) * spread + 1e-7)


# --------------------------------------------------------------------------------------------- streams, graphs, refusals
def test_on_another_stream():
    host, at, see, kw = attn_case(dict(B=2, Nq=1, Nk=3000, H=8, Hkv=2, D=64), torch.bfloat16)
    dev = [host[n].to(DEV) for n in ('q', 'k', 'v', 'table')]
    x, w = rnd(64, 512, seed=1).bfloat16().to(DEV), torch.ones(512, device=DEV)
    want = (ops.biased_attention(*dev, **kw), ops.block_norm(x, x, post_weight=w, pre_weight=w)[1], ops.relative_position_bias(dev[3], 100, 100))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (ops.biased_attention(*dev, **kw), ops.block_norm(x, x, post_weight=w, pre_weight=w)[1], ops.relative_position_bias(dev[3], 100, 100))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_captured_calls_replay_on_new_inputs():
    """Forward and gradients of all three in a graph, and a split single-token call in another one, replayed with eager work between."""
    shape = dict(B=2, Nq=96, Nk=96, H=4, Hkv=2, D=64)
    few = dict(B=2, Nq=1, Nk=4000, H=4, Hkv=2, D=64)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
        return dict(q=r(2, 96, 4, 64).bfloat16(), k=r(2, 96, 2, 64).bfloat16(), v=r(2, 96, 2, 64).bfloat16(), t=r(32, 4), x=r(2, 96, 256).float(),
                    w1=1 + 0.1 * r(256), w2=1 + 0.1 * r(256), gate=r(2, 256), do=r(2, 96, 256).float(), dh=r(2, 96, 256).bfloat16(), db=r(4, 50, 60).float(),
                    fq=r(2, 1, 4, 64).bfloat16(), fk=r(2, 4000, 2, 64).bfloat16(), fv=r(2, 4000, 2, 64).bfloat16())

    def train(s):
        leaves = [s[n].detach().requires_grad_(True) for n in ('q', 'k', 'v', 't', 'x', 'w1', 'w2', 'gate')]
        q, k, v, t, x, w1, w2, gate = leaves
        y = ops.biased_attention(q, k, v, t, causal=True).reshape(2, 96, 256)
        xo, h = ops.block_norm(x, y, post_weight=w1, gate=gate, pre_weight=w2)
        b = ops.relative_position_bias(t, 50, 60)
        return (xo.detach(), h.detach(), b.detach()) + torch.autograd.grad([xo, h, b], leaves, [s['do'], s['dh'], s['db']])

    def token(s):
        with torch.no_grad():
            return (ops.biased_attention(s['fq'], s['fk'], s['fv'], s['t'], causal=True, q_start=3999),)

    static = {n: t.to(DEV) for n, t in inputs(0).items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train(static)
            token(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for f in (train, token):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f(static)
        graphs.append((g, out, f))
    for seed in (1, 2, 3):
        for n, t in inputs(seed).items():
            static[n].copy_(t)
        for g, out, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out, f in graphs:
            want = f(static)                                   # eager, between the replays
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        torch.cuda.synchronize()


def test_captured_backward_beside_an_eager_graph_is_refused():
    """... before torch joins the capture to the default stream; the capture itself stays whole, and one without the eager graph goes on."""
    x, y, w = rnd(5, 64, seed=1).float().to(DEV), rnd(5, 64, seed=2).float().to(DEV), torch.ones(64, device=DEV, requires_grad=True)
    d = torch.ones_like(x)
    eager = ops.block_norm(x, y, post_weight=w)[0]
    refused, ok = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(refused):
        out = ops.block_norm(x, y, post_weight=w)[0]
        with pytest.raises(RuntimeError, match='eager graph of the default stream'):
            torch.autograd.grad(out, w, d)
    refused.replay()
    assert torch.equal(out, eager)
    want, = torch.autograd.grad(eager, w, d)
    del eager, out
    with torch.cuda.graph(ok):
        got, = torch.autograd.grad(ops.block_norm(x, y, post_weight=w)[0], w, d)
    for n in (1, 2):
        y.mul_(2 * n)
        ok.replay()
        torch.cuda.synchronize()
        eager = ops.block_norm(x, y, post_weight=w)[0]
        assert torch.equal(got, torch.autograd.grad(eager, w, d)[0])
    assert not torch.equal(got, want)


def test_refusals():
    z = lambda *s, **k: torch.zeros(s, device=DEV, **k)  # noqa: E731
    b16 = dict(dtype=torch.bfloat16)
    q, k, t = z(2, 4, 4, 64, **b16), z(2, 6, 2, 64, **b16), z(32, 4)
    bad = [(TypeError, dict(q=q.float())), (TypeError, dict(k=k.half())), (ValueError, dict(k=z(2, 6, 3, 64, **b16))), (ValueError, dict(k=z(3, 6, 2, 64, **b16))),
           (ValueError, dict(k=z(2, 6, 2, 32, **b16))), (ValueError, dict(k=k[0])), (ValueError, dict(t=z(32, 2))), (ValueError, dict(t=z(32, 4, **b16))),
           (ValueError, dict(t=z(31, 4))), (ValueError, dict(scale=0.0)), (ValueError, dict(scale=float('nan'))), (ValueError, dict(max_distance=2000)),
           (ValueError, dict(k_lens=z(2, dtype=torch.int64))), (ValueError, dict(k_lens=z(3, dtype=torch.int32))), (ValueError, dict(q_start=z(1, dtype=torch.int32))),
           (ValueError, dict(key_mask=z(2, 6))), (ValueError, dict(key_mask=z(2, 5, dtype=torch.bool))), (ValueError, dict(q_start=1 << 30)),
           (RuntimeError, dict(k=k.cpu())), (RuntimeError, dict(k_lens=torch.zeros(2, dtype=torch.int32))), (TypeError, dict(q=None))]
    for err, kw in bad:
        a = dict(q=q, k=k, t=t)
        a.update({n: kw.pop(n) for n in list(kw) if n in a})
        with pytest.raises(err):
            ops.biased_attention(a['q'], a['k'], a['k'], a['t'], **kw)
    for D in (4, 60, 136):
        with pytest.raises(ValueError):
            ops.biased_attention(z(1, 2, 2, D, **b16), z(1, 2, 2, D, **b16), z(1, 2, 2, D, **b16), z(32, 2))
    with pytest.raises(ValueError):
        ops.relative_position_bias(t, -1, 4)
    with pytest.raises(TypeError):
        ops.relative_position_bias(t, 4, 4, dtype=torch.float64)
    x, w = z(2, 3, 64), torch.ones(64, device=DEV)
    for err, a, kw in [(ValueError, (x, x), dict(kind='batch')), (TypeError, (x.double(), x), {}), (TypeError, (x.bfloat16(), x), {}), (TypeError, (x.bfloat16(), x.half()), {}),
                       (ValueError, (x, x[:1]), {}), (ValueError, (x, x), dict(post_weight=w[:32])), (TypeError, (x, x), dict(gate=w.half())),
                       (ValueError, (x, x), dict(post_weight=w.half())), (ValueError, (x, x), dict(post_bias=w)), (ValueError, (x, x), dict(pre_weight=w, pre_bias=w)),
                       (ValueError, (x, x), dict(gate=z(3, 64))), (ValueError, (x, x), dict(gate=z(2, 3, 1))), (ValueError, (x, None), {}),
                       (ValueError, (x, None), dict(pre_weight=w, gate=w)), (ValueError, (x, None), dict(pre_weight=w, residual_scale=0.5)),
                       (ValueError, (z(2, 8200), z(2, 8200)), {}), (ValueError, (z(2, 0), z(2, 0)), {}), (TypeError, (None, x), {})]:
        with pytest.raises(err):
            ops.block_norm(*a, **kw)


def test_second_derivatives_are_refused():
    x, w = rnd(4, 64, seed=1).float().to(DEV).requires_grad_(True), torch.ones(64, device=DEV)
    xo, h = ops.block_norm(x, x, pre_weight=w)
    g, = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_derivatives_are_refused(grad):
    q, t = rnd(1, 4, 2, 64, seed=1).bfloat16().to(DEV), rnd(32, 2, seed=2).float().to(DEV)
    x, w = rnd(4, 64, seed=3).float().to(DEV), torch.ones(64, device=DEV)
    calls = [(ops.biased_attention, [q, q, q, t]), (ops.relative_position_bias, [t, 4, 4]), (ops.block_norm, [x, x, w, None, w, 1.0, 1.0, w])]
    for f, args in calls:
        with torch.set_grad_enabled(grad), fwd.dual_level():
            for i, a in enumerate(args):
                if isinstance(a, torch.Tensor):
                    with pytest.raises(NotImplementedError):
                        f(*args[:i], fwd.make_dual(a, torch.ones_like(a)), *args[i + 1:])
            inside = f(*args)
        with torch.no_grad():
            outside = f(*args)
        first = lambda r: r[0] if isinstance(r, tuple) else r  # noqa: E731
        assert torch.equal(first(inside), first(outside))


def test_norm_of_no_tokens():
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    xo, h = ops.block_norm(x, torch.zeros(0, 64, device=DEV), post_weight=w, pre_weight=w.detach())
    assert xo.shape == h.shape == (0, 64)
    gx, gw = torch.autograd.grad([xo, h], [x, w], [torch.zeros_like(xo), torch.zeros_like(h)])
    assert gx.shape == (0, 64) and not gw.any()
