"""Token operators without a GPU: the buckets' definition, the plain implementations that the GPU tests compare with (their gradients
against differences), and what the C entry points refuse before any launch."""
import ctypes as C
import os
import subprocess
import sys
from fractions import Fraction

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tcvom_amd import _lib as L
from tcvom_amd import ops, token_ops
from test_gpu_token_ops import attention64, bucket_matrix, norm64, rnd


# --------------------------------------------------------------------------------------------- buckets
@pytest.mark.parametrize('n,far,bidir', [(32, 128, True), (32, 128, False), (8, 16, True), (64, 400, False), (128, 1000, True), (4, 3, True),
                                         (2, 2, False), (256, 1024, False), (256, 1024, True), (16, 5, True), (32, 17, False), (32, 1024, True)])
def test_bucket_borders_are_exact(n, far, bidir):
    b = token_ops.rel_buckets(n, far, bidir)
    side = n // 2 if bidir else n
    exact = side // 2
    m = side - exact
    assert (b.num_buckets, b.bidirectional, b.exact, b.n_starts) == (n, int(bidir), exact, m)
    starts = list(b.starts[:m])
    assert starts[0] == exact and starts == sorted(starts) and starts[-1] <= far
    for k, s in enumerate(starts):                       # (d / exact)^m >= (far / exact)^k holds at s and not at s - 1
        def over(d):
            return Fraction(d, exact) ** m >= Fraction(far, exact) ** k
        assert over(s) and (s == exact or not over(s - 1))


def test_buckets_of_near_and_far_positions():
    at = bucket_matrix(32, 128, True, 1, 601, 300)[0]                # relative positions -300 .. 300
    rel = {r: int(at[r + 300]) for r in range(-300, 301)}
    assert [rel[-d] for d in range(9)] == list(range(9)) and [rel[d] for d in range(1, 9)] == list(range(17, 25))
    assert rel[-16] == 10 and rel[-15] == 9 and rel[-32] == 12 and rel[-31] == 11 and rel[-64] == 14          # 8 (2, 4, 8) are borders
    assert rel[-300] == rel[-128] == 15 and rel[300] == rel[128] == 31
    one = bucket_matrix(32, 128, False, 1, 601, 300)[0]
    assert all(int(one[r + 300]) == 0 for r in range(0, 301)) and int(one[300 - 15]) == 15 and int(one[0]) == 31


@pytest.mark.parametrize('n,far,bidir', [(1, 128, False), (3, 128, True), (2, 128, True), (258, 128, True), (32, 8, True), (32, 1025, True),
                                         (32, 0, False), (0, 128, False)])
def test_bucket_refusals(n, far, bidir):
    with pytest.raises(ValueError):
        token_ops.rel_buckets(n, far, bidir)


# --------------------------------------------------------------------------------------------- the plain implementations
def test_plain_attention_gradient_against_differences():
    at = torch.stack([bucket_matrix(8, 6, True, 5, 7, s) for s in (0, 2)])
    see = torch.ones(2, 5, 7, dtype=torch.bool)
    see[0, :, 4:] = False
    see[1, 3] = False                                                     # an empty row
    see[1, 0, ::2] = False
    args = [rnd(2, 5, 4, 8, seed=1), rnd(2, 7, 2, 8, seed=2), rnd(2, 7, 2, 8, seed=3), rnd(8, 4, seed=4)]
    for a in args:
        a.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda q, k, v, t: attention64(q, k, v, t, at, see, 0.3)[0], args, atol=1e-7)


@pytest.mark.parametrize('layer', [False, True])
def test_plain_norm_gradient_against_differences(layer):
    args = [rnd(2, 3, 5, seed=1), rnd(2, 3, 5, seed=2), 1 + rnd(5, seed=3, std=0.1), rnd(5, seed=4), rnd(2, 5, seed=5), 1 + rnd(5, seed=6, std=0.1), rnd(5, seed=7)]
    for a in args:
        a.requires_grad_(True)

    def f(x, y, w1, b1, g, w2, b2):
        return norm64(x, y, w1, b1 if layer else None, g, 3, 0.7, 1.3, w2, b2 if layer else None, layer, 1e-6)

    assert torch.autograd.gradcheck(f, args if layer else [a for a in args], atol=1e-7)


# --------------------------------------------------------------------------------------------- refusals
ANY = 4096                                                                # a "pointer" that nothing may follow


def refused(name, *args):
    with pytest.raises(L.TcvomError) as e:
        L.call(name, *args)
    assert name[6:] in str(e.value), str(e.value)


def test_structures_match_the_header():
    assert C.sizeof(L.RelBuckets) == 4 * (4 + L.MAX_BUCKET_STARTS)
    assert C.sizeof(L.AttnDesc) == 664                                    # static_assert in csrc/attn.hip


def desc(**kw):
    d = L.AttnDesc(2, 64, 64, 4, 2, 64, 1, 0, 0, 0.125, (64 * 4 * 64, 4 * 64, 64), (64 * 2 * 64, 2 * 64, 64), (64 * 2 * 64, 2 * 64, 64), None,
                   None, None, token_ops.rel_buckets(32, 128, True))
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD = [dict(type=0), dict(type=3), dict(H=3), dict(H=0), dict(Hkv=0), dict(D=60), dict(D=136), dict(D=0), dict(Nq=-1), dict(Nk=-1), dict(Nq=1 << 29),
       dict(B=-1), dict(q_start=1 << 30), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf')),
       dict(q_stride=(8, 4, 8)), dict(k_stride=(8, 8, -8)), dict(v_stride=(8, 1 << 24, 8)),
       dict(buckets=L.RelBuckets(32, 1, 9, 8)), dict(buckets=L.RelBuckets(32, 1, 8, 0)), dict(buckets=L.RelBuckets(300, 0, 150, 150)),
       dict(buckets=L.RelBuckets(33, 1, 8, 8)), dict(B=1 << 20, Nq=1 << 12)]


@pytest.mark.parametrize('bad', BAD, ids=lambda b: '-'.join(b))
def test_attention_refusals(bad):
    d = C.byref(desc(**bad))
    refused('tcvom_attn_fwd', d, ANY, ANY, ANY, ANY, ANY, None, None, None, 0, None)
    refused('tcvom_attn_bwd', d, ANY, ANY, ANY, ANY, ANY, ANY, ANY, ANY, (C.c_int64 * 3)(8, 8, 8), ANY, ANY, ANY, ANY, ANY, 1 << 40, None)


def test_attention_refuses_missing_and_misplaced_tensors():
    d = C.byref(desc())
    refused('tcvom_attn_fwd', None, ANY, ANY, ANY, ANY, ANY, None, None, None, 0, None)
    for i in (1, 2, 3, 4, 5):
        args = [d, ANY, ANY, ANY, ANY, ANY, None, None, None, 0, None]
        refused('tcvom_attn_fwd', *(args[:i] + [None] + args[i + 1:]))
    refused('tcvom_attn_fwd', d, ANY + 8, ANY, ANY, ANY, ANY, None, None, None, 0, None)
    few = C.byref(desc(Nq=1, Nk=8192, B=1))
    need = L.call('tcvom_attn_fwd_work', few)
    assert need > 0
    refused('tcvom_attn_fwd', few, ANY, ANY, ANY, ANY, ANY, None, None, ANY, need - 1, None)
    refused('tcvom_attn_fwd', few, ANY, ANY, ANY, ANY, ANY, None, None, None, need, None)
    strides = (C.c_int64 * 3)(8, 8, 8)
    need = L.call('tcvom_attn_bwd_work', d)
    good = [d] + [ANY] * 8 + [strides] + [ANY] * 5
    for i in (1, 2, 3, 4, 5, 7, 8, 9, 10, 11, 12, 14):
        refused('tcvom_attn_bwd', *(good[:i] + [None] + good[i + 1:] + [need, None]))
    refused('tcvom_attn_bwd', *(good + [need - 1, None]))
    refused('tcvom_attn_bwd', *(good[:9] + [(C.c_int64 * 3)(8, 4, 8)] + good[10:] + [need, None]))
    # nothing to do is no error, whatever the pointers
    for e in (dict(B=0), dict(Nq=0)):
        assert L.call('tcvom_attn_fwd', C.byref(desc(**e)), None, None, None, None, None, None, None, None, 0, None) == 0


def test_bias_refusals():
    b = token_ops.rel_buckets(32, 128, True)
    refused('tcvom_relbias_fwd', None, ANY, C.byref(b), 2, 4, 4, 0, 0, None)
    refused('tcvom_relbias_fwd', ANY, None, C.byref(b), 2, 4, 4, 0, 0, None)
    refused('tcvom_relbias_fwd', ANY, ANY, None, 2, 4, 4, 0, 0, None)
    refused('tcvom_relbias_fwd', ANY, ANY, C.byref(b), 0, 4, 4, 0, 0, None)
    refused('tcvom_relbias_fwd', ANY, ANY, C.byref(b), 2, -4, 4, 0, 0, None)
    refused('tcvom_relbias_fwd', ANY, ANY, C.byref(b), 2, 4, 4, 0, 3, None)
    refused('tcvom_relbias_fwd', ANY, ANY, C.byref(b), 2, 4, 4, 1 << 50, 0, None)
    need = L.call('tcvom_relbias_bwd_work', C.byref(b), 2, 400)
    refused('tcvom_relbias_bwd', ANY, ANY, ANY, need - 1, C.byref(b), 2, 400, 4, 0, 0, None)
    refused('tcvom_relbias_bwd', ANY, ANY, None, need, C.byref(b), 2, 400, 4, 0, 0, None)
    refused('tcvom_relbias_bwd', ANY, ANY, ANY, need, C.byref(b), 2, 400, 0, 0, 0, None)


def test_norm_refusals():
    def fwd(x=ANY, y=ANY, w1=ANY, b1=None, gate=None, gate_rows=1, w2=ANY, b2=None, layer=0, xo=ANY, h=ANY, T=8, Cc=64, xt=1, yt=1):
        refused('tcvom_block_norm_fwd', x, y, w1, b1, gate, 0, gate_rows, w2, b2, 1.0, 1.0, 1e-6, layer, xo, h, None, T, Cc, xt, yt, None)

    for kw in (dict(x=None), dict(xo=None), dict(h=None), dict(b1=ANY), dict(b2=ANY), dict(gate=ANY, gate_rows=0), dict(gate=ANY, gate_rows=3),
               dict(T=-1), dict(T=1 << 31), dict(Cc=0), dict(Cc=8193), dict(xt=1, yt=2), dict(xt=1, yt=0), dict(xt=3, yt=3),
               dict(y=None, w1=ANY), dict(y=None, w1=None, w2=None), dict(y=None, w1=None, gate=ANY)):
        fwd(**kw)

    def bwd(x=ANY, y=ANY, w1=ANY, b1=None, gate=None, gate_rows=1, w2=ANY, layer=0, stats=ANY, dh=ANY, dx=ANY, dy=ANY, dw1=None, db1=None, dg=None,
            dw2=None, db2=None, work=ANY, n=1 << 40, T=8, Cc=64):
        refused('tcvom_block_norm_bwd', x, y, w1, b1, gate, 0, gate_rows, w2, 1.0, 1.0, layer, stats, ANY, dh, dx, dy, dw1, db1, dg, dw2, db2, work, n,
                T, Cc, 1, 1, None)

    for kw in (dict(x=None), dict(stats=None), dict(dx=None), dict(dy=None), dict(w1=None, dw1=ANY), dict(w2=None, dw2=ANY), dict(dh=None, dw2=ANY),
               dict(dg=ANY), dict(db1=ANY), dict(work=None), dict(n=8), dict(gate=ANY, gate_rows=3), dict(gate=ANY, gate_rows=2, T=2 * 32769),
               dict(Cc=8193)):
        bwd(**kw)


def test_cpu_tensors_are_refused():
    q, t = torch.zeros(1, 4, 2, 8, dtype=torch.bfloat16), torch.zeros(32, 2)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ops.biased_attention(q, q, q, t)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ops.relative_position_bias(t, 4, 4)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ops.block_norm(q, q, pre_weight=torch.ones(8))
    with pytest.raises(TypeError):
        ops.block_norm(None, q)


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_derivatives_are_refused(grad, monkeypatch):
    """A dual tensor needs no gradient and has an address: the call must not pass autograd by, which would drop the tangent."""
    monkeypatch.setattr(token_ops, '_check_cuda', lambda *a: None)
    monkeypatch.setattr(token_ops, '_rel_bias', lambda table, *a: table.detach().clone())
    monkeypatch.setattr(token_ops, '_attention', lambda q, *a: (q.detach().clone(), None, None))
    monkeypatch.setattr(token_ops, '_block_norm', lambda x, *a: (x.detach().clone(), None, None))
    t, q, x = torch.randn(32, 2), torch.randn(1, 4, 2, 8).bfloat16(), torch.randn(3, 8)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        dual = lambda a: fwd.make_dual(a, torch.ones_like(a))  # noqa: E731
        for call in (lambda: ops.relative_position_bias(dual(t), 4, 4), lambda: ops.biased_attention(q, dual(q), q, t),
                     lambda: ops.biased_attention(q, q, q, dual(t)), lambda: ops.block_norm(x, dual(x)), lambda: ops.block_norm(x, x, gate=dual(x))):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(ops.relative_position_bias(t, 4, 4), t)                 # no dual tensor among the arguments
    assert torch.equal(ops.relative_position_bias(t, 4, 4), t)


def test_what_the_gradient_cannot_do_is_refused_by_the_call(monkeypatch):
    """A call whose backward would be refused is refused itself, and only then."""
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda device: 0)
    monkeypatch.setattr(token_ops, '_check_cuda', lambda *a: None)
    monkeypatch.setattr(token_ops, '_rel_bias', lambda table, *a: table.detach())
    monkeypatch.setattr(token_ops, '_attention', lambda q, *a: (q.detach(), None, None))
    t = torch.zeros(32, 2)
    leaf = torch.zeros(32, 2, requires_grad=True)
    limit = L.MAX_RELBIAS_BWD_QUERIES
    ops.relative_position_bias(t, limit + 1, 1)
    ops.relative_position_bias(leaf, limit, 1)
    with pytest.raises(ValueError, match='with a gradient'):
        ops.relative_position_bias(leaf, limit + 1, 1)
    b = token_ops.rel_buckets(32, 128, True)
    for n, why in ((limit, 'workspace'), (limit + 1, 'lengths')):
        with pytest.raises(L.TcvomError, match=why):
            L.call('tcvom_relbias_bwd', ANY, ANY, ANY, 0, C.byref(b), 2, n, 4, 0, 0, None)
    q, rows = torch.zeros(4, 1, 2, 8).bfloat16(), lambda n: torch.zeros(4, 1, 1, 8).bfloat16().expand(4, n, 1, 8)
    many, most = rows(1 << 28), rows((1 << 28) - 128)
    ops.biased_attention(q, many, many, t)
    ops.biased_attention(q, most, most, leaf)
    with pytest.raises(ValueError, match='with gradients'):
        ops.biased_attention(q, many, many, leaf)
    with fwd.dual_level():                                   # (such calls pass through autograd, but nothing asks for a gradient)
        ops.relative_position_bias(t, limit + 1, 1)
        ops.biased_attention(q, many, many, t)
        with torch.no_grad():
            ops.relative_position_bias(leaf, limit + 1, 1)


@pytest.mark.parametrize('kw,why', [(dict(B=1, Nq=1, Nk=1 << 25, H=64, Hkv=1, D=8), 'workspace'), (dict(B=4, Nq=1, Nk=1 << 28, H=2, Hkv=1, D=8), 'keys'),
                                    (dict(B=4, Nq=1, Nk=(1 << 28) - 128, H=2, Hkv=1, D=8), 'workspace'), (dict(B=1, Nq=1, Nk=128 * 2047, H=8192, Hkv=1, D=8), 'workspace')])
def test_long_keys_and_the_gradient(kw, why):
    """The limit counts the workgroups that there are: of key heads (64 heads on one of 2^25 keys are 2^18), apart only where they fit."""
    with pytest.raises(L.TcvomError, match=why):
        L.call('tcvom_attn_bwd', C.byref(desc(**kw)), ANY, ANY, ANY, ANY, ANY, ANY, ANY, ANY, (C.c_int64 * 3)(8, 8, 8), ANY, ANY, ANY, ANY, ANY, 0, None)


def test_captured_backward_beside_an_eager_graph_is_refused(monkeypatch):
    """Refused while a graph of the default stream holds the leaf, and no longer; by all three, for any of their leaves."""
    where = dict(stream=0, capturing=False)
    monkeypatch.setattr(token_ops, '_check_cuda', lambda *a: None)
    monkeypatch.setattr(token_ops, '_launch', lambda *a: None)
    monkeypatch.setattr(token_ops, '_rel_bias', lambda t, *a: t.new_zeros(2, 4, 4))
    monkeypatch.setattr(token_ops, '_attention', lambda q, *a: (q.detach().clone(), q.detach().float(), q.new_zeros(1, 2, 4).float()))
    monkeypatch.setattr(token_ops, '_block_norm', lambda x, *a: (x.detach().clone(), None, x.new_zeros(3, 4)))
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda device: where['stream'])
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: where['capturing'])

    def on(stream, capturing=False):
        where.update(stream=stream, capturing=capturing)

    t, q, x, y = torch.randn(32, 2), torch.randn(1, 4, 2, 8).bfloat16(), torch.randn(3, 8), torch.randn(3, 8)
    calls = [(lambda t: ops.relative_position_bias(t, 4, 4), t), (lambda t: ops.biased_attention(q, q, q, t), t), (lambda k: ops.biased_attention(q, k, q, t), q),
             (lambda y: ops.block_norm(x, y)[0], y), (lambda g: ops.block_norm(x, y, gate=g)[0], y)]
    for call, value in calls:
        leaf = value.clone().requires_grad_(True)

        def captured(source=leaf):
            on(7, True)
            out = call(source)
            return torch.autograd.grad(out, leaf, torch.zeros_like(out))

        on(0)
        eager = call(leaf)
        with pytest.raises(RuntimeError, match='eager graph of the default stream'):
            captured()
        captured(leaf * 1)                                   # not through this operator's own leaf
        on(0)
        torch.autograd.grad(eager, leaf, torch.zeros_like(eager))                  # the eager pass itself
        del eager
        captured()
        on(3)
        eager = call(leaf)                                   # another stream: the capture joins it and leaves it again
        captured()
        on(0)
        with torch.no_grad():
            call(leaf)
        del eager
        captured()


@pytest.mark.parametrize('causal,heads,most', [(0, 4, 447), (1, 8, 512), (1, 3, 2047)])
def test_workspace_of_heads_apart(causal, heads, most):
    """Partial sums of every head only where few workgroups would own the keys."""
    def floats(wgs, H=64):
        B, Hkv, Nk, Nq = heads, 1, 128 * wgs // heads, 128
        rows = B * H * Nq + B * H * 32
        return L.call('tcvom_attn_bwd_work', C.byref(desc(B=B, Hkv=Hkv, H=H, Nk=Nk, Nq=Nq, causal=causal))) - rows, 2 * B * Nk * H * 64

    below, above = most // heads * heads, (most // heads + 1) * heads
    got, partial = floats(below)
    assert got == partial
    assert floats(above)[0] == 0
    assert floats(below, H=1)[0] == 0


@pytest.mark.parametrize('mode', ['no_grad', 'inference_mode'])
def test_first_import_without_gradients(mode):
    code = 'import torch\nwith torch.%s():\n    from tcvom_amd import ops, token_ops\n' % mode
    code += 'x = torch.zeros(2, requires_grad=True)\nassert type((x * 2).grad_fn.next_functions[0][0]) is token_ops._AccumulateGrad'
    subprocess.run([sys.executable, '-c', code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=300)
