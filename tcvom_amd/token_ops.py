"""Operators on token sequences: a learned relative position bias, the attention that adds it inside, the norms around a block.

They stand beside the attention and the norms of `ops` (re-exported there): TAM and GuidedCxtAtten know no positions and work on maps,
BatchNorm / GroupNorm normalise over pixels; a block over tokens -- the frames of a clip, the pixels of a stride-8 or -16 map --
needs these.  The reference has no counterpart.

    h = ops.block_norm(x, None, pre_weight=w0)[1]
    y = attention_projection(ops.biased_attention(q(h), k(h), v(h), table))
    x, h = ops.block_norm(x, y, post_weight=w1, gate=g, pre_weight=w2)        # h enters the next block

Element types are arguments: bf16, fp16 and, for the bias matrix and the norms, fp32, in either build of the library.  16-bit results are
rounded to nearest even without saturation.  Gradients are added in a fixed order: equal calls give equal bits.  First derivatives
only, in reverse mode.  A call may be captured into a graph, its backward too -- while no graph that an eager call on the default
stream made of the same leaves lives: torch would join the capture to that stream and end the process.  Such a backward is refused where the
eager call was one of these operators (a leaf that only other operations hold is not known here).
"""
import ctypes as C
import functools
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_cuda(name, needed, *others):
    """`needed`: a tuple of tensors, `others`: tensors or None; all of one GPU."""
    index = None
    for n, t in enumerate(needed + others):
        if t is None and n >= len(needed):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError('%s: expected a tensor, got %s' % (name, type(t).__name__))
        i = t.get_device()
        if i != index:
            if i < 0:
                raise RuntimeError('tcvom_amd ops run on the GPU through libtcvom_hip.so only (no CPU fallback); %s got a %s tensor'
                                   % (name, t.device))
            if index is not None:
                raise RuntimeError('%s: tensors on cuda:%d and cuda:%d' % (name, index, i))
            index = i


def _c(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _p(t):
    return None if t is None else t.data_ptr()


def _launch(device, name, *args):
    """An entry point of the library on the current stream of the tensors' device, whatever the current device is.  (The stream's
    handle is asked for directly: a call's host time is what its smallest sizes cost.)"""
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch.cuda.current_device() == device:
        return L.call(name, *args, stream)
    with torch.cuda.device(device):
        return L.call(name, *args, stream)


_AccumulateGrad = torch._C._functions.AccumulateGrad
_ON_DEFAULT_STREAM = 'tcvom_amd: leaf of an eager graph on the default stream'


def _mark_leaves(device, out):
    """Marks the nodes that will add the gradients of the leaves of `out`, made by a call on the default stream.  Such a node belongs to the
    stream of its first use and is shared by every graph of its leaf; it, and the mark, go with the last of them."""
    if out.grad_fn is not None and torch._C._cuda_getCurrentRawStream(device) == 0:
        for node, _ in out.grad_fn.next_functions:
            if type(node) is _AccumulateGrad:
                node.metadata[_ON_DEFAULT_STREAM] = True


def _refuse_marked_leaves(ctx):
    """In a backward pass that is being captured."""
    for node, _ in ctx.next_functions:
        if type(node) is _AccumulateGrad and _ON_DEFAULT_STREAM in node.metadata:
            raise RuntimeError('%s: captured into a graph while an eager graph of the default stream holds the same leaf (shape %s).  Drop the '
                               'results of eager calls first, or make them on another stream' % (ctx.name(), tuple(node.variable.shape)))


def _first_order(backward):
    """once_differentiable, whose wrapping is left out of the usual backward (which builds no graph)."""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        if torch.cuda.is_current_stream_capturing():
            _refuse_marked_leaves(ctx)
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


def _differentiated(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _tracked(*tensors):
    """Whether autograd has to see the call: for gradients, or to refuse forward-mode derivatives (dual tensors need no gradient and
    have an address like others; torch raises NotImplementedError for a function without a rule for them, under no_grad too)."""
    return forward_ad._current_level >= 0 or _differentiated(*tensors)


# =============================================================================================
# buckets
# =============================================================================================
@functools.lru_cache(maxsize=64)
def rel_buckets(num_buckets, max_distance, bidirectional):
    """struct tcvom_rel_buckets: `num_buckets` buckets (half of them for each direction if bidirectional).  Half the buckets of a side
    hold one distance each; bucket exact + k of the others starts at the smallest distance d with
    (d / exact)^m >= (max_distance / exact)^k, m = their number -- in whole numbers, so that no border depends on a logarithm's
    rounding."""
    side = num_buckets // 2 if bidirectional else num_buckets
    if num_buckets < 2 or num_buckets > L.MAX_BUCKETS or (bidirectional and num_buckets % 2) or side < 2:
        raise ValueError('%d buckets: 2..%d, even and at least 4 if bidirectional' % (num_buckets, L.MAX_BUCKETS))
    exact = side // 2
    m = side - exact
    if not exact < max_distance <= L.MAX_BUCKET_REACH:
        raise ValueError('max_distance %d: more than the %d distances with a bucket of their own, at most %d'
                         % (max_distance, exact, L.MAX_BUCKET_REACH))
    starts, d = [], exact
    for k in range(m):
        while d ** m * exact ** k < max_distance ** k * exact ** m:
            d += 1
        starts.append(d)
    b = L.RelBuckets(num_buckets, int(bidirectional), exact, m)
    b.starts[:m] = starts
    return b


def _check_table(name, table):
    if table.dim() != 2 or table.dtype != torch.float32:
        raise ValueError('%s: the table is fp32 [buckets, heads], got %s %s' % (name, table.dtype, tuple(table.shape)))


# =============================================================================================
# the bias as a matrix
# =============================================================================================
def _rel_bias(table, buckets, q_len, k_len, q_start, dtype):
    heads = table.shape[1]
    out = torch.empty((heads, q_len, k_len), dtype=dtype, device=table.device)
    _launch(table.get_device(), 'tcvom_relbias_fwd', _c(table).data_ptr(), out.data_ptr(), C.byref(buckets), heads, q_len, k_len, q_start,
            _TYPES[dtype])
    return out


class _RelBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, *args):
        ctx.args = (table.shape[1],) + args
        return _rel_bias(table, *args)

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        heads, buckets, q_len, k_len, q_start, dtype = ctx.args
        dtable = torch.empty((buckets.num_buckets, heads), dtype=torch.float32, device=dout.device)
        if q_len == 0 or k_len == 0:
            return dtable.zero_(), None, None, None, None, None
        dout = _c(dout)
        n = L.call('tcvom_relbias_bwd_work', C.byref(buckets), heads, q_len)
        work = torch.empty(n, dtype=torch.float32, device=dout.device)
        _launch(dout.get_device(), 'tcvom_relbias_bwd', dout.data_ptr(), dtable.data_ptr(), work.data_ptr(), n, C.byref(buckets), heads,
                q_len, k_len, q_start, _TYPES[dtype])
        return dtable, None, None, None, None, None


def relative_position_bias(table, q_len, k_len, max_distance=128, bidirectional=True, q_start=0, dtype=torch.float32):
    """bias[h, i, j] = table[bucket(j - i - q_start), h]: [heads, q_len, k_len] of `dtype`, to be added to attention logits.

    table: fp32 [buckets, heads].  Bidirectional: half the buckets for keys behind the query, half for keys after it (distance
    |j - i - q_start|); one-sided: every key after the query counts as distance 0.  The first half of a side's buckets hold one
    distance each, the others grow geometrically up to max_distance (at most 1024), the last holds everything beyond.  q_start:
    position of the first query.  Where the table needs a gradient: at most 1048560 queries."""
    _check_cuda('relative_position_bias', (table,))
    _check_table('relative_position_bias', table)
    if dtype not in _TYPES:
        raise TypeError('relative_position_bias: dtype %s' % dtype)
    if q_len < 0 or k_len < 0:
        raise ValueError('relative_position_bias: lengths %d, %d' % (q_len, k_len))
    if not -(1 << 40) < q_start < 1 << 40:
        raise ValueError('relative_position_bias: q_start %d' % q_start)
    buckets = rel_buckets(table.shape[0], int(max_distance), bool(bidirectional))
    if q_len > L.MAX_RELBIAS_BWD_QUERIES and _differentiated(table):
        raise ValueError('relative_position_bias: %d queries with a gradient (at most %d)' % (q_len, L.MAX_RELBIAS_BWD_QUERIES))
    args = (table, buckets, int(q_len), int(k_len), int(q_start), dtype)
    if not _tracked(table):
        return _rel_bias(*args)
    out = _RelBias.apply(*args)
    _mark_leaves(table.get_device(), out)
    return out


# =============================================================================================
# attention with the bias inside
# =============================================================================================
def _rows16(t):
    """[B, N, heads, width] as the kernels read it: innermost stride 1, the others multiples of 8, tokens less than 2^24 elements apart,
    16-byte aligned; a copy if not."""
    a, b, c, d = t.stride()
    if d == 1 and (a | b | c) % 8 == 0 and b < 1 << 24 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    a, b, c, _ = t.stride()
    x, y, z, _ = t.shape
    return a if x > 1 else 0, b if y > 1 else 0, c if z > 1 else 0


def _attn_desc(q, k, v, buckets, causal, scale, k_lens, key_mask, q_start, q_starts):
    B, Nq, H, D = q.shape
    return L.AttnDesc(B, Nq, k.shape[1], H, k.shape[2], D, _TYPES[q.dtype], causal, q_start, scale, _strides(q), _strides(k), _strides(v),
                      _p(k_lens), _p(q_starts), _p(key_mask), buckets)


def _attention(q, k, v, table, train, keep32, *args):
    """(out, out in 32 bits or None, lse or None) of tensors in the kernels' layout."""
    d = C.byref(_attn_desc(q, k, v, *args))
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device) if train else None
    out32 = torch.empty(q.shape, dtype=torch.float32, device=q.device) if keep32 else None
    n = L.call('tcvom_attn_fwd_work', d)
    work = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    _launch(q.get_device(), 'tcvom_attn_fwd', d, q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), out.data_ptr(), _p(out32), _p(lse),
            _p(work), n)
    return out, out32, lse


class _BiasedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, *args):
        q, k, v, table = _rows16(q), _rows16(k), _rows16(v), _c(table)
        out, out32, lse = _attention(q, k, v, table, True, ctx.needs_input_grad[3], *args)
        buckets, causal, scale, k_lens, key_mask, q_start, q_starts = args
        ctx.save_for_backward(q, k, v, table, out, out32, lse, k_lens, key_mask, q_starts)
        ctx.args = (buckets, causal, scale, q_start)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, dout):
        q, k, v, table, out, out32, lse, k_lens, key_mask, q_starts = ctx.saved_tensors
        buckets, causal, scale, q_start = ctx.args
        dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
        dtable = torch.empty_like(table) if ctx.needs_input_grad[3] else None
        if q.numel() == 0 or k.numel() == 0:
            return (dq.zero_(), dk.zero_(), dv.zero_(), None if dtable is None else dtable.zero_()) + (None,) * 7
        dout = _rows16(dout)
        d = C.byref(_attn_desc(q, k, v, buckets, causal, scale, k_lens, key_mask, q_start, q_starts))
        n = L.call('tcvom_attn_bwd_work', d)
        work = torch.empty(n, dtype=torch.float32, device=q.device)
        _launch(q.get_device(), 'tcvom_attn_bwd', d, q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), out.data_ptr(), _p(out32),
                lse.data_ptr(), dout.data_ptr(), (C.c_int64 * 3)(*_strides(dout)), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _p(dtable),
                work.data_ptr(), n)
        return dq, dk, dv, dtable, None, None, None, None, None, None, None


def biased_attention(q, k, v, table, max_distance=128, bidirectional=None, causal=False, scale=None, k_lens=None, key_mask=None,
                     q_start=0):
    """softmax(scale q k^T + bias) v with bias = relative_position_bias(table, ...), never formed as a matrix: [B, Nq, H, D].

    q [B, Nq, H, D], k / v [B, Nk, Hkv, D], bf16 or fp16, D a multiple of 8 up to 128; H a multiple of Hkv (consecutive heads share
    keys).  Any strides with contiguous rows of D; others are copied.
    table fp32 [buckets, H] and max_distance as in relative_position_bias; bidirectional: default not causal.  -inf takes a distance
    out; finite entries count as at most 90852 (2^17 in base 2) in size; those of distances that no query sees may hold anything.
    scale: default D ** -0.5, positive.  Key j sits at position j, query i of sequence b at i + q_start[b] (an int, or int32 [B]).
    Query i sees key j if j < k_lens[b] (int32 [B]; clamped to 0..Nk), key_mask[b, j] (bool or uint8 [B, Nk]) and, causal,
    j <= i + q_start[b].  A query that sees nothing gives zeros and no gradient.  What lies behind the lengths or under the mask
    may hold anything, NaN included (a NaN or inf that a later query sees can reach earlier ones of a causal call: 0 x inf).  For one
    new token against caches of Nk slots: k_lens = lengths with the new token, q_start = k_lens - 1, causal.

    Gradients of q, k, v and table.  Probabilities and their gradients are rounded to the 16-bit type as operands of the matrix
    products (in fp16 times powers of two, so that a small dout loses no bits of them and a large one does not overflow); where
    the table needs no gradient, <dout, out> of dq and dk is formed from the rounded result.  Everything else is held in 32 bits."""
    name = 'biased_attention'
    q_starts = None
    if isinstance(q_start, torch.Tensor):
        q_starts, q_start = q_start, 0
    _check_cuda(name, (q, k, v, table), k_lens, key_mask, q_starts)
    _check_table(name, table)
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError('%s: q, k, v are all bf16 or all fp16, got %s, %s, %s' % (name, q.dtype, k.dtype, v.dtype))
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError('%s: q [B, Nq, H, D], k and v [B, Nk, Hkv, D]; got %s, %s, %s' % (name, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    B, Nq, H, D = q.shape
    Nk, Hkv = k.shape[1:3]
    if D % 8 or not 8 <= D <= 128:
        raise ValueError('%s: head width %d (a multiple of 8 up to 128)' % (name, D))
    if H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError('%s: %d heads on %d key heads' % (name, H, Hkv))
    if table.shape[1] != H:
        raise ValueError('%s: the table has %d heads, q %d' % (name, table.shape[1], H))
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError('%s: scale %g' % (name, scale))
    for what, t in (('k_lens', k_lens), ('q_start', q_starts)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (B,)):
            raise ValueError('%s: %s is int32 [%d], got %s %s' % (name, what, B, t.dtype, tuple(t.shape)))
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != (B, Nk):
            raise ValueError('%s: key_mask is bool or uint8 [%d, %d], got %s %s' % (name, B, Nk, key_mask.dtype, tuple(key_mask.shape)))
        key_mask = _c(key_mask).view(torch.uint8)
    if not -(1 << 29) <= int(q_start) <= 1 << 29:
        raise ValueError('%s: q_start %d' % (name, q_start))
    buckets = rel_buckets(table.shape[0], int(max_distance), bool(not causal if bidirectional is None else bidirectional))
    args = (buckets, int(causal), scale, _c(k_lens), key_mask, int(q_start), _c(q_starts))
    if B * Hkv * -(-Nk // 128) + H > L.MAX_ATTN_WORKGROUPS and _differentiated(q, k, v, table):
        raise ValueError('%s: %d sequences x %d key heads x %d keys with gradients (at most 2^30 rows of keys)' % (name, B, Hkv, Nk))
    if _tracked(q, k, v, table):
        out = _BiasedAttention.apply(q, k, v, table, *args)
        _mark_leaves(q.get_device(), out)
        return out
    return _attention(_rows16(q), _rows16(k), _rows16(v), _c(table), False, False, *args)[0]


# =============================================================================================
# norms around a block
# =============================================================================================
def _block_norm(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, train, gate_rows, branch_scale, residual_scale, eps, layer):
    """(x', h, row statistics or None) of contiguous tensors."""
    channels = x.shape[-1]
    tokens = x.numel() // channels
    y_type = x.dtype if y is None else y.dtype
    xo = None if y is None else torch.empty_like(x)
    h = None if pre_weight is None else torch.empty_like(x if y is None else y)
    stats = torch.empty((tokens, 4), dtype=torch.float32, device=x.device) if train else None
    _launch(x.get_device(), 'tcvom_block_norm_fwd', x.data_ptr(), _p(y), _p(post_weight), _p(post_bias), _p(gate),
            int(gate is not None and gate.dtype == torch.float32), gate_rows, _p(pre_weight), _p(pre_bias), branch_scale, residual_scale, eps,
            layer, _p(xo), _p(h), _p(stats), tokens, channels, _TYPES[x.dtype], _TYPES[y_type])
    return xo, h, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_weight, post_bias, gate, pre_weight, pre_bias, *args):
        ctx.set_materialize_grads(False)
        x, y, post_weight, post_bias, gate, pre_weight, pre_bias = (_c(t) for t in (x, y, post_weight, post_bias, gate, pre_weight, pre_bias))
        xo, h, stats = _block_norm(x, y, post_weight, post_bias, gate, pre_weight, pre_bias, True, *args)
        ctx.save_for_backward(x, y, post_weight, post_bias, gate, pre_weight, stats)
        ctx.args = args
        return xo, h

    @staticmethod
    @_first_order
    def backward(ctx, dxo, dh):
        x, y, post_weight, post_bias, gate, pre_weight, stats = ctx.saved_tensors
        gate_rows, branch_scale, residual_scale, _, layer = ctx.args
        need = ctx.needs_input_grad
        if dxo is None and dh is None:
            return (None,) * 12
        dxo, dh = _c(dxo), _c(dh)

        def like(t, wanted=True):
            return torch.empty_like(t) if t is not None and wanted else None

        pre = dh is not None
        channels = x.shape[-1]
        tokens = x.numel() // channels
        dx, dy = like(x), like(y)
        dw1, db1, dg = like(post_weight, need[2]), like(post_bias, need[3]), like(gate, need[4])
        dw2 = like(pre_weight, need[5] and pre)
        db2 = torch.empty(channels, dtype=torch.float32, device=x.device) if need[6] and pre else None
        if tokens == 0:
            return tuple(None if t is None else t.zero_() for t in (dx, dy, dw1, db1, dg, dw2, db2)) + (None,) * 5
        groups = tokens // gate_rows if gate is not None and gate_rows > 1 else 1
        n = L.call('tcvom_block_norm_bwd_work', tokens, channels, groups)
        work = torch.empty(n, dtype=torch.float32, device=x.device)
        _launch(x.get_device(), 'tcvom_block_norm_bwd', x.data_ptr(), _p(y), _p(post_weight), _p(post_bias), _p(gate),
                int(gate is not None and gate.dtype == torch.float32), gate_rows, _p(pre_weight), branch_scale, residual_scale, layer,
                stats.data_ptr(), _p(dxo), _p(dh), dx.data_ptr(), _p(dy), _p(dw1), _p(db1), _p(dg), _p(dw2), _p(db2), work.data_ptr(), n,
                tokens, channels, _TYPES[x.dtype], _TYPES[x.dtype if y is None else y.dtype])
        return dx, dy, dw1, db1, dg, dw2, db2, None, None, None, None, None


def _gate_rows(shape, gate):
    """Tokens that share a row of the gate, from the shapes."""
    lead, g = shape[:-1], gate[:-1]
    n = len(g)
    while n and g[n - 1] == 1 and lead[n - 1:n] != (1,):
        n -= 1
    if len(gate) == 0 or gate[-1] != shape[-1] or len(g) > len(lead) or g[:n] != lead[:n]:
        raise ValueError('block_norm: a gate of %s for %s: one of each channel, of each leading index, or of each token'
                         % (tuple(gate), tuple(shape)))
    rows = max(math.prod(lead[n:]), 1)
    if rows > 1 and math.prod(lead[:n]) > 32768:
        raise ValueError('block_norm: %d gate rows of several tokens (at most 32768)' % math.prod(lead[:n]))
    return rows


def block_norm(x, y, post_weight=None, post_bias=None, gate=None, branch_scale=1.0, residual_scale=1.0, pre_weight=None, pre_bias=None,
               kind='rms', eps=1e-6):
    """(x', h): x' = residual_scale x + branch_scale gate N(y; post), h = N(x'; pre), in one pass.

    x [..., C]: the residual stream, y (same shape): what a block made of the last h; N: RMSNorm (kind 'rms') or LayerNorm ('layer') over
    the C <= 8192 channels, weights and biases fp32 [C] (biases with LayerNorm only).  Without post_weight y enters as it is; without
    pre_weight h is None; y None: (x, N(x; pre)), the norm in front of the first block.  h is formed from x' before x' is rounded.
    gate: [C], [lead..., C] where lead are the first dimensions of x (a gate of each sample), or the shape of x; fp32 or y's type.
    x and y of one type (fp32, bf16, fp16), or x fp32 with a 16-bit y; h has y's type.

    Gradients of every tensor argument."""
    name = 'block_norm'
    _check_cuda(name, (x,), y, post_weight, post_bias, gate, pre_weight, pre_bias)
    if kind not in ('rms', 'layer'):
        raise ValueError('%s: kind %r' % (name, kind))
    x_type, shape = x.dtype, x.shape
    y_type = x_type if y is None else y.dtype
    if x_type not in _TYPES or y_type not in _TYPES or (y_type != x_type and x_type != torch.float32):
        raise TypeError('%s: x %s, y %s' % (name, x_type, y_type))
    channels = shape[-1] if shape else 0
    if not 0 < channels <= L.MAX_NORM_CHANNELS:
        raise ValueError('%s: %s (1..%d channels)' % (name, tuple(shape), L.MAX_NORM_CHANNELS))
    if y is None:
        if pre_weight is None or post_weight is not None or post_bias is not None or gate is not None or residual_scale != 1.0:
            raise ValueError('%s: without y there is the pre norm only' % name)
    elif y.shape != shape:
        raise ValueError('%s: x %s, y %s' % (name, tuple(shape), tuple(y.shape)))
    for t in (post_weight, post_bias, pre_weight, pre_bias):
        if t is not None and (t.dtype != torch.float32 or t.dim() != 1 or t.size(0) != channels):
            raise ValueError('%s: weights and biases are fp32 [%d], got %s %s' % (name, channels, t.dtype, tuple(t.shape)))
    if (post_bias is not None and (post_weight is None or kind != 'layer')) or (pre_bias is not None and (pre_weight is None or kind != 'layer')):
        raise ValueError('%s: a bias goes with LayerNorm and a weight' % name)
    rows = 1
    if gate is not None:
        if gate.dtype != torch.float32 and gate.dtype != y_type:
            raise TypeError('%s: gate %s with y %s' % (name, gate.dtype, y_type))
        rows = _gate_rows(shape, gate.shape)
    args = (rows, float(branch_scale), float(residual_scale), float(eps), int(kind == 'layer'))
    tensors = (x, y, post_weight, post_bias, gate, pre_weight, pre_bias)
    if _tracked(*tensors):
        xo, h = _BlockNorm.apply(*tensors, *args)
        _mark_leaves(x.get_device(), h if xo is None else xo)
    else:
        xo, h, _ = _block_norm(*[_c(t) for t in tensors], False, *args)
    return (x if y is None else xo), h
