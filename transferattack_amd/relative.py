"""Attention whose scores carry a learned relative position bias, as HIP kernels (csrc/nn/attention*.hip):

    s_ij = scale q_i . k_j + table[bucket(i, j)][head] + mask_ij
    o_i  = sum_j softmax_j(s_ij) v_j

The window transformer the reference evaluates on (transferattack/utils.py:16-17) adds such a table to the scores of its
windows, a bucket for each 2-D offset; sequence models use logarithmic distance buckets.  ``RelativeBuckets`` is the plan that
says which bucket a pair has -- built once, like the module's ``relative_position_index`` buffer -- ``relative_attention`` the
operator, ``relative_attention_packed`` the same on a projection's output as it lies in memory.  Both have a backward pass
(queries, keys, values, table) and take single tokens against a long cache.  No scores are written to memory; the table's gradient
takes partial sums of their gradients, [parts, heads, m, n] for pairs, and with a mask for every sequence a part is a sequence.

No fallback: tensors must be on a HIP device."""
import torch
from torch.autograd.function import once_differentiable

from . import _nn

FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_DIM = 128


class RelativeBuckets:
    """Which row of a bias table a (query, key) pair takes.

    ``from_index(index)``              any [queries, keys] tensor of bucket numbers (a window's ``relative_position_index``)
    ``by_distance(buckets, first)``    buckets[d - first] for distance d = key position - query position; further distances take
                                       the nearer end's bucket.  Works for every number of queries and keys.
    ``logarithmic(...)``               ``by_distance`` with the usual rule: half of a side's buckets one distance each, the others
                                       logarithmic up to ``max_distance``

    A plan lives on one device (``to`` makes it anew on another) and never changes."""

    def __init__(self):
        raise TypeError("use RelativeBuckets.from_index, .by_distance or .logarithmic")

    @classmethod
    def _new(cls, **fields):
        self = object.__new__(cls)
        self.__dict__.update(fields)
        if self.device.type == "cuda":                   # ready for every stream: a module keeps its plan from the first call on
            torch.cuda.current_stream(self.device).synchronize()
        return self

    @classmethod
    def from_index(cls, index):
        _check_buckets(index, 2, "index")
        m, n = index.shape
        flat = index.reshape(-1).to(torch.int64)
        buckets = int(flat.max()) + 1
        if int(flat.min()) < 0 or buckets > 65536:
            raise ValueError("bucket numbers must be 0 .. 65535, got %d .. %d" % (int(flat.min()), buckets - 1))

        def padded(t):                                   # 16-bit bucket numbers, rows a multiple of 4 apart
            rows, cols = t.shape
            out = torch.zeros((rows, (cols + 3) // 4 * 4), dtype=torch.int16, device=t.device)
            out[:, :cols] = t.to(torch.int32).to(torch.int16)
            return out

        order = torch.sort(flat, stable=True)[1].to(torch.int32)
        starts = torch.zeros(buckets + 1, dtype=torch.int64, device=index.device)
        starts[1:] = torch.cumsum(torch.bincount(flat, minlength=buckets), 0)
        return cls._new(source=index.detach().clone(), device=index.device, buckets=buckets, shape=(m, n), distances=0, first=0, index=padded(index),
                        index_t=padded(index.t()), order=order, starts=starts.to(torch.int32))

    @classmethod
    def by_distance(cls, buckets, first):
        _check_buckets(buckets, 1, "buckets")
        if not isinstance(first, int) or abs(first) >= 1 << 30 or buckets.numel() >= 1 << 29:
            raise ValueError("first must be an int below 2^30, got %r" % (first,))
        low, high = int(buckets.min()), int(buckets.max())
        if low < 0 or high > 65535:
            raise ValueError("bucket numbers must be 0 .. 65535, got %d .. %d" % (low, high))
        return cls._new(source=buckets.detach().clone(), device=buckets.device, buckets=high + 1, shape=None, distances=buckets.numel(), first=first,
                        index=buckets.to(torch.int32).contiguous().clone(), index_t=None, order=None, starts=None)

    @classmethod
    def logarithmic(cls, num_buckets=32, max_distance=128, bidirectional=True, device=None):
        """Bucket of distance d = key - query: with ``bidirectional`` the upper half of the buckets is for d > 0, else every
        d > 0 shares bucket 0 with d = 0.  Of a side's s buckets the first s // 2 take one distance each; bucket s // 2 + t
        begins where |d| >= near (max_distance / near)^(t / (s - near)), near = s // 2 -- decided in whole numbers."""
        side = num_buckets // 2 if bidirectional else num_buckets
        near = side // 2
        if near < 1 or max_distance <= near:
            raise ValueError("%d buckets up to distance %d" % (num_buckets, max_distance))
        far = side - near

        def one_side(d):
            if d < near:
                return d
            return near + sum(1 for t in range(1, far) if d ** far >= near ** (far - t) * max_distance ** t)

        away = [one_side(d) for d in range(max_distance + 1)]
        ahead = [side + b if bidirectional else 0 for b in away[1:]]
        buckets = torch.tensor(away[::-1] + ahead, dtype=torch.int32)
        return cls.by_distance(buckets if device is None else buckets.to(device), -max_distance)

    def to(self, device):
        if torch.device(device) == self.device:
            return self
        source = self.source.to(device)
        return type(self).by_distance(source, self.first) if self.distances else type(self).from_index(source)


def _check_buckets(t, dims, name):
    if not isinstance(t, torch.Tensor) or t.dim() != dims or t.numel() == 0 or t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise ValueError("%s must be a non-empty %d-D tensor of whole numbers" % (name, dims))


# ------------------------------------------------------------------------------------------------------------ the call
class _Call:
    """one call's options, checked; `tensors` are (mask, key lengths, query starts), each a tensor or None"""
    __slots__ = ("buckets", "scale", "causal", "start", "tensors")

    def keep(self):
        """the tensors, for ``save_for_backward``: changed before the backward pass they are an error, so no one else holds them"""
        tensors, self.tensors = self.tensors, None
        return _nn.kept(*tensors)


def _int32(t, low, high):
    """as the kernels take it; 64-bit numbers past ``low`` or ``high`` mean the same as those"""
    return (t if t.dtype == torch.int32 else t.clamp(low, high).to(torch.int32)).contiguous()


def _options(q, k, table, buckets, scale, mask, causal, key_lengths, query_start):
    if not isinstance(buckets, RelativeBuckets):
        raise TypeError("buckets must be RelativeBuckets, got %s" % type(buckets).__name__)
    batch, heads, m, dim = q.shape
    n = k.shape[2]
    if max(batch, heads, m, n) >= 1 << 30:               # (an expanded tensor may be that long; the library's sizes have 32 bits)
        raise ValueError("batch %d, %d heads, %d queries, %d keys (below 2^30 each)" % (batch, heads, m, n))
    _nn.check_tensor(table, "table", q, FLOATS)
    if table.dim() != 2 or table.shape[1] != heads:
        raise ValueError("table must be [buckets, %d heads], got %s" % (heads, tuple(table.shape)))
    if table.shape[0] < buckets.buckets:
        raise ValueError("the table has %d buckets, the plan uses %d" % (table.shape[0], buckets.buckets))
    if buckets.device != q.device:
        raise ValueError("buckets are on %s, not on %s" % (buckets.device, q.device))
    if buckets.shape is not None and buckets.shape != (m, n):
        raise ValueError("buckets are for %d queries and %d keys, not %d and %d" % (buckets.shape + (m, n)))
    o = _Call()
    o.buckets, o.causal = buckets, bool(causal)
    o.scale = dim ** -0.5 if scale is None else float(scale)
    view = lengths = starts = None
    if mask is not None:
        _nn.check_tensor(mask, "mask", q, FLOATS + (torch.bool,))
        if mask.requires_grad:
            raise ValueError("the mask has no gradient: a learned bias belongs into the table")
        if mask.dim() not in (2, 3, 4):
            raise ValueError("mask must be [m, n], [period, m, n] or [period, heads, m, n], got %s" % (tuple(mask.shape),))
        view = mask[None, None] if mask.dim() == 2 else mask[:, None] if mask.dim() == 3 else mask
        p, h, i, j = view.shape
        if p == 0 or batch % p or h not in (1, heads) or i not in (1, m) or j not in (1, n):
            raise ValueError("mask %s does not fit batch %d, %d heads, %d queries, %d keys" % (tuple(mask.shape), batch, heads, m, n))
    if key_lengths is not None:
        _nn.check_tensor(key_lengths, "key_lengths", q, (torch.int32, torch.int64))
        if key_lengths.shape != (batch,):
            raise ValueError("key_lengths must be [%d], got %s" % (batch, tuple(key_lengths.shape)))
        lengths = _int32(key_lengths, 0, n)
    o.start = 0
    if isinstance(query_start, torch.Tensor):
        _nn.check_tensor(query_start, "query_start", q, (torch.int32, torch.int64))
        if query_start.shape != (batch,):
            raise ValueError("query_start must be an int or [%d], got %s" % (batch, tuple(query_start.shape)))
        starts = _int32(query_start, -(1 << 31) + 1, (1 << 31) - 1)
    else:
        o.start = int(query_start)
        if abs(o.start) >= 1 << 30:
            raise ValueError("query_start %d" % o.start)
    o.tensors = view, lengths, starts
    return o


def _arguments(q, k, v, table, out, stats, o, tensors):
    mask, lengths, starts = tensors
    a = _nn.AttentionArgs()
    a.dtype, a.batch, a.heads, a.m, a.dim = _nn.DTYPES[q.dtype], q.shape[0], q.shape[1], q.shape[2], q.shape[3]
    a.kv_heads, a.n = k.shape[1], k.shape[2]
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.q_sb, a.q_sh, a.q_sm, _ = q.stride()
    a.k_sb, a.k_sh, a.k_sn, _ = k.stride()
    a.v_sb, a.v_sh, a.v_sn, _ = v.stride()
    a.o_sb, a.o_sh, a.o_sm, _ = out.stride()
    a.scale, a.table_dtype, a.buckets, a.table = o.scale, _nn.DTYPES[table.dtype], table.shape[0], table.data_ptr()
    b = o.buckets
    a.distances, a.first, a.index = b.distances, b.first, b.index.data_ptr()
    if b.index_t is not None:
        a.index_t, a.index_stride, a.index_t_stride = b.index_t.data_ptr(), b.index.stride(0), b.index_t.stride(0)
    if mask is not None:
        a.mask = mask.data_ptr()
        a.mask_kind = _nn.MASK_BOOL if mask.dtype == torch.bool else _nn.MASK_FLOAT + _nn.DTYPES[mask.dtype]
        a.mask_period = mask.shape[0]
        a.mask_sb, a.mask_sh, a.mask_sm, a.mask_sn = [0 if size == 1 else stride for size, stride in zip(mask.shape, mask.stride())]
    a.key_lengths, a.query_start, a.start, a.causal = _nn.ptr(lengths), _nn.ptr(starts), o.start, int(o.causal)
    a.stats = _nn.ptr(stats)
    return a


def _workspace(a, like, backward):
    floats = _nn.load().ta_nn_attention_workspace(a, int(backward))
    if floats == 0:
        return None
    ws = torch.empty(floats, dtype=torch.float32, device=like.device)
    a.workspace = ws.data_ptr()
    return ws


def _forward(q, k, v, table, out, o, save):
    """-> statistics for a backward pass, or None"""
    stats = torch.empty(q.shape[:3] + (2,), dtype=torch.float32, device=q.device) if save else None
    if out.numel() == 0:
        return stats
    if k.shape[2] == 0:
        out.zero_()
        return stats
    a = _arguments(q, k, v, table, out, stats, o, o.tensors)
    ws = _workspace(a, q, False)                         # kept alive until the launches are enqueued
    _nn._launch("ta_nn_attention", q, a)
    del ws
    return stats


def _backward(q, k, v, table, out, stats, grad, dq, dk, dv, table_grad, o, tensors):
    dtable = None
    if table_grad:                                       # rows behind the plan's last bucket are not written
        covered = table.shape[0] == o.buckets.buckets and out.numel() > 0 and k.shape[2] > 0
        dtable = torch.empty_like(table) if covered else torch.zeros_like(table)
    if out.numel() == 0 or k.shape[2] == 0:
        for t in (dq, dk, dv):
            t.zero_()
        return dtable
    grad = _dense_rows(grad)
    a = _arguments(q, k, v, table, out, stats, o, tensors)
    a.grad = grad.data_ptr()
    a.g_sb, a.g_sh, a.g_sm, _ = grad.stride()
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    a.dq_sb, a.dq_sh, a.dq_sm, _ = dq.stride()
    a.dk_sb, a.dk_sh, a.dk_sn, _ = dk.stride()
    a.dv_sb, a.dv_sh, a.dv_sn, _ = dv.stride()
    if dtable is not None:
        a.dtable, a.pair_order, a.pair_starts = dtable.data_ptr(), _nn.ptr(o.buckets.order), _nn.ptr(o.buckets.starts)
        a.buckets = o.buckets.buckets
    ws = _workspace(a, q, True)
    _nn._launch("ta_nn_attention_backward", q, a)
    del ws
    return dtable


def _token_major(batch, heads, tokens, dim, like):
    """[batch, heads, tokens, dim] in [batch, tokens, heads, dim] memory: what a projection reads or writes"""
    return torch.empty((batch, tokens, heads, dim), dtype=like.dtype, device=like.device).transpose(1, 2)


class _RelativeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, o):
        out = _token_major(q.shape[0], q.shape[1], q.shape[2], q.shape[3], q)
        stats = _forward(q, k, v, table, out, o, True)
        ctx.options = o
        ctx.save_for_backward(q, k, v, table, out, stats, *o.keep())
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, table, out, stats, *tensors = ctx.saved_tensors
        dq = _token_major(q.shape[0], q.shape[1], q.shape[2], q.shape[3], q)
        dk = _token_major(k.shape[0], k.shape[1], k.shape[2], k.shape[3], k)
        dv = _token_major(v.shape[0], v.shape[1], v.shape[2], v.shape[3], v)
        dtable = _backward(q, k, v, table, out, stats, grad, dq, dk, dv, ctx.needs_input_grad[3], ctx.options, tensors)
        return dq, dk, dv, dtable, None


def _packed_forward(qkv, table, o, save):
    b, n, _, heads, dim = qkv.shape
    out = torch.empty((b, n, heads, dim), dtype=qkv.dtype, device=qkv.device)
    q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
    return out, _forward(q, k, v, table, out.transpose(1, 2), o, save)


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, table, o):
        out, stats = _packed_forward(qkv, table, o, True)
        ctx.options = o
        ctx.save_for_backward(qkv, table, out, stats, *o.keep())
        return out.flatten(2)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        qkv, table, out, stats, *tensors = ctx.saved_tensors
        q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        dq, dk, dv = dqkv.permute(2, 0, 3, 1, 4).unbind(0)
        grad = grad.reshape(out.shape).transpose(1, 2)
        dtable = _backward(q, k, v, table, out.transpose(1, 2), stats, grad, dq, dk, dv, ctx.needs_input_grad[1], ctx.options, tensors)
        return dqkv, dtable, None


def _dense_rows(t, token=2):
    """as the kernels take it: the innermost dimension dense, tokens less than 2^23 elements apart"""
    dense = (t.stride(-1) == 1 or t.shape[-1] == 1) and t.stride(token) < 1 << 23
    return t if dense else t.contiguous()


def _padding(t):
    """elements that make a head's dimension whole 16-byte vectors; they are zeros, which no score sees"""
    return -t.shape[-1] % (4 if t.dtype == torch.float32 else 8)


def relative_attention(q, k, v, table, buckets, scale=None, mask=None, causal=False, key_lengths=None, query_start=0):
    """Attention with ``table[bucket][head]`` added to every score.

    q [batch, heads, m, dim], k / v [batch, kv_heads, n, dim] in fp32, bf16 or fp16, any strides (copied if the innermost
    dimension is not dense, padded if it is not whole 16-byte vectors); heads a multiple of kv_heads (head h uses key head h // (heads // kv_heads)); dim <= 128.
    table [buckets, heads], fp32, bf16 or fp16.  ``scale`` defaults to dim ** -0.5.
    mask         bool (True: may be seen) or additive, [m, n], [period, m, n] or [period, heads, m, n] with 1 for a dimension it
                 does not depend on; sequence b takes mask b % period (windows of an image).  No gradient.
    causal       key j is seen by queries at positions >= j
    key_lengths  [batch] keys in use; what lies behind them is not read and its gradients are 0.  (This, the mask and query_start must
                 not change before a backward pass: autograd raises if they do)
    query_start  position of query 0 (an int, or [batch] tensor): query i stands at query_start + i, key j at j
    A query that sees no key gives zeros and takes no gradient.  Keys that only a mask hides have to be finite (0 * inf is
    NaN); those past ``key_lengths`` may hold anything.  The table's gradient with distance buckets needs an int ``query_start``.
    Returns [batch, heads, m, dim] in q's type, laid out [batch, m, heads, dim]."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _nn.check_tensor(t, name, q if name != "q" else None, FLOATS)
        if t.dim() != 4 or t.dtype != q.dtype:
            raise ValueError("%s must be [batch, heads, tokens, dim] of q's type, got %s %s" % (name, tuple(t.shape), t.dtype))
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError("q %s, k %s and v %s do not fit together" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not 1 <= q.shape[3] <= MAX_DIM:
        raise ValueError("head dimension %d (1 .. %d)" % (q.shape[3], MAX_DIM))
    o = _options(q, k, table, buckets, scale, mask, causal, key_lengths, query_start)
    _nn.no_tangents(q, k, v, table, mask)
    save = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or table.requires_grad)
    if save and table.requires_grad and o.tensors[2] is not None and buckets.distances:
        raise ValueError("the table's gradient needs one query_start for all sequences (an int)")
    dim, pad = q.shape[3], _padding(q)
    if pad:
        q, k, v = (torch.nn.functional.pad(t, (0, pad)) for t in (q, k, v))
    out = _call(_dense_rows(q), _dense_rows(k), _dense_rows(v), table.contiguous(), o, save)
    return out[..., :dim] if pad else out


def _call(q, k, v, table, o, save):
    if save:
        return _RelativeAttention.apply(q, k, v, table, o)
    out = _token_major(q.shape[0], q.shape[1], q.shape[2], q.shape[3], q)
    _forward(q, k, v, table, out, o, False)
    return out


def relative_attention_packed(qkv, table, buckets, scale=None, mask=None, causal=False, key_lengths=None):
    """``relative_attention`` on a projection's output: qkv [batch, n, 3, heads, dim] -> [batch, n, heads * dim].  The gradient
    of qkv is written in the same layout, without a copy."""
    _nn.check_tensor(qkv, "qkv", None, FLOATS)
    if qkv.dim() != 5 or qkv.shape[2] != 3 or not 1 <= qkv.shape[4] <= MAX_DIM or qkv.shape[3] < 1:
        raise ValueError("qkv must be [batch, n, 3, heads, dim <= %d], got %s" % (MAX_DIM, tuple(qkv.shape)))
    q = qkv.detach().select(2, 0).transpose(1, 2)
    o = _options(q, q, table, buckets, scale, mask, causal, key_lengths, 0)
    _nn.no_tangents(qkv, table, mask)
    save = torch.is_grad_enabled() and (qkv.requires_grad or table.requires_grad)
    dim, pad = qkv.shape[4], _padding(qkv)
    if pad:
        qkv = torch.nn.functional.pad(qkv, (0, pad))
    qkv, table = _dense_rows(qkv, 1), table.contiguous()
    out = _PackedAttention.apply(qkv, table, o) if save else _packed_forward(qkv, table, o, False)[0].flatten(2)
    return out.unflatten(2, (qkv.shape[3], dim + pad))[..., :dim].flatten(2) if pad else out
