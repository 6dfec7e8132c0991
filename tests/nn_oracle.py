"""The operators of transferattack_amd.relative / .distill in plain 64-bit torch on the CPU, with how far a kernel may be off.

Bounds.  u = 2^-24 is half a step of fp32 (the accumulators), t half a step of the tensors' type (torch.finfo(type).eps / 2; fp32:
u).  A score is a sum of dim products, a scaling, a bias and a mask: |error| <= e = (dim + 4) u (scale sum |q k| + |bias| + |mask|).
A probability is exp of a difference of two scores over a sum of such: relative error <= 2 e_max + 4 u |s - max| + (n + 8) u; where it
is an operand of a 16-bit product it is rounded once more, t.  Every result is a sum of products of those with exact inputs, so its
error is at most the sum of the terms' magnitudes times their relative errors, plus the accumulation's (terms u) and one
rounding to the tensors' type, t |result|.  All of it is evaluated entry by entry below, in 64 bits."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, table, bucket, scale, allowed, added, grad, dtype):
    """bucket [batch or 1, m, n]; allowed / added broadcast to [batch, heads, m, n] or None.  -> {name: (value, bound)}"""
    t = half_step(dtype)
    t16 = 0.0 if dtype == torch.float32 else t
    q, k, v, table = (x.detach().cpu().double() for x in (q, k, v, table))
    batch, heads, m, dim = q.shape
    kv, n = k.shape[1], k.shape[2]
    group = heads // kv
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    bias = table[bucket].movedim(-1, 1)
    s = q @ kk.transpose(-2, -1) * scale + bias
    size = q.abs() @ kk.abs().transpose(-2, -1) * abs(scale) + bias.abs()
    if added is not None:
        finite = added.clamp_min(-1e38)
        s = s + torch.where(added == -torch.inf, added, finite)
        size = size + torch.where(finite <= -1e38, torch.zeros_like(finite), finite.abs())
        # beside the lowest value a score vanishes in 32 bits, here too: such a row averages
        s = torch.where(s <= -1e37, s.float().double(), s)
    size = size.expand_as(s)
    if allowed is not None:
        s = s.masked_fill(~allowed, -torch.inf)
    seen = s > -torch.inf
    top = torch.where(seen.any(-1, keepdim=True), s.amax(-1, keepdim=True), torch.zeros(1, dtype=s.dtype)) if n else s.sum(-1, keepdim=True)
    e = torch.where(seen, s - top, torch.full_like(s, -torch.inf)).exp()
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total.clamp_min(1e-300), torch.zeros_like(e))
    err_s = torch.where(seen, (dim + 4) * U * size, torch.zeros_like(s))
    spread = torch.where(p > 0, (top - s).clamp(0, 200), torch.zeros_like(s))
    rel = 2 * (err_s.amax(-1, keepdim=True) if n else 0) + 4 * U * spread + (n + 8) * U
    tiny = 2.0 ** -120                                   # what the exponential may flush
    out = p @ vv
    got = {"out": (out, (p * (rel + t16 + n * U) + tiny) @ vv.abs() + t * out.abs() + 1e-30)}
    if grad is None:
        return got
    g = grad.detach().cpu().double()
    dp = g @ vv.transpose(-2, -1)
    dp_err = (dim + 4) * U * (g.abs() @ vv.abs().transpose(-2, -1))
    delta = (out * g).sum(-1, keepdim=True)
    # dq's kernel takes delta from the rounded output; for the keys and the table it is sum_j p dp in 32 bits
    delta_q = (got["out"][1] * g.abs()).sum(-1, keepdim=True) + (dim + 4) * U * (out * g).abs().sum(-1, keepdim=True)
    delta_k = ((p * (rel + n * U) + tiny) * dp.abs() + p * dp_err).sum(-1, keepdim=True)
    ds = p * (dp - delta)

    def ds_err(delta_err):
        return (p * rel + tiny) * (dp - delta).abs() + p * (1 + rel) * (dp_err + delta_err) + 2 * U * p * (dp.abs() + delta.abs())

    pe = p * (rel + t16 + m * group * U) + tiny
    dse_q = ds_err(delta_q) + (t16 + n * U) * ds.abs()
    dse_k = ds_err(delta_k) + (t16 + m * group * U) * ds.abs()

    def shared(x):
        return x.view(batch, kv, group, n, dim).sum(2)

    dq, dk, dv = ds @ kk * scale, shared(ds.transpose(-2, -1) @ q) * scale, shared(p.transpose(-2, -1) @ g)
    a = abs(scale)
    got["dq"] = (dq, dse_q @ kk.abs() * a + (t + 2 * U) * dq.abs() + 1e-30)
    got["dk"] = (dk, shared(dse_k.transpose(-2, -1) @ q.abs()) * a + (t + 2 * U) * dk.abs() + 1e-30)
    got["dv"] = (dv, shared(pe.transpose(-2, -1) @ g.abs()) + t * dv.abs() + 1e-30)
    flat = bucket.expand(batch, m, n).reshape(-1)
    dtable = torch.zeros_like(table).index_add_(0, flat, ds.movedim(1, -1).reshape(-1, heads))
    err = torch.zeros_like(table).index_add_(0, flat, ds_err(delta_k).movedim(1, -1).reshape(-1, heads))
    mass = torch.zeros_like(table).index_add_(0, flat, ds.abs().movedim(1, -1).reshape(-1, heads))
    got["dtable"] = (dtable, err + (batch + 64) * U * mass)
    return got


def close(name, value, want, table_dtype=None):
    """every entry within its bound, NaN nowhere"""
    ref, bound = want
    if table_dtype is not None:
        bound = bound + half_step(table_dtype) * ref.abs()
    value = value.detach().cpu().double()
    assert value.shape == ref.shape, (name, value.shape, ref.shape)
    off = (value - ref).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d entries off; worst %.3g against %.3g at value %.6g" % (
        name, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound[bad][off[bad].argmax()]), float(ref[bad][off[bad].argmax()]))


# ------------------------------------------------------------------------------------------------------------ distillation
def top_logits(x, top, temperature, dtype):
    """values, classes, (rest, its bound): the rest's sum of exponentials of up to `classes` terms has a relative error of the
    exponentials' (argument and result: (2 |x - m| / T + 4) u, weighted like the terms) plus the sum's (1000 u: a thread adds up
    to 128 terms in 32 bits, the rest is 64-bit)"""
    x = x.detach().cpu().double() + 0.0
    key = torch.where(torch.isnan(x), torch.full_like(x, torch.inf), x)
    nan = torch.isnan(x).double()
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    order = order.gather(1, torch.sort(nan.gather(1, order), dim=-1, descending=True, stable=True)[1])
    classes = order[:, :top]
    left = x.gather(1, order[:, top:]) / temperature
    rest = torch.logsumexp(left, -1) if left.shape[1] else torch.full((x.shape[0],), -torch.inf, dtype=x.dtype)
    if left.shape[1]:
        away = (left.amax(-1, keepdim=True) - left).clamp(0, 200).nan_to_num(0.0)
        w = torch.softmax(left, -1).nan_to_num(0.0)
        bound = ((2 * away + 4) * U * w).sum(-1) + 200 * U + U * rest.abs().nan_to_num(0.0, 0.0, 0.0)
    else:
        bound = torch.zeros_like(rest)
    return x.gather(1, classes), classes, (rest, bound)


def distillation(x, values, classes, rest, temperature, weight, dtype, scale):
    """Per row: (loss times weight, bound), and (gradient times ``scale`` [rows], bound).  The sums over a row carry a relative error
    r (as in top_logits); they move log q_R and log Z, so the loss by at most r (|p_R - q_R| + q_R) T^2, and every q by r; what
    concerns the classes answered is 64-bit."""
    x = x.detach().cpu().double()
    rows, n = x.shape
    values, classes = values.detach().cpu().double() / temperature, classes.detach().cpu().long()
    rest = None if rest is None else rest.detach().cpu().double()
    w = torch.ones(rows, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    losses, grads, bl, bg = [], [], [], []
    t = half_step(dtype)
    for i in range(rows):
        if w[i] == 0:
            losses.append(0.0), bl.append(0.0)
            grads.append(torch.zeros(n, dtype=torch.float64)), bg.append(torch.zeros(n, dtype=torch.float64))
            continue
        c = classes[i]
        ok = c >= 0
        bins = values[i][ok] if rest is None else torch.cat([values[i][ok], rest[i:i + 1]])
        c = c[ok]
        if bins.numel() == 0:
            losses.append(0.0), bl.append(0.0)
            grads.append(torch.zeros(n, dtype=torch.float64)), bg.append(torch.zeros(n, dtype=torch.float64))
            continue
        log_p = torch.log_softmax(bins, 0)
        s = x[i] / temperature
        log_q = torch.log_softmax(s, 0)
        others = torch.ones(n, dtype=torch.bool)
        others[c] = False
        at = log_q[c]
        log_rest = torch.logsumexp(log_q[others], 0) if others.any() else torch.tensor(-torch.inf, dtype=torch.float64)
        if rest is not None:
            at = torch.cat([at, log_rest[None]])
        p = log_p.exp()
        terms = torch.where(p > 0, p * (log_p - at), torch.zeros_like(p))
        losses.append(float(temperature ** 2 * terms.sum() * w[i]))
        q = log_q.exp()
        away = (s.max() - s).clamp(0, 200)
        r = float(((2 * away + 4) * U * q).sum() + 200 * U)
        q_rest = float(log_rest.exp())
        p_rest = float(p[-1]) if rest is not None else 0.0
        bl.append(temperature ** 2 * float(w[i]) * (r * (abs(p_rest - q_rest) + q_rest) + r * r * p_rest) + 2 * U * abs(losses[-1]) + 1e-12 * (1 + abs(losses[-1])))
        pv = torch.zeros(n, dtype=torch.float64).index_add_(0, c, p[:c.numel()])
        share = torch.where(others, q * (1.0 if rest is None else (q_rest - p_rest) / max(q_rest, 1e-300)), q - pv)
        f = float(scale[i]) * float(w[i]) * temperature
        grads.append(f * share)
        # the factor of the other classes is (q_R - p_R) / s: its numerator is off by r q_R, the exponential by its own error
        off = torch.where(others, (r + (2 * away + 6) * U) * q * max(1.0, 1 + p_rest / max(q_rest, 1e-300)), r * q + 1e-12)
        bg.append(abs(f) * (off + 3 * U * share.abs() + 2.0 ** -120) + t * abs(f) * share.abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-30))
    as64 = lambda v: torch.tensor(v, dtype=torch.float64)        # noqa: E731
    return (as64(losses), as64(bl)), (torch.stack(grads), torch.stack(bg))
