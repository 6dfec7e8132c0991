"""Checks of the operators in transferattack_amd.relative / .distill against nn_oracle, shared by the host tier (kernel sources
on tests/hipcpu's stand-in) and the GPU tier: the same functions, the device given by the caller."""
import torch

import nn_oracle
from transferattack_amd.distill import TopLogits, distillation_loss, distillation_loss_and_grad, top_logits
from transferattack_amd.relative import RelativeBuckets, relative_attention, relative_attention_packed

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def window_index(side):
    at = torch.arange(side * side)
    y, x = at // side, at % side
    return (y[:, None] - y[None] + side - 1) * (2 * side - 1) + x[:, None] - x[None] + side - 1


def case(dtype=F32, batch=2, heads=2, kv=None, m=5, n=None, dim=32, pairs=True, mask=None, causal=False, lengths=None, start=0,
         scale=None, layout="heads", table_dtype=F32, buckets=7, seed=0, train=True, spread=1.0):
    return dict(locals())


def _layout(t, layout):
    """the same values with other strides (the innermost dimension dense, except for 'inner')"""
    if layout == "tokens":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "padded":                               # rows further apart than they are long, at an odd offset
        room = torch.full(t.shape[:-1] + (t.shape[-1] + 3,), float("nan"), dtype=t.dtype, device=t.device)
        room[..., 1:1 + t.shape[-1]] = t
        return room[..., 1:1 + t.shape[-1]]
    if layout == "inner":
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)
    return t


def make_attention(c, device):
    gen = torch.Generator().manual_seed(c["seed"])
    batch, heads, m, dim = c["batch"], c["heads"], c["m"], c["dim"]
    n, kv = c["n"] or m, c["kv"] or heads
    randn = lambda *s: torch.randn(s, generator=gen) * c["spread"]      # noqa: E731
    q, k, v, grad = (randn(*s).to(c["dtype"]) for s in ((batch, heads, m, dim), (batch, kv, n, dim), (batch, kv, n, dim), (batch, heads, m, dim)))
    table = torch.randn((c["buckets"], heads), generator=gen).to(c["table_dtype"])
    key, query = torch.arange(n), torch.arange(m)
    start = c["start"]
    position = (torch.tensor(start)[:, None] + query if isinstance(start, (list, tuple)) else start + query[None])      # [batch or 1, m]
    if c["pairs"]:
        index = torch.randint(0, c["buckets"], (m, n), generator=gen)
        bucket, plan = index[None], (lambda: RelativeBuckets.from_index(index.to(device)))
    else:
        reach = 6
        line = torch.randint(0, c["buckets"], (2 * reach + 2,), generator=gen)
        line[-1] = c["buckets"] - 1
        bucket = line[(key[None, None] - position[..., None] + reach).clamp(0, 2 * reach + 1)]
        plan = lambda: RelativeBuckets.by_distance(line.to(device), -reach)      # noqa: E731
    allowed = added = mask = None
    if c["mask"] == "bool":
        mask = torch.rand((batch, 1, m, n), generator=gen) < 0.6
        mask[0, 0, 0] = False                            # a query that sees nothing
        allowed = mask
    elif c["mask"] == "key":                             # [m or 1, n]
        mask = torch.rand((1, n), generator=gen) < 0.7
        allowed = mask
    elif c["mask"] == "none":
        mask = torch.zeros((m, n), dtype=torch.bool)
        allowed = mask
    elif c["mask"] == "windows":                         # [period, m, n], additive
        mask = (torch.rand((max(1, batch // 2), m, n), generator=gen) < 0.3).float() * -100.0
        added = mask[torch.arange(batch) % mask.shape[0]][:, None].double()
    elif c["mask"] == "heads":
        mask = torch.randn((1, heads, m, n), generator=gen)
        added = mask.double()
    elif c["mask"] == "lowest":                          # a row of nothing but the type's lowest value
        mask = torch.zeros((m, n), dtype=c["dtype"])
        mask[:, ::2] = torch.finfo(c["dtype"]).min
        mask[0] = torch.finfo(c["dtype"]).min
        added = mask.double()
    elif c["mask"] == "infinite":
        mask = torch.zeros((m, n))
        mask[:, 1::2] = -torch.inf
        mask[-1] = -torch.inf
        added = mask.double()
    if c["causal"]:
        past = (key[None, None] <= position[..., None])[:, None]
        allowed = past if allowed is None else allowed & past
    if c["lengths"] is not None:
        used = (key[None] < torch.tensor(c["lengths"])[:, None])[:, None, None]
        allowed = used if allowed is None else allowed & used
        for b, u in enumerate(c["lengths"]):             # nothing behind the keys in use may matter
            k[b, :, max(u, 0):], v[b, :, max(u, 0):] = float("nan"), float("inf")
    scale = dim ** -0.5 if c["scale"] is None else c["scale"]
    k0, v0 = k.clone(), v.clone()
    if c["lengths"] is not None:
        k0, v0 = k0.nan_to_num(0.0, 0.0, 0.0), v0.nan_to_num(0.0, 0.0, 0.0)
        for b, u in enumerate(c["lengths"]):
            k0[b, :, max(u, 0):], v0[b, :, max(u, 0):] = 0.0, 0.0
    allowed = None if allowed is None else allowed.expand(batch, heads, m, n)
    added = None if added is None else added.expand(batch, heads, m, n)
    want = nn_oracle.attention(q, k0, v0, table, bucket, scale, allowed, added, grad if c["train"] else None, c["dtype"])
    on = lambda t: None if t is None else t.to(device)   # noqa: E731
    tensors = {"q": _layout(on(q), c["layout"]), "k": _layout(on(k), c["layout"]), "v": _layout(on(v), c["layout"]),
               "grad": _layout(on(grad), c["layout"]), "table": on(table)}
    options = {"scale": c["scale"], "mask": on(mask), "causal": c["causal"],
               "key_lengths": None if c["lengths"] is None else torch.tensor(c["lengths"], dtype=torch.int32).to(device),
               "query_start": torch.tensor(start, dtype=torch.int32).to(device) if isinstance(start, (list, tuple)) else start}
    return tensors, plan(), options, want


def check_attention(c, device):
    x, plan, options, want = make_attention(c, device)
    if not c["train"]:
        out = relative_attention(x["q"], x["k"], x["v"], x["table"], plan, **options)
        nn_oracle.close("out", out, want["out"])
        return out
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "table")]
    out = relative_attention(*leaves, plan, **options)
    nn_oracle.close("out", out, want["out"])
    for name, got in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, x["grad"])):
        nn_oracle.close(name, got, want[name], c["table_dtype"] if name == "dtable" else None)
    return out


def check_packed(c, device):
    x, plan, options, want = make_attention(c, device)
    options.pop("query_start")
    qkv = torch.stack([x["q"], x["k"], x["v"]], dim=0).permute(1, 3, 0, 2, 4).contiguous().requires_grad_(True)
    table = x["table"].requires_grad_(True)
    out = relative_attention_packed(qkv, table, plan, **options)
    b, n, _, heads, dim = qkv.shape
    nn_oracle.close("out", out.view(b, n, heads, dim).transpose(1, 2), want["out"])
    dqkv, dtable = torch.autograd.grad(out, (qkv, table), x["grad"].transpose(1, 2).reshape(b, n, heads * dim))
    for i, name in enumerate(("dq", "dk", "dv")):
        nn_oracle.close(name, dqkv[:, :, i].transpose(1, 2), want[name])
    nn_oracle.close("dtable", dtable, want["dtable"], c["table_dtype"])


ATTENTION_SMALL = {
    "one token": case(m=1),
    "one key": case(m=3, n=1, dtype=BF16),
    "odd pairs fp32": case(m=17, n=23, dim=24, batch=3),
    "odd pairs bf16": case(m=17, n=23, dim=40, dtype=BF16),
    "odd pairs fp16": case(m=9, n=70, dim=33, dtype=F16),
    "two tiles fp32": case(m=67, n=66, dim=32, batch=1, heads=1),
    "two tiles bf16": case(m=66, n=131, dim=64, batch=1, heads=1, dtype=BF16),
    "wide fp32": case(m=5, dim=128, batch=1),
    "wide bf16": case(m=5, dim=96, batch=1, dtype=BF16),
    "distance": case(m=13, n=21, pairs=False, start=3),
    "distance causal": case(m=19, pairs=False, causal=True, dtype=F16),
    "distance two tiles": case(m=70, n=75, pairs=False, causal=True, batch=1, heads=1, start=2),
    "behind every key": case(m=4, n=9, pairs=False, causal=True, start=-2),
    "shared heads": case(m=7, n=11, heads=6, kv=2, dtype=BF16),
    "one key head": case(m=3, n=5, heads=4, kv=1, pairs=False),
    "lengths": case(m=6, n=12, batch=4, lengths=[12, 5, 1, 0], pairs=False),
    "lengths bf16": case(m=6, n=70, batch=3, lengths=[70, 65, 3], dtype=BF16),
    "bool mask": case(m=9, n=10, mask="bool"),
    "key mask": case(m=9, n=10, mask="key", dtype=BF16),
    "sees nothing": case(m=4, n=6, mask="none"),
    "windows": case(m=16, batch=6, mask="windows"),
    "mask of heads": case(m=6, mask="heads", dtype=F16, heads=3),
    "lowest fp32": case(m=5, n=8, mask="lowest"),
    "lowest bf16": case(m=5, n=8, mask="lowest", dtype=BF16),
    "infinite": case(m=5, n=8, mask="infinite"),
    "tokens layout": case(m=10, n=12, layout="tokens", dtype=BF16),
    "padded layout": case(m=10, n=12, layout="padded", dim=30),
    "padded layout bf16": case(m=10, n=12, layout="padded", dim=32, dtype=BF16),
    "inner layout": case(m=10, n=12, layout="inner"),
    "table bf16": case(m=8, table_dtype=BF16),
    "negative scale": case(m=8, scale=-0.3),
    "many buckets": case(m=8, n=9, buckets=7000, heads=1, batch=1),
    "large scores": case(m=8, n=9, spread=6.0),
    "token against a cache": case(m=1, n=37, batch=3, heads=4, kv=2, pairs=False, lengths=[37, 20, 1], start=[36, 19, 0], train=False, dtype=BF16),
    "tokens at positions": case(m=3, n=37, batch=2, pairs=False, causal=True, lengths=[37, 30], start=[34, 27], train=False),
}


# ------------------------------------------------------------------------------------------------------------ distillation
def check_top(rows, classes, top, dtype, device, temperature=1.0, seed=0, kind="normal", stride=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, classes), generator=gen) * 3
    if kind == "equal":
        x = torch.full((rows, classes), 0.25)
    elif kind == "few values":
        x = torch.randint(-2, 3, (rows, classes), generator=gen).float()
        x[:, ::7] = -0.0
    elif kind == "infinite":
        x[:, ::3] = -torch.inf
        x[0] = -torch.inf
    elif kind == "rising":
        x = torch.arange(classes).float()[None].repeat(rows, 1) / classes
    elif kind == "nan":
        x[:, classes // 2] = torch.nan
    x = x.to(dtype)
    values, order, (rest, bound) = nn_oracle.top_logits(x, top, temperature, dtype)
    dev = x.to(device)
    if stride:
        room = torch.zeros((rows, classes + stride), dtype=dtype, device=device)
        room[:, :classes] = dev
        dev = room[:, :classes]
    got = top_logits(dev, top, temperature=temperature)
    assert torch.equal(got.classes.cpu(), order)
    assert torch.equal(got.values.cpu().double().nan_to_num(7e7), values.nan_to_num(7e7))
    inf = rest == -torch.inf
    assert torch.equal(got.rest.cpu().double() == -torch.inf, inf)
    if kind != "nan" or top > 1:
        ok = inf | ((got.rest.cpu().double() - rest).abs() <= bound) | (rest.isnan() & got.rest.cpu().isnan())
        assert ok.all(), (got.rest.cpu().double() - rest).abs().max()
    assert top_logits(dev, top, rest=False).rest is None


def distil_inputs(rows, classes, top, dtype, seed=0, rest=True, weighted=False, near=False, temperature=2.0):
    gen = torch.Generator().manual_seed(seed)
    base = torch.randn((rows, classes), generator=gen)
    teacher = base * 2 + torch.randn((rows, classes), generator=gen)
    values, order = torch.topk(teacher, top, dim=-1)
    left = None
    if rest:
        left = torch.logsumexp(teacher.scatter(1, order, -torch.inf) / temperature, -1)
    student = teacher + 0.01 * torch.randn((rows, classes), generator=gen) if near else base * 2 + torch.randn((rows, classes), generator=gen)
    weight = None
    if weighted:
        weight = torch.rand(rows, generator=gen) + 0.5
        weight[rows // 2:] = 0.0
        student[rows // 2:] = torch.nan                  # rows that do not count are not looked at
    return student.to(dtype), values, order, left, weight


def check_distil(rows, classes, top, dtype, device, temperature=2.0, rest=True, weighted=False, near=False, seed=0, int32=False, stride=0,
                 change=None, reduction="mean"):
    student, values, order, left, weight = distil_inputs(rows, classes, top, dtype, seed, rest, weighted, near, temperature)
    if change is not None:
        student, values, order, left, weight = change(student, values, order, left, weight)
    total = float(rows) if weight is None else float(weight.double().sum())
    by = 1.0 if reduction != "mean" else 1.0 / total if total else 0.0
    (loss, loss_bound), (grad, grad_bound) = nn_oracle.distillation(student, values, order, left, temperature, weight, dtype, torch.full((rows,), by))
    on = lambda t: None if t is None else t.to(device)   # noqa: E731
    answers = TopLogits(on(values), on(order.int() if int32 else order), on(left), temperature)
    x = on(student)
    if stride:
        room = torch.zeros((rows, classes + stride), dtype=dtype, device=device)
        room[:, :classes] = x
        x = room[:, :classes]
    x.requires_grad_(True)
    got = distillation_loss(x, answers, weight=on(weight), reduction=reduction)
    (dx,) = torch.autograd.grad(got, x, torch.ones_like(got) if reduction == "none" else None)
    if reduction == "none":
        nn_oracle.close("loss", got, (loss, loss_bound))
    else:
        nn_oracle.close("loss", got, (loss.sum() * by, loss_bound.sum() * by + 2 * nn_oracle.U * loss.abs().sum() * by + 1e-30))
    nn_oracle.close("gradient", dx, (grad, grad_bound))
    if reduction != "none":
        both = distillation_loss_and_grad(x, answers, weight=on(weight), reduction=reduction)
        nn_oracle.close("loss of the one-pass form", both[0], (loss.sum() * by, loss_bound.sum() * by + 2 * nn_oracle.U * loss.abs().sum() * by + 1e-30))
        nn_oracle.close("gradient of the one-pass form", both[1], (grad, grad_bound))
    return got, dx


def _twice(s, v, c, r, w):
    c[:, 1] = c[:, 0]                                    # a class given twice counts with both masses
    return s, v, c, r, w


def _none(s, v, c, r, w):
    c[:, 1:] = -1
    c[0] = -1                                            # a row without any answer
    return s, v, c, r, w


def _minus_infinity(s, v, c, r, w):
    s[:, 0] = -torch.inf                                 # the student rules out a class that was not answered
    c[c == 0] = 1
    v[0, -1] = -torch.inf                                # the teacher rules out one it answers
    return s, v, c, r, w


def _nothing_counts(s, v, c, r, w):
    return s, v, c, r, torch.zeros_like(w)


DISTIL_ODD = {
    "twice": (dict(rows=3, classes=50, top=4, rest=True, change=_twice)),
    "twice without rest": (dict(rows=3, classes=50, top=4, rest=False, change=_twice)),
    "no answers": (dict(rows=3, classes=50, top=4, rest=True, change=_none)),
    "no answers without rest": (dict(rows=3, classes=50, top=4, rest=False, change=_none)),
    "minus infinity": (dict(rows=4, classes=60, top=5, rest=True, change=_minus_infinity)),
    "nothing counts": (dict(rows=4, classes=60, top=5, rest=True, weighted=True, change=_nothing_counts)),
    "nothing counts, sum": (dict(rows=4, classes=60, top=5, rest=True, weighted=True, change=_nothing_counts, reduction="sum")),
}


def check_distil_odd(name, device, dtype=F32):
    options = dict(DISTIL_ODD[name])
    rows, classes, top = (options.pop(k) for k in ("rows", "classes", "top"))
    check_distil(rows, classes, top, dtype, device, **options)


def check_class_out_of_range(device):
    """such a row's loss and gradient are NaN, its neighbours are not touched"""
    student, values, order, left, _ = distil_inputs(3, 40, 4, F32)
    order[1, 2] = 40
    answers = TopLogits(values.to(device), order.to(device), left.to(device), 2.0)
    x = student.to(device).requires_grad_(True)
    loss = distillation_loss(x, answers, reduction="none")
    (dx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert torch.equal(loss.isnan().cpu(), torch.tensor([False, True, False]))
    assert not dx[0].isnan().any() and dx[1].isnan().all() and not dx[2].isnan().any()
    got = distillation_loss_and_grad(x, answers)[1]
    assert got[1].isnan().all() and not got[0].isnan().any()


def check_differences(device):
    """the kernels' gradients against differences of the 64-bit definitions along a random direction: (f(x + h d) - f(x - h d)) / 2h
    is off by h^2 / 6 times a third derivative (of order 10 here) and 2^-52 |f| / h: below 1e-8 for h = 1e-5"""
    h = 1e-5
    c = case(m=11, n=13, heads=4, kv=2, pairs=False, causal=True, seed=3)
    x, plan, options, want = make_attention(c, device)
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v", "table")]
    grads = torch.autograd.grad(relative_attention(*leaves, plan, **options), leaves, x["grad"])
    gen = torch.Generator().manual_seed(5)
    key, query = torch.arange(13), torch.arange(11)
    allowed = (key[None] <= query[:, None]).expand(2, 4, 11, 13)
    line = plan.source.cpu()
    bucket = line[(key[None] - query[:, None] + 6).clamp(0, 13)][None]
    base = [t.detach().cpu().double() for t in leaves]
    for i, name in enumerate(("dq", "dk", "dv", "dtable")):
        d = torch.randn(base[i].shape, generator=gen).double()
        f = []
        for sign in (1, -1):
            moved = [b + sign * h * d if j == i else b for j, b in enumerate(base)]
            out = nn_oracle.attention(*moved, bucket, 32 ** -0.5, allowed, None, None, F32)["out"][0]
            f.append(float((out * x["grad"].cpu().double()).sum()))
        along = float((grads[i].detach().cpu().double() * d).sum())
        assert abs(along - (f[0] - f[1]) / (2 * h)) <= float((want[name][1] * d.abs()).sum()) + 1e-7, name
    student, values, order, left, _ = distil_inputs(4, 70, 5, F32, seed=9)
    answers = TopLogits(values.to(device), order.to(device), left.to(device), 2.0)
    (loss, _), (_, bound) = nn_oracle.distillation(student, values, order, left, 2.0, None, F32, torch.full((4,), 0.25))
    grad = distillation_loss_and_grad(student.to(device), answers)[1].cpu().double()
    d = torch.randn(student.shape, generator=gen).double()
    f = [nn_oracle.distillation(student.double() + s * h * d, values, order, left, 2.0, None, F32, torch.full((4,), 0.25))[0][0].mean() for s in (1, -1)]
    assert abs(float((grad * d).sum()) - float(f[0] - f[1]) / (2 * h)) <= float((bound * d.abs()).sum()) + 1e-7


def check_few_keys(dtype, device):
    """two keys whose values are neighbours in `dtype`: dp_j - sum p dp is of the order of one step of the values, so dq's kernel must
    not take that sum from the rounded output.  With t half a step of dtype and U of fp32: ds is off by t |ds| from its rounding, by
    p 2 rel |dp_0 - dp_1| from probabilities off by rel = 2 (dim + 4) U size + 16 U each, and by p 2 (dim + 8) U |grad| . |v| from dp and
    its sum; dq by those over |k|, and by t |dq| from its own rounding."""
    gen = torch.Generator().manual_seed(11)
    m, dim, U, t = 70, 32, 2.0 ** -24, nn_oracle.half_step(dtype)
    q, grad = (torch.randn(2, 3, m, dim, generator=gen).to(dtype) for _ in range(2))
    k = torch.randn(2, 3, 2, dim, generator=gen).to(dtype)
    first = torch.rand(2, 3, 1, dim, generator=gen).add(1.0).to(dtype)
    v = torch.cat([first, (first.float() + 2 * t).to(dtype)], 2)          # in [1, 2): the next value
    table = torch.randn(4, 3, generator=gen)
    index = torch.randint(0, 4, (m, 2), generator=gen)
    leaves = [x.to(device).requires_grad_(True) for x in (q, k, v)]
    out = relative_attention(*leaves, table.to(device), RelativeBuckets.from_index(index.to(device)))
    (dq,) = torch.autograd.grad(out, leaves[:1], grad.to(device))
    q, k, v, grad = (x.double() for x in (q, k, v, grad))
    scale = dim ** -0.5
    bias = table.double()[index].movedim(-1, 0)
    size = (q.abs() @ k.abs().transpose(-2, -1) * scale + bias.abs()).amax(-1, keepdim=True)
    p = (q @ k.transpose(-2, -1) * scale + bias).softmax(-1)
    dp = grad @ v.transpose(-2, -1)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    rel = 2 * (dim + 4) * U * size + 16 * U
    apart = (dp[..., :1] - dp[..., 1:]).abs()
    off = t * ds.abs() + p * (2 * rel * apart + 2 * (dim + 8) * U * (grad.abs() @ v.abs().transpose(-2, -1)).amax(-1, keepdim=True))
    want = ds @ k * scale
    assert ((dq.cpu().double() - want).abs() <= 1.01 * (off @ k.abs() * scale + t * want.abs())).all()


def check_broadcast_inputs(device):
    """inputs expanded over the batch (stride 0): read as they are, their gradients summed by autograd"""
    gen = torch.Generator().manual_seed(1)
    q, k, grad = (torch.randn(s, generator=gen).to(device) for s in ((3, 2, 6, 32), (1, 2, 9, 32), (3, 2, 6, 32)))
    v, table = torch.randn((1, 2, 9, 32), generator=gen).to(device), torch.randn((5, 2), generator=gen).to(device)
    plan = RelativeBuckets.from_index(torch.randint(0, 5, (6, 9), generator=gen).to(device))
    results = []
    for copy in (False, True):
        kk, vv = k.clone().requires_grad_(True), v.clone().requires_grad_(True)
        ke, ve = kk.expand(3, -1, -1, -1), vv.expand(3, -1, -1, -1)
        out = relative_attention(q, ke.contiguous() if copy else ke, ve.contiguous() if copy else ve, table, plan)
        results.append((out,) + torch.autograd.grad(out, (kk, vv), grad))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def check_empty(device):
    """no sequence, no query, no key, no row"""
    table = torch.zeros((3, 2), device=device, requires_grad=True)
    plan = RelativeBuckets.by_distance(torch.tensor([0, 1, 2]).to(device), -1)
    for batch, m, n in ((0, 4, 5), (2, 0, 5), (2, 4, 0)):
        q = torch.randn(batch, 2, m, 16, device=device, requires_grad=True)
        k, v = (torch.randn(batch, 2, n, 16, device=device, requires_grad=True) for _ in range(2))
        out = relative_attention(q, k, v, table, plan)
        assert out.shape == q.shape and not out.any()
        for g, t in zip(torch.autograd.grad(out, (q, k, v, table), torch.ones_like(out)), (q, k, v, table)):
            assert g.shape == t.shape and not g.any()
    assert len(top_logits(torch.empty(0, 9, device=device), 3)) == 0
    x = torch.empty(0, 9, device=device, requires_grad=True)
    answers = top_logits(x, 3)
    loss = distillation_loss(x, answers)
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss, x)[0].shape == x.shape
    assert float(distillation_loss_and_grad(x, answers)[0]) == 0.0
