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
