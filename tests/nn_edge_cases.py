"""Calls of the operators in transferattack_amd.relative / .distill that nn_cases does not make, shared by the host tier and the GPU
tier: the same functions, the device given by the caller.

Bounds are counted as in nn_oracle: u = 2^-24 is half a step of fp32, t half a step of the tensors' type."""
import pytest
import torch

import nn_oracle
from nn_cases import BF16, F16, F32, case, check_attention, make_attention  # noqa: F401
from transferattack_amd.distill import TopLogits, distillation_loss, distillation_loss_and_grad, top_logits
from transferattack_amd.relative import RelativeBuckets, relative_attention, relative_attention_packed

U = nn_oracle.U


def distil_rows_64(x, values, classes, rest, temperature):
    """-> loss [rows] and its gradient [rows, n] in 64 bits, from logarithms throughout (a share of a mass that underflows is kept), and
    what bounds them: w [rows, n], every other class's share of the others, and log q_R"""
    x, values = x.detach().cpu().double() / temperature, values.detach().cpu().double() / temperature
    bins = values if rest is None else torch.cat([values, rest.detach().cpu().double()[:, None]], 1)
    log_p = torch.log_softmax(bins, 1)
    log_q = torch.log_softmax(x, 1)
    answered = torch.zeros_like(x, dtype=torch.bool).scatter_(1, classes.cpu(), True)
    log_rest = log_q.masked_fill(answered, -torch.inf).logsumexp(1, keepdim=True)
    at = log_q.gather(1, classes.cpu())
    w = torch.softmax(x.masked_fill(answered, -torch.inf), 1).nan_to_num(0.0)      # (0: no other class; log_q - log_rest would lose log n beside a masking constant)
    p = log_p.exp()
    p_rest = torch.zeros_like(log_rest)
    if rest is not None:
        at, p_rest = torch.cat([at, log_rest], 1), p[:, -1:]
    loss = temperature ** 2 * torch.where(p > 0, p * (log_p - at), torch.zeros_like(p)).sum(1)
    grad = log_q.exp() - w * p_rest
    grad.scatter_add_(1, classes.cpu(), -p[:, :classes.shape[1]])
    return loss, temperature * grad, w, log_rest, p_rest


def check_masked_rest(dtype, masked, temperature, device):
    """a teacher whose classes but six are ruled out by a constant: the answers take those six and two of the others, and what is left is
    the constant's: log 290 + masked / T.  The logarithm of a sum of 290 exponentials of 0, whose error is 2 u of each, and the
    result's rounding, u"""
    gen = torch.Generator().manual_seed(0)
    x = torch.full((3, 298), masked, dtype=torch.float64).to(dtype)
    x[:, 5:11] = torch.randn(3, 6, generator=gen).to(dtype)
    got = top_logits(x.to(device), 8, temperature=temperature)
    want = x[0, 0].double() / temperature + torch.tensor(290.0).double().log()
    assert torch.equal(got.classes.cpu()[:, 6:], torch.tensor([[0, 1]]).expand(3, 2))
    assert ((got.rest.cpu().double() - want).abs() <= 4 * U + U * want.abs()).all(), (got.rest, want)


def check_masked_student(dtype, masked, temperature, rest, device):
    """a student that rules out every class not answered by a constant, in both forms.  The sum of the others (292 exponentials of 0) is
    off by 4 u at most, and so is each one's share; what concerns the answers is 64-bit, and rounded to 32 bits once or twice"""
    gen = torch.Generator().manual_seed(1)
    rows, n, top = 3, 300, 8
    x = torch.full((rows, n), masked, dtype=torch.float64).to(dtype)
    classes = torch.stack([torch.randperm(n, generator=gen)[:top] for _ in range(rows)])
    x.scatter_(1, classes, torch.randn(rows, top, generator=gen).to(dtype))
    values = torch.randn(rows, top, generator=gen)
    left = torch.full((rows,), -3.0) if rest else None
    loss, grad, w, log_rest, p_rest = distil_rows_64(x, values, classes, left, temperature)
    answers = TopLogits(values.to(device), classes.to(device), None if left is None else left.to(device), temperature)
    xx = x.to(device).requires_grad_(True)
    got = distillation_loss(xx, answers, reduction="sum")
    (dx,) = torch.autograd.grad(got, xx)
    both = distillation_loss_and_grad(xx, answers, reduction="sum")
    t = nn_oracle.half_step(dtype)
    # a class answered: q off by 2 u (1 / Z kept in 32 bits); any other: its share by 8 u, and the smallest number of the type
    off = temperature * (2 * U + 8 * U * w * p_rest) + (t + 2 * U) * grad.abs() + float(torch.finfo(dtype).smallest_normal) * 2 * t
    for l, g in ((got, dx), both):
        assert abs(float(l.detach()) - float(loss.sum())) <= 8 * U * float(loss.abs().sum()) + 8 * U * temperature ** 2, (float(l.detach()), float(loss.sum()))
        assert ((g.cpu().double() - grad).abs() <= off).all(), (g.cpu().double() - grad).abs().max()


MASKING = [(F32, -1e10), (F32, -1e20), (F32, -1e30), (F32, torch.finfo(F32).min), (BF16, -1e10), (BF16, torch.finfo(BF16).min),
           (F16, torch.finfo(F16).min)]


def check_top_repeats(rows, classes, top, dtype, device, turns=12):
    """the same answers, to the bit, whatever ran before and in whatever order a row's waves came"""
    gen = torch.Generator().manual_seed(2)
    x = (torch.randn(rows, classes, generator=gen) * 3).to(dtype).to(device)
    first = top_logits(x, top, temperature=2.0)
    want = nn_oracle.top_logits(x, top, 2.0, dtype)[2]
    assert ((first.rest.cpu().double() - want[0]).abs() <= want[1]).all()
    for _ in range(turns):
        got = top_logits(x, top, temperature=2.0)
        assert torch.equal(got.values, first.values) and torch.equal(got.classes, first.classes)
        assert torch.equal(got.rest, first.rest), int((got.rest != first.rest).sum())


REPEATED = [(2351, 1541, 55, F32), (325, 4721, 11, BF16), (900, 1000, 64, F32), (700, 30000, 40, F16)]


def check_changed_before_backward(device):
    """what a backward pass reads again is kept as autograd keeps its inputs: changed in between, it raises instead of mixing old and new"""
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(2, 2, 70, 16, generator=gen).to(device).requires_grad_(True)
    table = torch.randn(5, 2, generator=gen).to(device)
    line = RelativeBuckets.by_distance(torch.arange(5).to(device), -2)
    lengths, start = torch.tensor([10, 20], dtype=torch.int32).to(device), torch.tensor([0, 3], dtype=torch.int32).to(device)
    mask, added = torch.ones(70, 70, dtype=torch.bool).to(device), torch.zeros(2, 70, 70).to(device)
    for name, changed in (("key_lengths", lengths), ("query_start", start), ("mask", mask), ("mask", added)):
        out = relative_attention(q, q, q, table, line, **{name: changed})
        changed.add_(1) if changed.dtype != torch.bool else changed.zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
    qkv = torch.randn(2, 70, 3, 2, 16, generator=gen).to(device).requires_grad_(True)
    out = relative_attention_packed(qkv, table, line, mask=added, key_lengths=lengths)
    lengths.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    x = torch.randn(3, 40, generator=gen).to(device).requires_grad_(True)
    values, classes, rest, weight = (torch.randn(3, 4, generator=gen).to(device), torch.arange(12).view(3, 4).to(device), torch.zeros(3).to(device),
                                     torch.ones(3).to(device))
    for changed in (values, classes, rest, weight):
        loss = distillation_loss(x, TopLogits(values, classes, rest, 2.0), weight=weight)
        changed.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def check_saved_tensor_hooks(device):
    """what is kept passes by saved-tensor hooks (offloading, checkpoints), the options' tensors too"""
    gen = torch.Generator().manual_seed(4)
    q, table = torch.randn(2, 2, 9, 16, generator=gen).to(device).requires_grad_(True), torch.randn(5, 2, generator=gen).to(device)
    plan = RelativeBuckets.by_distance(torch.arange(5).to(device), -2)
    lengths, mask = torch.tensor([9, 4], dtype=torch.int32).to(device), torch.zeros(9, 9).to(device)
    x, answers = torch.randn(3, 40, generator=gen).to(device).requires_grad_(True), TopLogits(torch.zeros(3, 2).to(device), torch.tensor([[0, 1]] * 3).to(device))
    weight = torch.ones(3).to(device)
    steps = (lambda: torch.autograd.grad(relative_attention(q, q, q, table, plan, mask=mask, key_lengths=lengths).sum(), q)[0],
             lambda: torch.autograd.grad(distillation_loss(x, answers, weight=weight), x)[0])
    for step, kept in zip(steps, ((mask, lengths), (answers.values, answers.classes, weight))):
        seen = []
        plain = step()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.data_ptr()) or t.clone(), lambda t: t):
            assert torch.equal(step(), plain)
        assert {t.data_ptr() for t in kept} <= set(seen)


def check_made_in_inference_mode(device):
    """a teacher under torch.inference_mode, a mask and lengths made there: the student's step takes them, and has its own copy"""
    gen = torch.Generator().manual_seed(5)
    logits, q = torch.randn(3, 40, generator=gen).to(device), torch.randn(2, 2, 9, 16, generator=gen).to(device).requires_grad_(True)
    table, plan = torch.randn(5, 2, generator=gen).to(device), RelativeBuckets.by_distance(torch.arange(5).to(device), -2)
    x = torch.randn(3, 40, generator=gen).to(device).requires_grad_(True)
    with torch.inference_mode():
        answers, weight = top_logits(logits, 5), torch.ones(3, device=device)
        lengths, mask = torch.tensor([9, 4], dtype=torch.int32).to(device), torch.zeros(9, 9, device=device)
    plain = TopLogits(answers.values.clone(), answers.classes.clone(), answers.rest.clone())
    loss = distillation_loss(x, answers, weight=weight)
    out = relative_attention(q, q, q, table, plan, mask=mask, key_lengths=lengths)
    with torch.inference_mode():
        answers.values.zero_(), weight.zero_(), lengths.zero_()
    assert torch.equal(torch.autograd.grad(loss, x)[0], torch.autograd.grad(distillation_loss(x, plain, weight=torch.ones(3, device=device)), x)[0])
    want = relative_attention(q, q, q, table, plan, mask=mask.clone(), key_lengths=torch.tensor([9, 4], dtype=torch.int32).to(device))
    assert torch.equal(torch.autograd.grad(out.sum(), q)[0], torch.autograd.grad(want.sum(), q)[0])


def check_forward_mode(device):
    """tangents are refused where the tensor requires a gradient (by autograd) and where it does not"""
    import torch.autograd.forward_ad as fwd
    gen = torch.Generator().manual_seed(6)
    q, x = torch.randn(2, 9, 3, 2, 16, generator=gen).to(device), torch.randn(3, 40, generator=gen).to(device)
    table, plan = torch.randn(5, 2, generator=gen).to(device), RelativeBuckets.by_distance(torch.arange(5).to(device), -2)
    heads, weight = q[:, :, 0].transpose(1, 2).contiguous(), torch.ones(3).to(device)
    answers = top_logits(x, 3)
    attention = lambda q, k, v, t: relative_attention(q, k, v, t, plan)              # noqa: E731
    for needs in (False, True):
        with fwd.dual_level():
            dual = lambda t: fwd.make_dual(t.clone().requires_grad_(needs), torch.ones_like(t))      # noqa: E731
            for call in (lambda: attention(dual(heads), heads, heads, table), lambda: attention(heads, dual(heads), heads, table),
                         lambda: attention(heads, heads, dual(heads), table), lambda: attention(heads, heads, heads, dual(table)),
                         lambda: relative_attention_packed(dual(q), table, plan), lambda: relative_attention_packed(q, dual(table), plan),
                         lambda: distillation_loss(dual(x), answers), lambda: distillation_loss_and_grad(dual(x), answers)):
                with pytest.raises(RuntimeError):
                    call()
            attention(heads, heads, heads, table)        # no tangent among them: as ever
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            distillation_loss(x, answers, weight=fwd.make_dual(weight, weight))


def check_far_positions(device):
    """positions near either end of 32 bits take the ends of the distances, in every kernel: few queries, tiles, windows, both ways"""
    gen = torch.Generator().manual_seed(8)
    table = torch.randn(5, 2, generator=gen).to(device)
    low, high = -(1 << 31) + 1, (1 << 31) - 1
    for m, n, first in ((3, 70, -2), (70, 80, -2), (70, 80, -(1 << 30) + 1)):
        plan = RelativeBuckets.by_distance(torch.arange(5).to(device), first)
        q, k = (torch.randn(2, 2, t, 16, generator=gen).to(device).requires_grad_(True) for t in (m, n))
        for start, bucket in ((low, 4), (high, 0)):
            every = RelativeBuckets.from_index(torch.full((m, n), bucket).to(device))
            out = relative_attention(q, k, k, table, plan, query_start=torch.tensor([start, start], dtype=torch.int32).to(device))
            want = relative_attention(q, k, k, table, every)
            # the same scores plus the same constant: what differs is which kernel adds them up, some 100 roundings
            assert (out - want).abs().max() <= 200 * U * want.abs().max()
            for a, b in zip(torch.autograd.grad(out.square().sum(), (q, k)), torch.autograd.grad(want.square().sum(), (q, k))):
                assert (a - b).abs().max() <= 1000 * U * b.abs().max()
    plan = RelativeBuckets.by_distance(torch.arange(5).to(device), -(1 << 30) + 1)
    q = torch.randn(2, 2, 9, 16, generator=gen).to(device)
    got = relative_attention(q, q, q, table, plan, query_start=-(1 << 30) + 1)
    want = relative_attention(q, q, q, table, RelativeBuckets.from_index(torch.full((9, 9), 4).to(device)))
    assert torch.equal(got, want)


def check_64_bit_positions(device):
    """lengths and positions of 64 bits beyond what 32 hold: all keys, none, the ends of the distances"""
    gen = torch.Generator().manual_seed(7)
    q, k = torch.randn(4, 2, 3, 16, generator=gen).to(device), torch.randn(4, 2, 7, 16, generator=gen).to(device)
    table, plan = torch.randn(5, 2, generator=gen).to(device), RelativeBuckets.by_distance(torch.arange(5).to(device), -2)
    ints = lambda *v: torch.tensor(v).to(device)         # noqa: E731
    top = torch.iinfo(torch.int64).max
    got = relative_attention(q, k, k, table, plan, key_lengths=ints(top, 1 << 32, -(1 << 32) + 3, -top - 1))
    assert torch.equal(got, relative_attention(q, k, k, table, plan, key_lengths=ints(7, 7, 0, 0).int()))
    for causal in (False, True):
        got = relative_attention(q, k, k, table, plan, causal=causal, query_start=ints(top, 1 << 32, -(1 << 32) + 3, -top - 1))
        assert torch.equal(got, relative_attention(q, k, k, table, plan, causal=causal, query_start=ints(100, 100, -100, -100)))


def check_rows_of_answers(device):
    """a batch of answers indexed and iterated like a batch of labels"""
    answers = TopLogits(torch.arange(6.0).view(3, 2).to(device), torch.arange(6).view(3, 2).to(device), torch.arange(3.0).to(device), 2.0)
    parts = list(answers)
    assert len(parts) == 3 and all(len(p) == 1 and torch.equal(p.values, answers.values[i:i + 1]) and torch.equal(p.rest, answers.rest[i:i + 1])
                                   for i, p in enumerate(parts))
    assert torch.equal(answers[-1].values, answers[2].values) and torch.equal(answers[-3].values, answers[0].values)
    for at in (3, -4, 1 << 40):
        with pytest.raises(IndexError):
            answers[at]
    assert list(answers[:0]) == [] and len(answers[torch.tensor([True, False, True]).to(device)]) == 2 and len(answers[torch.tensor([2, 2]).to(device)]) == 2
    one, two, three = answers
    assert torch.equal(three.classes, answers[2:].classes)


# The attacks that take a victim's answers, checked against themselves: with one class answered and no mass for the others the
# loss at temperature 1 is -log q of that class, cross entropy on its label.
REFUSING = {"mig", "vaifgsm", "anda", "foolmix", "su", "everywhere", "adaea", "smer"}
ENSEMBLES = {"ens", "svre", "cwa", "adaea", "smer"}
SMALL = dict(epoch=1, num_neighbor=2, num_sample=3, num_scale=2, num_warping=2, num_spectrum=2, num_ens=2, transpoint=0, adv_steps=2, max_iter=2,
             num_sample_neighbor=2, num_sample_operator=2, K=2)


def attack_on_toys(name, device, **kw):
    import inspect
    import transferattack_amd as ta
    from transferattack_amd import backbones
    from transferattack_amd.utils import EnsembleModel, wrap_model
    base = ta.load_attack_class(name)
    models = [backbones.create("toy_cnn", seed=3 + i, verbose=False) for i in range(2 if name in ENSEMBLES else 1)]

    def load_model(self, model_name):
        wrapped = [wrap_model(m.eval().to(device)) for m in models]
        return EnsembleModel(wrapped) if name in ENSEMBLES else wrapped[0]

    kw = dict({k: v for k, v in SMALL.items() if k in inspect.signature(base.__init__).parameters}, **kw)
    cls = type("Toy" + base.__name__, (base,), {"load_model": load_model})
    return cls(model_name=["a", "b"] if name in ENSEMBLES else "injected", **kw)


def check_attack_on_answers(name, device):
    import random
    import numpy as np
    if name in REFUSING:
        with pytest.raises(Exception, match="Unsupported loss distillation|unexpected keyword argument 'loss'"):
            attack_on_toys(name, device, loss="distillation", **({"targeted": True} if name == "everywhere" else {}))
        return
    x = torch.randint(0, 256, (2, 3, 224, 224), generator=torch.Generator().manual_seed(0)).float() / 255
    label = torch.tensor([3, 7])
    answers = TopLogits(torch.zeros(2, 1), label[:, None])
    got = {}
    for loss, y in (("crossentropy", label), ("distillation", answers)):
        atk = attack_on_toys(name, device, loss=loss)
        torch.manual_seed(5), np.random.seed(5), random.seed(5)
        got[loss] = atk(x, y).cpu()
    a, b = got["crossentropy"], got["distillation"]
    assert float(b.abs().max()) > 0 and float(b.abs().max()) <= 16 / 255 + 1e-7
    # the two gradients are the same but for a few roundings of 2^-24: steps of the gradient's sign differ where it is within those of 0,
    # steps of its value by as much
    differ = float(((a - b).abs() > 1e-5).float().mean())
    assert differ <= 0.02, differ


def check_near_the_teacher(rest, twice, device):
    """a student within 1e-6 of its teacher: the gradients of the classes answered, q - p, are a millionth of either, and both forms have
    them to what the row's sums leave.  With every class answered all of it is 64-bit, and only the result is rounded.  With more
    classes the sum of the others is off by r = 200 u + (2 |x - m| / T + 4) u at most, so q by r q_R q, weighted like the terms"""
    gen = torch.Generator().manual_seed(10)
    rows, n = 4, 50
    top = 10 if rest else n
    teacher = torch.randn(rows, n, generator=gen, dtype=torch.float64)
    student = (teacher + 1e-6 * torch.randn(rows, n, generator=gen, dtype=torch.float64)).float()
    values, classes = torch.topk(teacher.float(), top, dim=1)
    left = teacher.float().double().scatter(1, classes, -torch.inf).logsumexp(1).float() if rest else None
    if twice:                                            # a class given twice, each time with half of its mass
        values[:, 1], classes[:, 1] = values[:, 0], classes[:, 0]
        values[:, :2] -= torch.tensor(2.0).log()
    loss, grad, w, log_rest, p_rest = distil_rows_64(student, values, classes, left, 1.0)
    q = torch.log_softmax(student.double(), 1).exp()
    away = (student.double().amax(1, keepdim=True) - student.double())
    r = 200 * U + ((2 * away + 4) * U * w).sum(1, keepdim=True) if rest or twice else torch.zeros(rows, 1, dtype=torch.float64)
    off = (r * log_rest.exp() * q + (r + (2 * away + 6) * U) * w * (log_rest.exp() + p_rest) * (w > 0) + 3 * U * grad.abs() + 1e-13)
    answers = TopLogits(values.to(device), classes.to(device), None if left is None else left.to(device), 1.0)
    x = student.to(device).requires_grad_(True)
    (dx,) = torch.autograd.grad(distillation_loss(x, answers, reduction="sum"), x)
    both = distillation_loss_and_grad(x, answers, reduction="sum")[1]
    for g in (dx, both):
        assert ((g.cpu().double() - grad).abs() <= off).all(), ((g.cpu().double() - grad).abs() / off).max()
    # the two forms have the same numbers of the classes answered, but for what 1 / Z kept in two parts leaves (2^-48) and one rounding
    at = classes.to(device)
    assert ((dx - both).gather(1, at).abs() <= 2 * U * both.gather(1, at).abs() + 1e-13).all()


def attention_64(q, k, v, grad, bias):
    """softmax(q k^T dim^-0.5 + bias) v and its gradients in 64 bits (every pair seen), with what the kernels' 32-bit arithmetic may leave at the
    steps of nn_oracle's docstring: scores, probabilities (rel), dp, delta and ds.  -> dict"""
    q, k, v, grad, bias = (x.detach().cpu().double() for x in (q, k, v, grad, bias))
    dim, n, m, scale = q.shape[-1], k.shape[-2], q.shape[-2], q.shape[-1] ** -0.5
    s = q @ k.transpose(-2, -1) * scale + bias
    size = q.abs() @ k.abs().transpose(-2, -1) * scale + bias.abs()
    p = s.softmax(-1)
    rel = 2 * (dim + 4) * U * size.amax(-1, keepdim=True) + 4 * U * (s.amax(-1, keepdim=True) - s).clamp(0, 200) + (n + 8) * U
    out, dp = p @ v, grad @ v.transpose(-2, -1)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dp_err = (dim + 4) * U * (grad.abs() @ v.abs().transpose(-2, -1))
    delta_err = (p * (rel + n * U) * dp.abs() + p * dp_err).sum(-1, keepdim=True)
    ds_err = p * rel * (dp - delta).abs() + p * (1 + rel) * (dp_err + delta_err) + 2 * U * p * (dp.abs() + delta.abs()) + 2.0 ** -120
    return dict(q=q, k=k, v=v, grad=grad, p=p, rel=rel, out=out, ds=ds, ds_err=ds_err, scale=scale, n=n, m=m, dim=dim,
                dq=ds @ k * scale, dk=ds.transpose(-2, -1) @ q * scale, dv=p.transpose(-2, -1) @ grad)


def dq_bound(x, t, smallest=0.0, of_terms=None):
    """of dq where ds is rounded once (t of it) and delta is sum p dp: the delta that ds is formed with is out . grad, off by what out is
    rounded by twice (its probabilities, itself); put right it leaves that times t, of ds and of p.  `smallest`: half a step of the
    type's smallest numbers, for the result; `of_terms`: what ds is rounded by, if not t"""
    of_terms = t if of_terms is None else of_terms
    out_err = (x["p"] * (x["rel"] + t + x["n"] * U)) @ x["v"].abs() + t * x["out"].abs()
    apart = (out_err * x["grad"].abs()).sum(-1, keepdim=True) + (x["dim"] + 4) * U * (x["out"] * x["grad"]).abs().sum(-1, keepdim=True)
    terms = x["ds_err"] + (of_terms + x["n"] * U) * x["ds"].abs() + (2 * t + x["n"] * U) * x["p"] * apart
    return terms @ x["k"].abs() * x["scale"] + (t + 2 * U) * x["dq"].abs() + smallest


def check_dq_of_few_heavy_keys(dtype, pairs, spread, device):
    """200 keys of which a few hold a row's mass (queries `spread` times as large): dp - delta of those nearly cancels, so delta must not
    come from the rounded output"""
    gen = torch.Generator().manual_seed(12)
    m, n, dim = 70, 200, 64
    q, k, v, grad = (torch.randn(1, 2, t, dim, generator=gen) for t in (m, n, n, m))
    q, k, v, grad = (t.to(dtype) for t in (q * spread, k, v, grad))
    table = torch.randn(5, 2, generator=gen)
    if pairs:
        index = torch.randint(0, 5, (m, n), generator=gen)
        plan = RelativeBuckets.from_index(index.to(device))
    else:
        index = (torch.arange(n)[None] - torch.arange(m)[:, None] + 2).clamp(0, 4)
        plan = RelativeBuckets.by_distance(torch.arange(5).to(device), -2)
    leaf = q.to(device).requires_grad_(True)
    out = relative_attention(leaf, k.to(device), v.to(device), table.to(device), plan)
    (dq,) = torch.autograd.grad(out, leaf, grad.to(device))
    x = attention_64(q, k, v, grad, table[index].movedim(-1, 0))
    off, bound = (dq.cpu().double() - x["dq"]).abs(), dq_bound(x, nn_oracle.half_step(dtype), 2.0 ** -25 if dtype == F16 else 0.0)
    assert (off <= bound).all(), (off / bound).max()


def attention_gradients(x, plan, table, device, **options):
    leaves = [t.to(device).requires_grad_(True) for t in (x["q"], x["k"], x["v"])]
    out = relative_attention(*leaves, table.to(device), plan, **options)
    return out, torch.autograd.grad(out, leaves, x["grad"].to(device))


def check_range_of_fp16(n, size, pairs, device):
    """gradients far from 1 and keys and queries that bring the results back into fp16's range: score gradients of `size` / n and less (below
    2^-14, or past 65504) are rounded by half a step of fp16 like any others.  Bounds: dq_bound; dk likewise, with the exact delta"""
    gen = torch.Generator().manual_seed(13)
    m, dim, t = 40, 32, nn_oracle.half_step(F16)
    q, k, v, grad = (torch.randn(1, 2, r, dim, generator=gen) for r in (m, n, n, m))
    # products q.k stay of order 1 while one of the two takes a factor, dq = sum ds k and dk = sum ds q stay near 1
    up = min(200.0, max(0.02, 10.0 / size))
    table = torch.randn(5, 2, generator=gen)
    if pairs:
        index = torch.randint(0, 5, (m, n), generator=gen)
        plan = RelativeBuckets.from_index(index.to(device))
    else:
        index = (torch.arange(n)[None] - torch.arange(m)[:, None] + 2).clamp(0, 4)
        plan = RelativeBuckets.by_distance(torch.arange(5).to(device), -2)
    for which in ("dq", "dk"):
        qq, kk = (q / up, k * up) if which == "dq" else (q * up, k / up)
        raw = {"q": qq.half(), "k": kk.half(), "v": (v * 30 if size > 1 else v).half(), "grad": (grad * size).half()}
        assert all(r.isfinite().all() for r in raw.values())
        out, grads = attention_gradients(raw, plan, table, device)
        x = attention_64(raw["q"], raw["k"], raw["v"], raw["grad"], table[index].movedim(-1, 0))
        got, want = dict(zip(("dq", "dk", "dv"), (g.cpu().double() for g in grads))), x
        smallest = 2.0 ** -25
        bounds = {"dq": dq_bound(x, t, smallest),
                  "dk": (x["ds_err"] + (t + m * U) * x["ds"].abs()).transpose(-2, -1) @ x["q"].abs() * x["scale"] + (t + 2 * U) * x["dk"].abs() + smallest,
                  "dv": (x["p"] * (x["rel"] + t + m * U)).transpose(-2, -1) @ x["grad"].abs() + t * x["dv"].abs() + smallest}
        for name in (which, "dv"):
            ok = want[name].abs() < 65504
            off = (got[name] - want[name]).abs()
            assert (off <= bounds[name])[ok].all(), (which, name, (off / bounds[name])[ok].max())


def check_many_equal_keys(n, device):
    """many equal probabilities below fp16's smallest normal number: their rounding, the same for all, would not average out.  Each is off
    by half a step of fp16 as any number is, t, and the result by as much once more; n u of the sums"""
    gen = torch.Generator().manual_seed(14)
    dim, t = 8, nn_oracle.half_step(F16)
    k, v = torch.zeros(1, 1, n, dim), (torch.rand(1, 1, n, dim, generator=gen) + 1.0).half()
    k[0, 0, 0] = 1.0                                     # one key e^12.3 above the others: what they are compared with (76.3 steps of 2^-24)
    plan = RelativeBuckets.from_index(torch.zeros(17, n, dtype=torch.int64).to(device))
    for m in (1, 17):
        q = torch.full((1, 1, m, dim), 12.3 * dim ** -0.5)
        raw = {"q": q.half(), "k": k.half(), "v": v, "grad": torch.ones(1, 1, m, dim).half()}
        here = plan if m == 17 else RelativeBuckets.from_index(torch.zeros(1, n, dtype=torch.int64).to(device))
        out, grads = attention_gradients(raw, here, torch.zeros(1, 1), device)
        x = attention_64(*(raw[r] for r in ("q", "k", "v", "grad")), torch.zeros(1, 1))
        off = (out.detach().cpu().double() - x["out"]).abs()
        assert (off <= (2 * t + (n + 400) * U) * x["out"]).all(), (off / x["out"]).max() / t
        dv = grads[2].cpu().double()
        assert ((dv - x["dv"]).abs() <= (2 * t + (n + 400) * U) * x["dv"] + 2.0 ** -25).all(), ((dv - x["dv"]).abs() / x["dv"]).max() / t


# ---- loops that go round more than once, and kernels that small cases do not reach
MANY = {
    "windows, five to a workgroup": case(m=5, batch=900, heads=4, dim=32),
    "windows in turn, bf16": case(m=9, batch=900, heads=4, dim=64, dtype=BF16),
    "windows with masks, two to a workgroup": case(m=16, batch=512, heads=8, dim=32, mask="windows"),
    "windows with masks, fp16": case(m=16, batch=512, heads=8, dim=32, mask="windows", dtype=F16),
    "windows by distance": case(m=7, n=12, batch=900, heads=4, pairs=False, causal=True, start=4),
    "table of distances": case(m=70, batch=300, heads=2, pairs=False, lengths=[(29 * i) % 71 for i in range(300)], dtype=BF16),
    "table of distances fp32": case(m=66, batch=300, heads=2, pairs=False, causal=True),
    "table of pairs": case(m=66, n=67, batch=256, heads=2, dtype=BF16, dim=64),
    "table of pairs, masked": case(m=66, n=67, batch=256, heads=2, dtype=F16, dim=64, mask="key"),
    "table of pairs, lengths": case(m=66, n=67, batch=256, heads=2, dtype=F16, lengths=[(31 * i) % 68 for i in range(256)]),
}
WIDE = ("table of pairs", "table of pairs, masked", "table of pairs, lengths")       # 32 queries to a wave, too: 16-bit pairs, 512 workgroups


def sequences_of_a_workgroup(c):
    """how many sequences share a part of the table's sums, from the workspace that the library asks for"""
    from transferattack_amd import _nn
    a = _nn.AttentionArgs()
    heads, m, n, batch = c["heads"], c["m"], c["n"] or c["m"], c["batch"]
    a.dtype, a.batch, a.heads, a.kv_heads, a.m, a.n, a.dim = _nn.DTYPES[c["dtype"]], batch, heads, c["kv"] or heads, m, n, c["dim"]
    a.buckets, a.distances, a.start, a.causal, a.dtable = c["buckets"], 0 if c["pairs"] else 14, c["start"], int(c["causal"]), 1
    a.first = -6
    if c["mask"] == "windows":
        a.mask_kind, a.mask_period = _nn.MASK_FLOAT, batch // 2
    elif c["mask"] == "key":
        a.mask_kind, a.mask_period = _nn.MASK_BOOL, 1
    a.key_lengths = None if c["lengths"] is None else 1
    floats = _nn.load().ta_nn_attention_workspace(a, 1) - batch * heads * m
    q_tiles, k_tiles = -(-m // 64), -(-n // 64)
    if c["pairs"]:
        return batch * m * n * heads / floats
    floats -= batch * heads * q_tiles * 2 + heads * (q_tiles + k_tiles - 1) * 128
    return batch * q_tiles * min(k_tiles, 3) * 128 * heads / floats


def check_many(name, device):
    c = MANY[name]
    assert sequences_of_a_workgroup(c) >= 2, sequences_of_a_workgroup(c)
    check_attention(c, device)


OTHER_BIASES = {
    "distances, bool mask": case(m=70, n=75, pairs=False, mask="bool", dtype=BF16),
    "distances, mask of heads": case(m=70, n=75, pairs=False, mask="heads", causal=True, lengths=[75, 40], kv=1),
    "distances, additive masks": case(m=66, n=66, pairs=False, mask="windows", batch=4, dtype=F16, dim=64),
    "distances, mask of infinities": case(m=40, n=70, pairs=False, mask="infinite", start=30),
    "few queries, distances, mask": case(m=2, n=90, pairs=False, mask="bool", kv=1, heads=4, start=60),
    "large table of pairs": case(m=66, n=70, buckets=7000, dtype=BF16),
}


def check_many_distances(dtype, m, n, causal, device):
    """a line of 9000 distances, each its own bucket for the most part: more than the kernels keep on the chip, so the table is read where it is"""
    gen = torch.Generator().manual_seed(16)
    batch, heads, dim, start = 2, 2, 32, n - m
    q, k, v, grad = (torch.randn(batch, heads, t, dim, generator=gen).to(dtype) for t in (m, n, n, m))
    line = torch.arange(9000) % 8500
    table = torch.randn(8500, heads, generator=gen)
    distance = torch.arange(n)[None] - torch.arange(m)[:, None] - start
    bucket = line[(distance + 4500).clamp(0, 8999)][None]
    allowed = (distance <= 0).expand(batch, heads, m, n) if causal else None
    want = nn_oracle.attention(q, k, v, table, bucket, dim ** -0.5, allowed, None, grad, dtype)
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, v, table)]
    plan = RelativeBuckets.by_distance(line.to(device), -4500)
    out = relative_attention(*leaves, plan, causal=causal, query_start=start)
    nn_oracle.close("out", out, want["out"])
    # (a result below 2^-14 is rounded by half a step of fp16's smallest numbers, 2^-25, not by a share of itself as the oracle counts)
    smallest = 2.0 ** -25 if dtype == F16 else 0.0
    for name, got in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, grad.to(device))):
        nn_oracle.close(name, got, (want[name][0], want[name][1] + (0.0 if name == "dtable" else smallest)), F32 if name == "dtable" else None)


def check_frozen_table(c, device):
    """a frozen surrogate: gradients of what it is given, none of its table -- the bits of the call that has both, packed and not"""
    x, plan, options, _ = make_attention(c, device)
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "v")]
    alone = torch.autograd.grad(relative_attention(*leaves, x["table"], plan, **options), leaves, x["grad"])
    table = x["table"].clone().requires_grad_(True)
    both = torch.autograd.grad(relative_attention(*leaves, table, plan, **options), leaves + [table], x["grad"])
    assert all(torch.equal(a, b) for a, b in zip(alone, both))
    (only,) = torch.autograd.grad(relative_attention(*[t.detach() for t in leaves], table, plan, **options), table, x["grad"])
    assert torch.equal(only, both[3])
    options.pop("query_start")
    qkv = torch.stack([t.detach() for t in leaves]).permute(1, 3, 0, 2, 4).contiguous().requires_grad_(True)
    (dqkv,) = torch.autograd.grad(relative_attention_packed(qkv, x["table"], plan, **options), qkv, x["grad"].transpose(1, 2).flatten(2))
    assert all(torch.equal(dqkv[:, :, i].transpose(1, 2), alone[i]) for i in range(3))


FROZEN = {
    "windows": case(m=49, batch=6, heads=3, dim=32, mask="windows"),
    "pairs bf16": case(m=70, batch=2, dim=64, dtype=BF16),
    "distances fp16": case(m=70, batch=2, pairs=False, causal=True, dtype=F16),
}


def check_no_rows(device):
    """a batch of no rows has the shape of one, and gradients"""
    x = torch.randn(0, 3, 9, device=device, requires_grad=True)
    answers = top_logits(x, 2)
    loss = distillation_loss(x, answers, reduction="none")
    assert loss.shape == (0, 3) and torch.autograd.grad(loss.sum(), x)[0].shape == x.shape
    for reduction in ("mean", "sum"):
        assert distillation_loss(x, answers, reduction=reduction).shape == () and distillation_loss_and_grad(x, answers, reduction=reduction)[1].shape == x.shape


def check_plan_keeps_its_buckets(device):
    """a plan never changes: not with the tensor it was made from, nor does its copy on another device"""
    index, line = torch.arange(12).view(3, 4).to(device), torch.arange(5).to(device)
    plans = RelativeBuckets.from_index(index), RelativeBuckets.by_distance(line, -2)
    q, k = torch.randn(1, 2, 3, 8, device=device), torch.randn(1, 2, 4, 8, device=device)
    table = torch.randn(12, 2, device=device)
    before = [relative_attention(q, k, k, table, p) for p in plans]
    index.zero_(), line.zero_()
    other = "cpu:0" if device == "cpu" else "cpu"        # (another device than "cpu" by name: made anew)
    for p, want in zip(plans, before):
        moved = p.to(other)
        assert torch.equal(moved.source.cpu(), torch.arange(12).view(3, 4) if p.shape else torch.arange(5))
        assert torch.equal(relative_attention(q, k, k, table, p), want)
        assert torch.equal(relative_attention(q, k, k, table, moved.to(device)), want)


SHORT = [(BF16, 5, 5, 3, 3, 32), (F16, 4, 4, 3, 3, 64), (BF16, 49, 49, 2, 2, 32), (F16, 64, 64, 2, 2, 64), (F16, 3, 9, 2, 2, 40),      # windows
         (BF16, 20, 30, 4, 2, 32), (F16, 2, 2, 4, 4, 128), (BF16, 16, 64, 8, 2, 72), (F16, 33, 12, 3, 3, 96), (BF16, 3, 3, 6, 1, 64)]  # tiles


def check_two_parts(dtype, m, n, heads, kv, dim, device):
    """over few terms probabilities and score gradients enter the products in two 16-bit parts, which leave t^2 of them: results are as far
    off as their own rounding, t, and 32-bit arithmetic allow"""
    gen = torch.Generator().manual_seed(17)
    t = nn_oracle.half_step(dtype)
    raw = {"q": torch.randn(2, heads, m, dim, generator=gen), "k": torch.randn(2, kv, n, dim, generator=gen), "v": torch.randn(2, kv, n, dim, generator=gen),
           "grad": torch.randn(2, heads, m, dim, generator=gen)}
    raw = {k: v.to(dtype) for k, v in raw.items()}
    table, index = torch.randn(5, heads, generator=gen), torch.randint(0, 5, (m, n), generator=gen)
    out, (dq, dk, dv) = attention_gradients(raw, RelativeBuckets.from_index(index.to(device)), table, device)
    group = heads // kv
    x = attention_64(raw["q"], raw["k"].repeat_interleave(group, 1), raw["v"].repeat_interleave(group, 1), raw["grad"], table[index].movedim(-1, 0))
    shared = lambda y: y.view(2, kv, group, n, dim).sum(2)                           # noqa: E731
    smallest = 2.0 ** -25 if dtype == F16 else 0.0
    terms = m * group * U
    want = {"out": x["out"], "dq": x["dq"], "dk": shared(x["dk"]), "dv": shared(x["dv"])}
    bound = {"out": (x["p"] * (x["rel"] + t * t + n * U)) @ x["v"].abs() + t * x["out"].abs(),
             "dq": dq_bound(x, t, 0.0, t * t),
             "dk": shared((x["ds_err"] + (t * t + terms) * x["ds"].abs()).transpose(-2, -1) @ x["q"].abs()) * x["scale"] + (t + 2 * U) * want["dk"].abs(),
             "dv": shared((x["p"] * (x["rel"] + t * t + terms)).transpose(-2, -1) @ x["grad"].abs()) + t * want["dv"].abs()}
    windows = m <= 64 and n <= 64 and dim <= 64 and heads == kv
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        if name == "out" and not windows and m * group > 16:
            continue                                     # (tiles' forward pass: one part)
        off = (got.detach().cpu().double() - want[name]).abs()
        assert (off <= bound[name] + smallest).all(), (name, (off / bound[name]).max())


def check_two_parts_token(dtype, n, device):
    gen = torch.Generator().manual_seed(18)
    t = nn_oracle.half_step(dtype)
    q, k, v = (torch.randn(2, h, r, 64, generator=gen).to(dtype) for h, r in ((8, 1), (2, n), (2, n)))
    table = torch.randn(5, 8, generator=gen)
    plan = RelativeBuckets.by_distance(torch.arange(5).to(device), -4)
    out = relative_attention(q.to(device), k.to(device), v.to(device), table.to(device), plan, query_start=n - 1)
    index = (torch.arange(n) - (n - 1) + 4).clamp(0, 4)[None]
    x = attention_64(q, k.repeat_interleave(4, 1), v.repeat_interleave(4, 1), torch.zeros_like(q), table[index].movedim(-1, 0))
    off = (out.cpu().double() - x["out"]).abs()
    bound = (x["p"] * (x["rel"] + t * t + n * U)) @ x["v"].abs() + t * x["out"].abs() + (2.0 ** -25 if dtype == F16 else 0.0)
    assert (off <= bound).all(), (off / bound).max()


def check_temperatures(device):
    """temperatures whose reciprocal 32 bits do not hold are refused; the outermost others give a distribution: the hottest all classes alike,
    the coldest the largest alone"""
    x, classes = torch.tensor([[3.0, -torch.inf, 1.0, 2.0, 2.5]]), torch.tensor([[0, 3]])
    for t in (2.0 ** -127, 1e-46, 2.0 ** 127, 1e300, 0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            top_logits(x.to(device), 2, temperature=t)
        with pytest.raises(ValueError, match="temperature"):
            TopLogits(x[:, :2].to(device), classes.to(device), None, t)
    hot, cold = top_logits(x.to(device), 2, temperature=2.0 ** 126), top_logits(x.to(device), 2, temperature=2.0 ** -100)
    assert abs(float(hot.rest) - float(torch.tensor(2.0).log())) <= 4 * U and float(cold.rest) == 2.0 ** 101
    for t in (2.0 ** 30, 2.0 ** -100):
        answers = TopLogits(torch.tensor([[3.0, 2.0]]).to(device), classes.to(device), None, t)
        loss, grad = distillation_loss_and_grad(x.to(device), answers, reduction="sum")
        assert torch.isfinite(loss) and torch.isfinite(grad).all() and float(grad[0, 1].abs()) == 0.0
