"""Attention with a learned relative position bias and distillation from top logits where there is no GPU: the kernel sources
compiled for the host (tests/hipcpu_nn), driven through the package's binding, and the refusals of the public functions."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "hipcpu_nn"))
import nn_cases as cases            # noqa: E402
import nn_host_build                # noqa: E402
from nn_cases import BF16, F16, F32  # noqa: E402


@pytest.fixture
def host(monkeypatch):
    nn_host_build.install(monkeypatch)


@pytest.mark.parametrize("name", sorted(cases.ATTENTION_SMALL))
def test_attention(host, name):
    cases.check_attention(cases.ATTENTION_SMALL[name], "cpu")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed(host, dtype):
    cases.check_packed(cases.case(m=9, heads=3, dim=32, dtype=dtype), "cpu")


@pytest.mark.parametrize("rows,classes,top,dtype,kind", [
    (3, 1, 1, F32, "normal"), (2, 37, 5, F32, "normal"), (2, 300, 7, BF16, "normal"), (2, 1100, 20, F32, "normal"),
    (1, 130, 130, F16, "normal"), (2, 2500, 3, F32, "equal"), (1, 2500, 900, BF16, "few values"), (2, 90, 40, F32, "infinite"),
    (1, 300, 9, F32, "rising"), (2, 50, 4, F32, "nan"), (1, 5000, 64, F16, "rising")])
def test_top_logits(host, rows, classes, top, dtype, kind):
    cases.check_top(rows, classes, top, dtype, "cpu", temperature=2.0, kind=kind, stride=3 if classes == 37 else 0)


@pytest.mark.parametrize("rows,classes,top,dtype,options", [
    (3, 10, 2, F32, {}), (2, 37, 5, BF16, dict(stride=5)), (4, 300, 7, F32, dict(weighted=True)), (2, 1100, 20, F16, dict(rest=False)),
    (2, 40, 40, F32, {}), (2, 40, 40, F32, dict(rest=False)), (3, 90, 4, F32, dict(near=True)), (3, 90, 1, F32, dict(near=True, rest=False)),
    (2, 64, 3, F32, dict(int32=True, reduction="sum")), (4, 64, 3, BF16, dict(reduction="none", weighted=True)), (1, 1, 1, F32, {})])
def test_distillation(host, rows, classes, top, dtype, options):
    cases.check_distil(rows, classes, top, dtype, "cpu", **options)


@pytest.mark.parametrize("name", sorted(cases.DISTIL_ODD))
def test_distillation_odd(host, name):
    cases.check_distil_odd(name, "cpu")


def test_class_out_of_range(host):
    cases.check_class_out_of_range("cpu")


def test_gradients_against_differences(host):
    cases.check_differences("cpu")


@pytest.mark.parametrize("dtype", [cases.BF16, cases.F16])
def test_few_keys(host, dtype):
    cases.check_few_keys(dtype, "cpu")


def test_broadcast_inputs(host):
    cases.check_broadcast_inputs("cpu")


def test_empty(host):
    cases.check_empty("cpu")


def test_logarithmic_buckets():
    """against the rule in exact fractions, and its parts: one bucket per near distance, the last from max_distance on"""
    from fractions import Fraction
    from transferattack_amd.relative import RelativeBuckets
    plan = RelativeBuckets.logarithmic(32, 128)
    line, first = plan.source.tolist(), plan.first
    assert (first, len(line), plan.buckets) == (-128, 257, 32)
    for d, b in zip(range(-128, 129), line):
        away, side = abs(d), 16
        want = away if away < 8 else 8 + max(t for t in range(8) if Fraction(away, 8) ** 8 >= 16 ** t)
        assert b == want + (side if d > 0 else 0), d
    causal = RelativeBuckets.logarithmic(32, 128, bidirectional=False)
    assert causal.source[128:].eq(0).all() and causal.source[:112].ge(16).all() and causal.source[112] == 16 and causal.buckets == 32


def test_refusals(host):
    """what the functions do not take is an error that says so, before anything is launched"""
    from transferattack_amd.distill import TopLogits, distillation_loss, distillation_loss_and_grad, top_logits
    from transferattack_amd.relative import RelativeBuckets, relative_attention, relative_attention_packed
    q, k = torch.randn(2, 4, 5, 16), torch.randn(2, 2, 7, 16)
    table, plan = torch.zeros(6, 4), RelativeBuckets.from_index(torch.arange(35).view(5, 7) % 6)
    line = RelativeBuckets.by_distance(torch.arange(6), -2)
    ok = dict(q=q, k=k, v=k, table=table, buckets=plan)
    relative_attention(**ok)
    for error, change in [
            (TypeError, dict(q=q.double())), (ValueError, dict(k=k.half(), v=k.half())), (ValueError, dict(q=q[0])),
            (ValueError, dict(k=k[:, :, :, :8])), (ValueError, dict(v=k[:, :, :6])), (ValueError, dict(k=k[:1], v=k[:1])),
            (ValueError, dict(q=torch.randn(2, 3, 5, 16))), (ValueError, dict(table=table[:5])), (ValueError, dict(table=table[:, :3])),
            (TypeError, dict(table=table.double())), (TypeError, dict(buckets=torch.zeros(5, 7))),
            (ValueError, dict(buckets=RelativeBuckets.from_index(torch.zeros(5, 6, dtype=torch.int64)))),
            (ValueError, dict(mask=torch.zeros(3, 5, 7))), (ValueError, dict(mask=torch.zeros(2, 3, 5, 7))), (ValueError, dict(mask=torch.zeros(7))),
            (ValueError, dict(mask=torch.zeros(0, 5, 7))), (ValueError, dict(mask=torch.zeros(5, 6))), (TypeError, dict(mask=torch.zeros(5, 7, dtype=torch.int32))),
            (ValueError, dict(mask=torch.zeros(5, 7, requires_grad=True))), (ValueError, dict(key_lengths=torch.tensor([7]))),
            (TypeError, dict(key_lengths=torch.tensor([7.0, 7.0]))), (ValueError, dict(query_start=torch.tensor([1, 2, 3]))),
            (ValueError, dict(query_start=1 << 30)),
            (ValueError, dict(buckets=line, table=torch.zeros(6, 4, requires_grad=True), query_start=torch.tensor([0, 1])))]:
        with pytest.raises(error):
            relative_attention(**dict(ok, **change))
    wide = torch.randn(1, 1, 3, 129)
    with pytest.raises(ValueError, match="129"):
        relative_attention(wide, wide, wide, torch.zeros(6, 1), line)
    with pytest.raises(ValueError):
        relative_attention_packed(torch.randn(2, 5, 2, 4, 16), table, line)
    for bad in (torch.zeros(0, 3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64), torch.zeros(2, 2), torch.tensor([[-1, 0]]), torch.tensor([[65536]])):
        with pytest.raises(ValueError):
            RelativeBuckets.from_index(bad)
    with pytest.raises(ValueError):
        RelativeBuckets.by_distance(torch.tensor([0, -1]), 0)
    with pytest.raises(ValueError):
        RelativeBuckets.logarithmic(2, 128)
    with pytest.raises(TypeError):
        RelativeBuckets()

    x, values, classes = torch.randn(3, 9), torch.randn(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    answers = TopLogits(values, classes)
    for args, kw in [((values.double(), classes), {}), ((values, classes.float()), {}), ((values, classes[:2]), {}), ((values[0], classes[0]), {}),
                     ((values, classes, torch.zeros(2)), {}), ((values, classes), dict(temperature=0.0)), ((values, classes), dict(temperature=float("nan"))),
                     ((torch.zeros(1, 1025), torch.zeros(1, 1025, dtype=torch.int64)), {})]:
        with pytest.raises((TypeError, ValueError)):
            TopLogits(*args, **kw)
    for bad in (lambda: distillation_loss(x, classes), lambda: distillation_loss(x[:2], answers), lambda: distillation_loss(x, answers, weight=torch.ones(2)),
                lambda: distillation_loss(x, answers, weight=torch.ones(3).half()), lambda: distillation_loss(x, answers, reduction="batch"),
                lambda: distillation_loss(x, answers, weight=torch.ones(3, requires_grad=True)), lambda: distillation_loss(x.double(), answers),
                lambda: distillation_loss_and_grad(x, answers, reduction="none"), lambda: top_logits(x, 0), lambda: top_logits(x, 10),
                lambda: top_logits(x, 2, temperature=-1.0), lambda: top_logits(torch.randn(3, 0), 1)):
        with pytest.raises((TypeError, ValueError)):
            bad()
    assert len(answers.repeat(3)) == 9 and len(answers[1:]) == 2 and len(answers[-1]) == 1 and answers.detach().clone().to("cpu").temperature == 1.0


def test_library_refuses_by_itself():
    """the C entry points check what the binding passes: an error code and a text, nothing is launched"""
    from transferattack_amd import _nn
    lib = _nn.load()
    a = _nn.AttentionArgs()
    assert lib.ta_nn_attention(None, None) == -1 and b"null" in lib.ta_nn_last_error()
    for field, value in (("batch", 1), ("heads", 3), ("kv_heads", 2), ("m", 4), ("n", 4), ("dim", 200)):
        setattr(a, field, value)
    assert lib.ta_nn_attention(a, None) == -1 and b"share" in lib.ta_nn_last_error()
    a.kv_heads = 3
    assert lib.ta_nn_attention(a, None) == -1 and b"200" in lib.ta_nn_last_error()
    a.dim, a.dtype = 32, 9
    assert lib.ta_nn_attention_backward(a, None) == -1 and b"type" in lib.ta_nn_last_error()
    assert lib.ta_nn_attention_workspace(None, 0) == 0
    assert lib.ta_nn_top_logits(None, 0, 0, 0, 0, 0, 0.0, None, None, None, None) == -1
    assert lib.ta_nn_distil(None, 0, 0, 0, 0, None, None, 0, 0, None, None, 1.0, 1.0, None, None, None, None, 0, None) == -1
    assert lib.ta_nn_distil_backward(None, 0, 0, 0, 0, None, None, 0, 0, None, None, 1.0, 1.0, None, None, 0, None, None, 0, None) == -1
    assert lib.ta_nn_distil_total(None, None, 0, 0, None, None, None) == -1


def test_no_cpu_fallback():
    from transferattack_amd import _hip
    from transferattack_amd.distill import top_logits
    from transferattack_amd.relative import RelativeBuckets, relative_attention
    q = torch.randn(1, 1, 2, 8)
    with pytest.raises(_hip.HipExtensionError, match="cpu"):
        relative_attention(q, q, q, torch.zeros(1, 1), RelativeBuckets.from_index(torch.zeros(2, 2, dtype=torch.int64)))
    with pytest.raises(_hip.HipExtensionError, match="cpu"):
        top_logits(torch.randn(2, 5), 2)


def test_abi_symbols_exported():
    """libta_nn.so exports what include/ta_nn.h declares, and the binding's structure has its fields in its order"""
    import re
    from transferattack_amd import _nn
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = open(os.path.join(root, "include", "ta_nn.h")).read()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    assert set(re.findall(r"\b(ta_nn_[a-z0-9_]+)\s*\(", header)) == set(_nn.SIGNATURES)
    lib = _nn.load()
    assert all(hasattr(lib, name) for name in _nn.SIGNATURES) and lib.ta_nn_abi_version() == _nn.ABI_VERSION == 1
    body = re.search(r"typedef struct ta_nn_attention_args \{(.*?)\} ta_nn_attention_args;", header, re.S).group(1)
    names = [n for line in body.split(";") for n in re.findall(r"\*?\s*(\w+)\s*(?=,|$)", line.strip())]
    assert names == [f[0] for f in _nn.AttentionArgs._fields_]


def test_attack_takes_answers(host, monkeypatch):
    """every attack's loss='distillation': answers in the place of labels, through clone / to / repeat / targeted"""
    from transferattack_amd.attack import Attack
    from transferattack_amd.distill import DistillationLoss, TopLogits, distillation_loss
    attack = object.__new__(Attack)
    attack.loss, attack.targeted, attack.device = attack.loss_function("distillation"), False, torch.device("cpu")
    assert isinstance(attack.loss, DistillationLoss)
    student, values, order, left, _ = cases.distil_inputs(3, 20, 4, F32)
    answers = TopLogits(values, order, left, 2.0)
    assert torch.equal(attack.get_loss(student, answers), distillation_loss(student, answers))
    attack.targeted = True
    assert torch.equal(attack.get_loss(student.repeat(2, 1), answers.repeat(2)), -distillation_loss(student.repeat(2, 1), answers.repeat(2)))
    with pytest.raises(Exception, match="Unsupported loss"):
        attack.loss_function("hinge")
