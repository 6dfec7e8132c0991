"""Attention with a learned relative position bias and distillation from top logits on the GPU (libta_nn.so)."""
import pytest
import torch

import nn_cases as cases
import nn_oracle
from nn_cases import BF16, F16, F32, case

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("name", sorted(cases.ATTENTION_SMALL))
def test_attention_small(name):
    cases.check_attention(cases.ATTENTION_SMALL[name], DEV)


LARGE = {
    "windows fp32": case(m=49, batch=96, heads=3, dim=32, mask="windows", buckets=169),
    "windows bf16": case(m=49, batch=96, heads=3, dim=32, mask="windows", buckets=169, dtype=BF16),
    "windows of 64": case(m=64, batch=5, heads=4, dim=32, buckets=225),
    "grid fp32": case(m=196, batch=3, heads=4, dim=64, buckets=729),
    "grid fp16": case(m=197, batch=3, heads=4, dim=64, buckets=729, dtype=F16),
    "sequence bf16": case(m=333, batch=2, heads=4, kv=2, dim=64, pairs=False, lengths=[333, 200], dtype=BF16),
    "sequence fp32": case(m=301, batch=1, heads=2, dim=96, pairs=False, causal=True),
    "sequence fp16": case(m=513, batch=1, heads=3, kv=1, dim=128, pairs=False, causal=True, dtype=F16),
    "wide fp32": case(m=130, batch=1, heads=2, dim=128, pairs=False),
    "few queries many keys": case(m=5, n=3000, batch=2, heads=4, kv=2, dim=80, pairs=False, start=2990, causal=True, dtype=BF16),
    "many queries few keys": case(m=1500, n=3, batch=2, heads=2, dim=32, pairs=False),
    "token bf16": case(m=1, n=5000, batch=3, heads=8, kv=2, dim=128, pairs=False, lengths=[5000, 1, 2777], start=[4999, 0, 2776], train=False, dtype=BF16),
    "token fp32": case(m=1, n=1029, batch=2, heads=3, dim=64, pairs=False, lengths=[1029, 0], start=[1028, 0], train=False),
    "token fp16": case(m=1, n=4097, batch=1, heads=12, dim=40, pairs=False, start=4096, train=False, dtype=F16),
}


@pytest.mark.parametrize("name", sorted(LARGE))
def test_attention_large(name):
    cases.check_attention(LARGE[name], DEV)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_packed(dtype):
    cases.check_packed(case(m=49, batch=8, heads=3, dim=32, dtype=dtype, buckets=169, mask="windows"), DEV)


@pytest.mark.parametrize("rows,classes,top,dtype,kind", [
    (3, 1, 1, F32, "normal"), (2, 37, 5, F32, "normal"), (33, 1000, 5, F32, "normal"), (2, 1100, 20, F32, "normal"),
    (1, 130, 130, F16, "normal"), (2, 2500, 3, F32, "equal"), (1, 2500, 900, BF16, "few values"), (2, 90, 40, F32, "infinite"),
    (1, 300, 9, F32, "rising"), (2, 50, 4, F32, "nan"), (5, 21841, 17, BF16, "normal"), (3, 65536, 64, BF16, "normal"),
    (2, 65537, 1024, F32, "normal"), (2, 140001, 100, BF16, "rising"), (2, 200000, 33, F16, "equal")])
def test_top_logits(rows, classes, top, dtype, kind):
    cases.check_top(rows, classes, top, dtype, DEV, temperature=2.0, kind=kind, stride=3 if classes in (37, 65536) else 0)


@pytest.mark.parametrize("rows,classes,top,dtype,options", [
    (3, 10, 2, F32, {}), (2, 37, 5, BF16, dict(stride=5)), (40, 1000, 7, F32, dict(weighted=True)), (9, 1100, 20, F16, dict(rest=False)),
    (2, 40, 40, F32, {}), (2, 40, 40, F32, dict(rest=False)), (30, 900, 4, F32, dict(near=True)), (3, 90, 1, F32, dict(near=True, rest=False)),
    (2, 64, 3, F32, dict(int32=True, reduction="sum")), (4, 64, 3, BF16, dict(reduction="none", weighted=True)), (1, 1, 1, F32, {}),
    (7, 21841, 17, F32, dict(weighted=True)), (6, 32768, 32, BF16, dict(stride=1)), (3, 65537, 1024, F16, {}), (2, 300001, 5, F32, {})])
def test_distillation(rows, classes, top, dtype, options):
    cases.check_distil(rows, classes, top, dtype, DEV, **options)
