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
