"""nn_edge_cases where there is no GPU: the kernel sources compiled for the host, driven through the package's binding."""
import os
import subprocess
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "hipcpu_nn"))
import host_kernels                  # noqa: E402
import nn_edge_cases as edges        # noqa: E402
import nn_host_build                 # noqa: E402
import transferattack_amd            # noqa: E402


@pytest.fixture
def host(monkeypatch):
    nn_host_build.install(monkeypatch)


@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("dtype,masked", edges.MASKING)
def test_masked_rest(host, dtype, masked, temperature):
    edges.check_masked_rest(dtype, masked, temperature, "cpu")


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("dtype,masked", edges.MASKING)
def test_masked_student(host, dtype, masked, temperature, rest):
    edges.check_masked_student(dtype, masked, temperature, rest, "cpu")


def test_top_logits_repeat(host):
    edges.check_top_repeats(3, 1541, 55, edges.F32, "cpu", turns=1)


def test_changed_before_backward(host):
    edges.check_changed_before_backward("cpu")


def test_saved_tensor_hooks(host):
    edges.check_saved_tensor_hooks("cpu")


def test_made_in_inference_mode(host):
    edges.check_made_in_inference_mode("cpu")


def test_forward_mode(host):
    edges.check_forward_mode("cpu")


def test_far_positions(host):
    edges.check_far_positions("cpu")


def test_64_bit_positions(host):
    edges.check_64_bit_positions("cpu")


def test_rows_of_answers(host):
    edges.check_rows_of_answers("cpu")


def test_import_without_a_gpu_build_of_torch():
    """the package, its surrogates among it, imports where torch has no functions of a GPU"""
    code = ("import torch\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice', '_cuda_setDevice'):\n"
            "    hasattr(torch._C, n) and delattr(torch._C, n)\n"
            "import transferattack_amd.backbones, transferattack_amd.relative, transferattack_amd.distill, transferattack_amd.attack\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("name", sorted(transferattack_amd.attack_zoo))
def test_attack_on_answers(host, name, monkeypatch):
    host_kernels.install(monkeypatch)
    edges.check_attack_on_answers(name, "cpu")


@pytest.mark.parametrize("rest,twice", [(False, False), (True, False), (False, True), (True, True)])
def test_near_the_teacher(host, rest, twice):
    edges.check_near_the_teacher(rest, twice, "cpu")


@pytest.mark.parametrize("spread", [1.0, 8.0])
@pytest.mark.parametrize("dtype,pairs", [(edges.BF16, True), (edges.BF16, False), (edges.F16, True), (edges.F16, False)])
def test_dq_of_few_heavy_keys(host, dtype, pairs, spread):
    edges.check_dq_of_few_heavy_keys(dtype, pairs, spread, "cpu")


@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("size", [1e-6, 1e-4, 1e-2, 1e4])
@pytest.mark.parametrize("n", [40, 200])
def test_range_of_fp16(host, n, size, pairs):
    edges.check_range_of_fp16(n, size, pairs, "cpu")


@pytest.mark.parametrize("n", [20000])
def test_many_equal_keys(host, n):
    edges.check_many_equal_keys(n, "cpu")


@pytest.mark.parametrize("name", ["windows, five to a workgroup", "table of distances", "table of pairs, masked"])      # (the others: 1 to 50 s each here)
def test_many(host, name):
    edges.check_many(name, "cpu")


@pytest.mark.parametrize("name", sorted(edges.OTHER_BIASES))
def test_other_biases(host, name):
    edges.check_attention(edges.OTHER_BIASES[name], "cpu")


@pytest.mark.parametrize("dtype,m,n,causal", [(edges.F32, 70, 75, False), (edges.BF16, 70, 80, True), (edges.F16, 3, 90, True)])
def test_many_distances(host, dtype, m, n, causal):
    edges.check_many_distances(dtype, m, n, causal, "cpu")


@pytest.mark.parametrize("name", sorted(edges.FROZEN))
def test_frozen_table(host, name):
    edges.check_frozen_table(edges.FROZEN[name], "cpu")


def test_workspace_of_bad_sizes():
    """the C entry that sizes the workspace is asked before the call checks anything: it answers 0, it does not divide by them"""
    from transferattack_amd import _nn
    good = dict(dtype=1, batch=3, heads=4, kv_heads=2, m=70, n=80, dim=32, buckets=5, distances=5, dtable=1)

    def floats(lib, backward, **change):
        a = _nn.AttentionArgs()
        for field, value in dict(good, **change).items():
            setattr(a, field, value)
        return lib.ta_nn_attention_workspace(a, backward)

    lib = _nn.load()
    assert floats(lib, 1) > 0 and floats(lib, 1, dtable=None) == 3 * 4 * 70
    low = -(1 << 31)
    for change in (dict(mask_kind=1, mask_period=0), dict(mask_kind=2, mask_period=-3), dict(mask_kind=9), dict(heads=0), dict(heads=3), dict(heads=low),
                   dict(kv_heads=0), dict(batch=0), dict(batch=low), dict(m=low), dict(n=0), dict(dim=0), dict(dim=200), dict(distances=-1),
                   dict(distances=low), dict(buckets=0), dict(dtype=7), dict(table_dtype=-1), dict(m=1 << 30), dict(q_sm=-1)):
        for backward in (0, 1):
            for size in ({}, dict(m=5, n=5)):
                assert floats(lib, backward, **dict(size, **change)) == 0, change


def test_sizes_past_32_bits(host):
    """tensors expanded to more than the library's sizes hold are refused, not cut to their lower 32 bits"""
    import torch
    from transferattack_amd.distill import TopLogits, distillation_loss, top_logits
    from transferattack_amd.relative import RelativeBuckets, relative_attention, relative_attention_packed
    many = (1 << 32) + 7
    line, table, q = RelativeBuckets.by_distance(torch.arange(5), -2), torch.zeros(5, 1), torch.randn(1, 1, 3, 8)
    long = torch.randn(1, 1, 1, 8).expand(1, 1, many, 8)
    for call in (lambda: relative_attention(q, long, long, table, line), lambda: relative_attention(long, q, q, table, line),
                 lambda: relative_attention(q.expand(many, 1, 3, 8), q.expand(many, 1, 3, 8), q.expand(many, 1, 3, 8), table, line),
                 lambda: relative_attention_packed(torch.randn(1, 1, 3, 1, 8).expand(1, many, 3, 1, 8), table, line)):
        with pytest.raises(ValueError, match="2.30"):
            call()
    x = torch.zeros(1, 1)
    for call in (lambda: top_logits(x.expand(1, many), 3), lambda: top_logits(x.expand(1, (1 << 30) + 1), 3),
                 lambda: distillation_loss(x.expand(1, many), TopLogits(torch.zeros(1, 1), torch.zeros(1, 1, dtype=torch.int64)))):
        with pytest.raises(ValueError, match="classes"):
            call()
    from transferattack_amd import _nn
    at = x.data_ptr()                                    # the C entry, whose sizes are 32-bit already
    assert _nn._lib.ta_nn_top_logits(at, 0, 1 << 31, 1, (1 << 31) - 1, 1, 1.0, at, at, None, None) == -1
    assert b"2^30" in _nn._lib.ta_nn_last_error()


def test_no_rows(host):
    edges.check_no_rows("cpu")


def test_plan_keeps_its_buckets(host):
    edges.check_plan_keeps_its_buckets("cpu")


def test_plan_of_a_window_transformer():
    """built once, again when a checkpoint replaces the index, and for models made in inference mode, whose tensors have no version"""
    import torch
    from transferattack_amd.backbones.timm_victims import WindowAttention
    for made in (torch.no_grad, torch.inference_mode):
        with made():
            layer = WindowAttention(32, 4, 2)
        plan = layer._buckets()
        assert layer._buckets() is plan and plan.shape == (16, 16)
        if made is torch.no_grad:
            layer.load_state_dict(layer.state_dict())
            assert layer._buckets() is not plan


@pytest.mark.parametrize("dtype,m,n,heads,kv,dim", edges.SHORT)
def test_two_parts(host, dtype, m, n, heads, kv, dim):
    edges.check_two_parts(dtype, m, n, heads, kv, dim, "cpu")


@pytest.mark.parametrize("dtype,n", [(edges.BF16, 300), (edges.F16, 1500)])
def test_two_parts_token(host, dtype, n):
    edges.check_two_parts_token(dtype, n, "cpu")


def test_temperatures(host):
    edges.check_temperatures("cpu")
