"""nn_edge_cases on the GPU (libta_nn.so)."""
import pytest
import torch

import nn_edge_cases as edges
import transferattack_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("dtype,masked", edges.MASKING)
def test_masked_rest(dtype, masked, temperature):
    edges.check_masked_rest(dtype, masked, temperature, DEV)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("dtype,masked", edges.MASKING)
def test_masked_student(dtype, masked, temperature, rest):
    edges.check_masked_student(dtype, masked, temperature, rest, DEV)


@pytest.mark.parametrize("rows,classes,top,dtype", edges.REPEATED)
def test_top_logits_repeat(rows, classes, top, dtype):
    edges.check_top_repeats(rows, classes, top, dtype, DEV)


def test_changed_before_backward():
    edges.check_changed_before_backward(DEV)


def test_saved_tensor_hooks():
    edges.check_saved_tensor_hooks(DEV)


def test_made_in_inference_mode():
    edges.check_made_in_inference_mode(DEV)


def test_forward_mode():
    edges.check_forward_mode(DEV)


def test_far_positions():
    edges.check_far_positions(DEV)


def test_64_bit_positions():
    edges.check_64_bit_positions(DEV)


def test_rows_of_answers():
    edges.check_rows_of_answers(DEV)


@pytest.mark.parametrize("name", sorted(transferattack_amd.attack_zoo))
def test_attack_on_answers(name):
    edges.check_attack_on_answers(name, DEV)


@pytest.mark.parametrize("rest,twice", [(False, False), (True, False), (False, True), (True, True)])
def test_near_the_teacher(rest, twice):
    edges.check_near_the_teacher(rest, twice, DEV)


@pytest.mark.parametrize("spread", [1.0, 8.0])
@pytest.mark.parametrize("dtype,pairs", [(edges.BF16, True), (edges.BF16, False), (edges.F16, True), (edges.F16, False)])
def test_dq_of_few_heavy_keys(dtype, pairs, spread):
    edges.check_dq_of_few_heavy_keys(dtype, pairs, spread, DEV)


@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("size", [1e-6, 1e-4, 1e-2, 1e4])
@pytest.mark.parametrize("n", [40, 200])
def test_range_of_fp16(n, size, pairs):
    edges.check_range_of_fp16(n, size, pairs, DEV)


@pytest.mark.parametrize("n", [1000, 20000, 200000])
def test_many_equal_keys(n):
    edges.check_many_equal_keys(n, DEV)


@pytest.mark.parametrize("name", sorted(edges.MANY))
def test_many(name):
    edges.check_many(name, DEV)


@pytest.mark.parametrize("name", sorted(edges.OTHER_BIASES))
def test_other_biases(name):
    edges.check_attention(edges.OTHER_BIASES[name], DEV)


@pytest.mark.parametrize("dtype,m,n,causal", [(edges.F32, 70, 75, False), (edges.BF16, 70, 80, True), (edges.F16, 3, 90, True)])
def test_many_distances(dtype, m, n, causal):
    edges.check_many_distances(dtype, m, n, causal, DEV)


@pytest.mark.parametrize("name", sorted(edges.FROZEN))
def test_frozen_table(name):
    edges.check_frozen_table(edges.FROZEN[name], DEV)


def test_paths_of_the_cases():
    """the kernels that the cases above are there for are those that run: read from a trace"""
    names = set()
    for name in ("table of pairs", "table of pairs, masked", "windows with masks, two to a workgroup", "table of distances"):
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as trace:
            edges.check_attention(edges.MANY[name], DEV)
            torch.cuda.synchronize()
        names |= {e.name for e in trace.events()}
    print(sorted(n[:80] for n in names if "attention" in n or "window" in n))
    for want in ("attention_fwd<ta_nn::bf16, 64, 2, 1>", "attention_fwd<ta_nn::fp16, 64, 2, 2>", "window_fwd<float, 32>", "window_bwd<float, 32>",
                 "attention_bwd_table<ta_nn::bf16, 32, 0>", "attention_distance_sums"):
        assert any(want in n for n in names), (want, sorted(names))


def test_no_rows():
    edges.check_no_rows(DEV)


def test_plan_keeps_its_buckets():
    edges.check_plan_keeps_its_buckets(DEV)


def test_plan_on_other_streams():
    """a plan made on one stream is ready for all: nothing of its making is still under way, and calls elsewhere see it whole"""
    side = torch.cuda.Stream()
    index = torch.randint(0, 5000, (2100, 2100), generator=torch.Generator().manual_seed(0)).to(DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        plan = edges.RelativeBuckets.from_index(index)
        assert side.query()
        line = edges.RelativeBuckets.by_distance(torch.arange(100000, device=DEV) % 7, -5)
        assert side.query()
    assert torch.equal(plan.order, torch.sort(index.flatten(), stable=True)[1].int()) and torch.equal(line.index.cpu(), (torch.arange(100000) % 7).int())


def test_window_transformer_made_in_inference_mode(monkeypatch):
    from transferattack_amd.backbones.timm_victims import WindowAttention
    monkeypatch.setenv("TA_RELATIVE_ATTENTION", "1")
    torch.manual_seed(0)
    with torch.inference_mode():
        layer = WindowAttention(32, 4, 2).to(DEV)
        x = torch.randn(6, 16, 32, device=DEV)
        got = layer(x)
        monkeypatch.setenv("TA_RELATIVE_ATTENTION", "0")
        want = layer(x)
    # both sum some 100 products in 32 bits, in another order
    assert (got - want).abs().max() <= 200 * edges.U * want.abs().max()


@pytest.mark.parametrize("dtype,m,n,heads,kv,dim", edges.SHORT)
def test_two_parts(dtype, m, n, heads, kv, dim):
    edges.check_two_parts(dtype, m, n, heads, kv, dim, DEV)


@pytest.mark.parametrize("dtype,n", [(edges.BF16, 300), (edges.F16, 1500)])
def test_two_parts_token(dtype, n):
    edges.check_two_parts_token(dtype, n, DEV)


def test_temperatures():
    edges.check_temperatures(DEV)
