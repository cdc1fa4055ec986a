"""Steps over the cache in 8 bits kernel by kernel and from captured graphs: how attention shares out its work is chosen by the same numbers, so
a step's logits are the same bits whichever way it goes, with many heads, mixed steps and contexts that are shared out to workgroups."""
import random
import types

import pytest
import torch

from conftest import seeded_tokens


def spec_of(n_heads, n_kv_heads, dh, positions=4096):
    from denno_beta_amd.parts import DecoderSpec, LayerCall, LayerSpec
    E, p = 96, "L0."
    norm = lambda n: ("layernorm", dict(width=E, eps=1e-5, weight_name=n, bias_name=None))   # noqa: E731
    layer = LayerSpec(arrangement="pre_norm", parts=dict(
        norm1=norm(p + "n1"), norm2=norm(p + "n2"),
        mixer=("causal_attention", dict(width=E, n_heads=n_heads, n_kv_heads=n_kv_heads, head_dim=dh, scale=dh ** -0.5, qkv_weight=p + "qkv", qkv_bias=None,
                                        out_weight=p + "out", out_bias=None)),
        ffn=("dense_mlp", dict(width=E, inner=128, activation="gelu_tanh", up_weight=p + "up", up_bias=None, down_weight=p + "down", down_bias=None))))
    return DecoderSpec(vocab=61, width=E, max_positions=positions, token_table="tok", position=("rotary_pairs", dict(dims=dh, base=50.0, head_dim=dh)),
                       layers=[layer], run_order=[LayerCall(0, 0)], final_norm=norm("nf"))


def runner(spec, dtype, **more):
    from denno_beta_amd.config import EngineOptions
    from denno_beta_amd.engine import ModelRunner
    from denno_beta_amd.weights import draw_all
    t = draw_all(spec.param_specs(), 5, engine_dtype=dtype, device=torch.device("cuda:0"), stored=dtype)
    # (with weights of 0.02 attention hardly shows in the logits)
    t = {k: v * 8 if k.endswith(("qkv", "out")) else v for k, v in t.items()}
    return ModelRunner(spec, t, EngineOptions(**dict(dict(dtype=dtype, device="cuda:0", page_size=16, cache_tokens=8192, max_live=16, cache_dtype="float8"),
                                                     **more)))


def run(r, steps):
    """steps: [[(request, rows)]] -> the steps' logits, every row's."""
    from denno_beta_amd.engine.batch import StepEntry
    at, got = {}, []
    for step in steps:
        entries = []
        for rid, n in step:
            if rid not in at:
                r.start_request(rid)
                at[rid] = 0
            tokens = seeded_tokens(1000 + rid, at[rid] + n, 61)[at[rid]:]
            at[rid] += n
            entries.append(StepEntry(rid, tokens, list(range(n))))
        got.append(r.step(entries).cpu().clone())
    for rid in at:
        assert r.end_request(rid)
    return got


# 12 tokens beside a portion of 300 rows; 12 portions; a portion behind a long context, then two beside a single row, then single rows
MIXED = [[(i, 5 + 2 * i) for i in range(12)], [(i, 1) for i in range(12)] + [(12, 300)], [(i, 20 + i) for i in range(12)], [(i, 1) for i in range(13)]]
LONG = [[(0, 500)]] * 5 + [[(0, 40)], [(0, 9), (1, 7)], [(0, 1), (1, 33)], [(0, 3)], [(0, 1), (1, 1), (2, 1)], [(0, 1), (1, 1), (2, 1)]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,steps", [((25, 25, 64), MIXED), ((32, 8, 128), MIXED), ((4, 2, 64), LONG), ((8, 2, 128), LONG)],
                         ids=["mixed 25 of 64", "mixed 32 of 128", "long 4 of 64", "long 8 of 128"])
def test_the_same_bits_captured_and_kernel_by_kernel(dtype, heads, steps):
    spec = spec_of(*heads)
    want = run(runner(spec, dtype, use_graphs=False), steps)
    r = runner(spec, dtype)
    for turn in range(3):
        got = run(r, steps)
        torch.cuda.synchronize()
        x = torch.randn(64, 64, device="cuda:0")
        (x @ x).sum().item()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (turn, i, float((a - b).abs().max()))
    assert r.graphs.graphs and r.graphs.portions


# -- the numbers that both forms choose by ---------------------------------------------------------------------------------------

class ARunner:
    """What engine.graphs.DecodeGraphs asks of a runner here, without one."""

    def __init__(self, spec, dtype):
        self.model, self.runtime = spec.instantiate(), types.SimpleNamespace(act_dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [(25, 25, 64), (32, 8, 128), (4, 2, 64), (3, 1, 250)], ids=str)
def test_a_step_and_its_captured_form_have_one_plan(heads, dtype):
    from denno_beta_amd.engine.batch import StepEntry
    from denno_beta_amd.engine.graphs import DecodeGraphs, chosen_by, portion_bucket, portion_chosen_by, portion_context
    r = ARunner(spec_of(*heads), dtype)
    graphs, mixer, rng = DecodeGraphs(r), r.model.blocks[0].mixers()[0], random.Random(3)
    many = 0
    for _ in range(300):
        rows = [rng.choice([1, 1, 1, 2, 9, 40, 130, 300]) for _ in range(rng.choice([1, 2, 3, 12, 40]))]
        longest = int(max(rows) * (40000 / max(rows)) ** rng.random())
        entries = [StepEntry(i, [0] * n, []) for i, n in enumerate(rows)]
        by = chosen_by(entries, longest, 64, 40000)
        if all(n == 1 for n in rows):
            assert by[0] == by[1] >= len(rows) and by[2] >= longest and (by[2] % 256 == 0 or by[2] == 40000)
            continue
        bucket = portion_bucket(entries)
        if bucket is None:
            assert by is None
            continue
        T, S, _ = bucket
        least = graphs._same_plans(T, S, portion_context(longest))
        plan = mixer.plan_8_bits(*by, dtype)
        assert mixer.plan_8_bits(*portion_chosen_by(T, S, least), dtype) == plan
        assert least == 0 or mixer.plan_8_bits(*portion_chosen_by(T, S, least // 2 if least > 128 else 0), dtype) != plan
        many += plan[2] > 1
    assert many > 20 and len(set(graphs.contexts.values())) > 2


def test_contexts_in_powers_of_two():
    from denno_beta_amd.engine.graphs import portion_chosen_by, portion_context
    assert [portion_context(n) for n in (1, 127, 128, 255, 256, 1000, 1024, 30000)] == [0, 0, 128, 128, 256, 512, 1024, 16384]
    assert [portion_chosen_by(T, S, 7) for T, S in ((16, 1), (512, 1), (192, 1), (384, 16), (512, 512), (512, 2))] == [
        (16, 1, 7), (512, 4, 7), (192, 2, 7), (384, 16, 7), (512, 512, 7), (512, 4, 7)]


def test_a_step_behind_a_long_context_is_shared_out_as_in_a_direct_call():
    """32 rows of 32 heads of 128 behind 30,000 tokens: 8 shares, captured or not."""
    from denno_beta_amd.engine.graphs import portion_chosen_by, portion_context
    from denno_beta_amd.kernels import ops
    direct = ops.portions8_plan(32, 1, 30000, 32, 128, torch.bfloat16)
    assert direct == ops.portions8_plan(*portion_chosen_by(32, 1, portion_context(30000)), 32, 128, torch.bfloat16) and direct[2] == 8


@pytest.mark.parametrize("by", [(0, 1, 5), (1, 0, 5), (1, 1, -1), (1, 1), ()])
def test_numbers_that_cannot_be_are_refused(monkeypatch, by):
    from denno_beta_amd.kernels import ops
    from test_cache8 import attend_args, call_attend, host_checks_only
    with host_checks_only(monkeypatch), pytest.raises(ops.KernelError, match="chosen_by"):
        call_attend(attend_args(), chosen_by=by)
