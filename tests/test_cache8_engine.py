"""The engine with its cache in 8 bits (EngineOptions.cache_dtype): the two operators together, as steps call them."""
import json

import pytest
import torch

import cache8_refs as R
import replay_util as U
from conftest import TINY, seeded_tokens

FP8 = torch.float8_e4m3fn
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(params=[pytest.param("host", id="host"), pytest.param("gpu", marks=pytest.mark.gpu, id="gpu")])
def device(request):
    if request.param == "host":
        with R.emulated():
            yield "cpu"
    else:
        yield "cuda:0"


def options(device, dtype="float32", cache_dtype="float8", **more):
    from denno_beta_amd.config import EngineOptions
    return EngineOptions(**dict(dict(dtype=dtype, device=device, page_size=16, cache_tokens=512, max_live=4, cache_dtype=cache_dtype), **more))


def turned_spec(layers=3):
    """Attention with turned queries and keys: neighbouring pairs by the model's encoding, halves of a layer's own behind a window
    that keeps the first keys, with a sink, pairs with a soft cap; 8 query heads over 2 key heads of 32."""
    from denno_beta_amd.parts import DecoderSpec, LayerCall, LayerSpec
    E, dh = 96, 32
    extra = [dict(), dict(position=("rotary_halves", dict(dims=16, base=100.0, head_dim=dh)), window=24, keep_first=3, sink="sink"),
             dict(softcap=4.0)]
    specs = []
    for i in range(layers):
        p = f"L{i}."
        norm = lambda n: ("layernorm", dict(width=E, eps=1e-5, weight_name=p + n, bias_name=None))   # noqa: E731
        specs.append(LayerSpec(arrangement="pre_norm", parts=dict(
            norm1=norm("n1"), norm2=norm("n2"),
            mixer=("causal_attention", dict(dict(width=E, n_heads=8, n_kv_heads=2, head_dim=dh, scale=dh ** -0.5, qkv_weight=p + "qkv", qkv_bias=None,
                                                 out_weight=p + "out", out_bias=None), **{k: p + v if k == "sink" else v for k, v in extra[i].items()})),
            ffn=("dense_mlp", dict(width=E, inner=128, activation="gelu_tanh", up_weight=p + "up", up_bias=None, down_weight=p + "down",
                                   down_bias=None)))))
    return DecoderSpec(vocab=61, width=E, max_positions=256, token_table="tok", position=("rotary_pairs", dict(dims=dh, base=50.0, head_dim=dh)),
                       layers=specs, run_order=[LayerCall(i, i) for i in range(layers)],
                       final_norm=("layernorm", dict(width=E, eps=1e-5, weight_name="nf", bias_name=None)))


def turned_tensors(spec, device, dtype):
    from denno_beta_amd.weights import draw_all
    t = draw_all(spec.param_specs(), 5, engine_dtype=dtype, device=torch.device(device), stored=dtype)
    # (with weights of 0.02 attention hardly shows in the logits)
    return {k: v * 8 if k.endswith(("qkv", "out")) else v for k, v in t.items()}


def runner(device, dtype, **more):
    from denno_beta_amd.engine import ModelRunner
    spec = turned_spec()
    return ModelRunner(spec, turned_tensors(spec, device, dtype), options(device, dtype, **more))


def close_enough(got, want, what):
    """A cache in 8 bits holds a number within half a step, 2^-4 of itself at most; uniform within that, it is 2^-4 / sqrt(3) = 0.036 of
    itself off in the root of the mean square.  A layer's keys and values together: sqrt(2) of that, three layers: sqrt(3) of
    that, 0.088 of what attention adds to the logits, which is no more than their spread; activations in bfloat16 add 0.007
    (replay_util.BF16_MEAN).  A mean is no larger than the root of the mean square; the worst of some ten thousand is up to six
    times that, 0.6.  A lost key, a wrong page or a scale of another page moves logits by the spread itself."""
    spread = want.float().std(dim=1, keepdim=True)
    off = (got.float() - want.float()).abs() / spread
    assert off.max() <= 0.6 and off.mean() <= 0.095, (what, float(off.max()), float(off.mean()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_gpt2_in_every_cutting(device, model_folders, dtype):
    from denno_beta_amd.engine import ModelRunner
    lengths = (7, 33) if device == "cpu" else (7, 19, 33, 100)
    folder = model_folders("A", dtype)
    seqs = [seeded_tokens(11 + i, n, TINY["A"][0]["vocab_size"]) for i, n in enumerate(lengths)]
    want = U.replay(ModelRunner.from_folder(folder, options(device, dtype, None)), U.whole_trace(seqs))
    for kind, steps in {"whole": U.whole_trace(seqs), "tail": U.tail_decode_trace(seqs, 12), "chunks": U.chunk_trace(seqs),
                        "mixed": U.mixed_trace(seqs, seed=5)}.items():
        r = ModelRunner.from_folder(folder, options(device, dtype))
        assert r.cache.k[0].dtype == FP8 and r.cache.view(0, True).k_scale.shape == (r.cache.k[0].shape[1], r.cache.k[0].shape[2])
        got = U.replay(r, steps)
        r.cache.manager.check()
        for rid in want:
            close_enough(got[rid], want[rid], (kind, rid))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_turned_heads_windows_and_sinks(device, dtype):
    seqs = [seeded_tokens(3 + i, n, 61) for i, n in enumerate((5, 40) if device == "cpu" else (5, 40, 90, 130))]
    want = U.replay(runner(device, dtype, cache_dtype=None), U.whole_trace(seqs))
    for kind, steps in {"whole": U.whole_trace(seqs), "chunks": U.chunk_trace(seqs), "mixed": U.mixed_trace(seqs, seed=2)}.items():
        got = U.replay(runner(device, dtype), steps)
        for rid in want:
            close_enough(got[rid], want[rid], (kind, rid))


def same(a, b):
    a, b = a.cpu().double(), b.cpu().double()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,page", [("float32", 16), ("bfloat16", 16), ("bfloat16", 32), ("bfloat16", 8)])
def test_every_call_of_a_run_is_the_definitions(monkeypatch, dtype, page):
    """Portions beside single rows, pages given back and used again: what each call of both operators leaves is compared with the
    definition in 64 bits on the same inputs."""
    from denno_beta_amd.kernels import ops
    calls = {"append": 0, "attend": 0}
    real_append, real_attend = ops.kv_append8, ops.attention8

    def append(src, k_col, v_col, slot_map, k, v, ks, vs, **kw):
        want = [t.cpu().clone() for t in (k, v, ks, vs)]
        before = {n: t.cpu().clone() if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
        R.kv_append8(src.cpu().clone(), k_col, v_col, slot_map.cpu(), *want, **before)
        real_append(src, k_col, v_col, slot_map, k, v, ks, vs, **kw)
        assert all(same(a, b) for a, b in zip((k, v, ks, vs), want)), "append"
        if "q_out" in kw:
            q = before["q_out"].double()
            assert bool(((kw["q_out"].cpu().double() - q).abs() <= 2 * (HALF[src.dtype] + 2.0 ** -24) * q.abs() + 1e-300).all())
        calls["append"] += 1

    def attend(q, out, k, v, ks, vs, tables, tiles, heads, scale, window=0, **kw):
        extra = {n: kw[n] for n in ("sink", "keep_first", "softcap")}
        want, mass, most = R.attention_exact(q, k, v, ks, vs, tables, tiles, heads, scale, window, **extra)
        real_attend(q, out, k, v, ks, vs, tables, tiles, heads, scale, window, **kw)
        dh, n = k.shape[3], k.shape[2] * tables.shape[1]
        loss = (2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -23) + 2 * (dh + 8) * 2.0 ** -23 * most.repeat_interleave(dh, 1) + 2 * n * 2.0 ** -24
        loss = loss + 4 * extra["softcap"] * 2.0 ** -22
        rows = ~want.isnan().all(1)
        bad = (out.cpu().double() - want).abs() > HALF[q.dtype] * want.abs() + loss * mass * 1.01 + 1e-30
        assert bool(rows.any()) and not bool(bad[rows].any()), "attend"
        calls["attend"] += 1
        return out
    monkeypatch.setattr(ops, "kv_append8", append)
    monkeypatch.setattr(ops, "attention8", attend)
    seqs = [seeded_tokens(30 + i, n, 61) for i, n in enumerate((50, 33, 90, 17, 64))]
    steps = U.mixed_trace(seqs, seed=9, max_live=3)
    U.replay(runner("cuda:0", dtype, page_size=page, use_graphs=False, cache_tokens=256), steps)
    assert calls["append"] == calls["attend"] == 3 * len(steps)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_replay_the_same_bits(dtype):
    """Single rows and portions from captured graphs, several replays of each with eager work and synchronizations between them."""
    seqs = [seeded_tokens(40 + i, n, 61) for i, n in enumerate((60, 41, 90, 70))]
    steps = U.mixed_trace(seqs, seed=1, sizes=(1, 1, 1, 1, 8, 8))
    want = U.replay(runner("cuda:0", dtype, use_graphs=False), steps)
    r = runner("cuda:0", dtype)
    for _ in range(3):
        got = U.replay(r, steps)
        torch.cuda.synchronize()
        x = torch.randn(64, 64, device="cuda:0")
        (x @ x).sum().item()
        for rid in want:
            assert torch.equal(got[rid], want[rid]), rid
    assert r.graphs.graphs and r.graphs.portions


def test_generation_with_few_pages(device, model_folders):
    """Requests that preempt one another, in pages that others have used: every page comes back, and generation alone gives a
    request's tokens (32-bit; what a page holds depends on the order in which it was filled, so only an undisturbed request is compared)."""
    from denno_beta_amd.engine import Engine, SamplingParams
    folder = model_folders("A", "float32")
    prompts = [seeded_tokens(60 + i, n, TINY["A"][0]["vocab_size"]) for i, n in enumerate((9, 14, 11))]
    params = SamplingParams(max_tokens=12 if device == "cpu" else 40, temperature=0.0)
    eng = Engine.from_folder(folder, options(device, max_live=3, cache_tokens=48 if device == "cpu" else 112))
    got = eng.generate(prompts, params)
    eng.runner.cache.manager.check()
    assert all(len(t) > 0 for t in got)
    alone = Engine.from_folder(folder, options(device, max_live=1)).generate([prompts[0]], params)[0]
    assert got[0] == alone


def test_what_keeps_no_8_bits_is_refused(model_folders):
    from denno_beta_amd.config import EngineOptions
    from denno_beta_amd.engine.runner import refuse_8_bits
    from denno_beta_amd.parts import MIXERS
    with pytest.raises(ValueError, match="cache_dtype"):
        EngineOptions(cache_dtype="int4").validate()
    refuse_8_bits(turned_spec().instantiate())
    spec = turned_spec(2)
    kind, args = spec.layers[1].parts["mixer"]
    spec.layers[1].parts["mixer"] = (kind, dict({k: v for k, v in args.items() if k != "position"}, exact_turn=True))
    with pytest.raises(ValueError, match="causal_attention keeps no cache in 8 bits"):
        refuse_8_bits(spec.instantiate())
    assert [name for name, cls in MIXERS.items() if getattr(cls, "keeps_8_bits", False)] == ["causal_attention"]


def test_what_a_token_takes():
    from denno_beta_amd.cache import CacheStorage
    from denno_beta_amd.parts import PagedKV
    need = [PagedKV(25, 64), PagedKV(25, 64), PagedKV(2, 128, dtype="float32")]
    full = CacheStorage(need, kv_dtype=torch.bfloat16, page_size=16, cache_tokens=64, max_live=1, device="cpu")
    small = CacheStorage(need, kv_dtype=FP8, page_size=16, cache_tokens=64, max_live=1, device="cpu")
    own = 2 * 2 * 128 * 4          # (a cache that names its dtype keeps it)
    assert full.bytes_per_token() == 2 * 2 * 25 * 64 * 2 + own and small.bytes_per_token() == 2 * 2 * 25 * 64 + 25 + own
    assert small.k_scale[0].shape == (2, 4, 25) and small.k_scale[1] is None and small.view(2, True).k_scale is None and full.k_scale == [None, None]


@pytest.mark.gpu
def test_command_line(tmp_path, capsys):
    from denno_beta_amd.cli import main
    cfg = tmp_path / "c.json"
    cfg.write_text(json.dumps(TINY["A"][0]))
    assert main(["random-model", str(tmp_path / "m"), "--config", str(cfg), "--seed", "0", "--dtype", "bfloat16"]) == 0
    assert main(["generate", str(tmp_path / "m"), "--prompt-ids", "1,2,3", "--max-tokens", "6", "--temperature", "0", "--ignore-eos",
                 "--cache-dtype", "float8"]) == 0
    assert len(capsys.readouterr().out.strip().splitlines()[-1].split(",")) == 6
