"""The two sets of checks in front of the cache in 8 bits: what the short one (one expression, in front of ordinary calls) lets pass, the long one,
which says what is wrong, lets pass as well."""
import random

import pytest
import torch

import test_cache8 as C
from denno_beta_amd.kernels import ops

FP8 = torch.float8_e4m3fn


@pytest.fixture
def on_a_device(monkeypatch):
    """CPU tensors that say they lie on device 0, the current one."""
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(ops, "_device_now", lambda: 0)
    with C.host_checks_only(monkeypatch):
        yield


def append_holds(args, four, **kw):
    a = dict(dict(positions=None, freq=None, q_out=None, q_col=0, n_heads=0), **dict(args, **kw))
    return ops._append8_holds(a["src"], a["k_col"], a["v_col"], a["slot_map"], *four, a["positions"], a["freq"], a["q_out"], a["q_col"], a["n_heads"])


def append_long(args, four, **kw):
    a = dict(dict(positions=None, freq=None, q_out=None, q_col=0, n_heads=0), **dict(args, **kw))
    shape = ops._pools8(*four, "kv_append8")
    ops._append8_checks(a["src"], a["k_col"], a["v_col"], a["slot_map"], a["positions"], a["freq"], a["q_out"], a["q_col"],
                        a["n_heads"], shape[1], shape[3])
    return shape


def attend_holds(a, four):
    return ops._attention8_holds(a["q"], a["out"], *four, a["block_tables"], a["tiles"], a["n_heads"])


def attend_long(a, four):
    shape = ops._pools8(*four, "attention8")
    ops._attention8_checks(a["q"], a["out"], a["block_tables"], a["tiles"], a["n_heads"], shape[1], shape[3])
    return shape


def cases_of(test):
    return [c for m in test.pytestmark if m.name == "parametrize" for c in m.args[1]]


def test_ordinary_calls_take_the_short_way(on_a_device):
    args, four = C.append_args()
    freq, pos = torch.ones(32), C.i32(0, 1, 2, 3)
    for kw in (dict(), dict(positions=pos, freq=freq), dict(positions=pos, freq=freq, q_out=args["src"][:, :256], n_heads=4),
               dict(positions=pos, freq=freq, q_out=torch.zeros(4, 256, dtype=torch.bfloat16), n_heads=4)):
        assert append_holds(args, four, **kw) == append_long(args, four, **kw) == (3, 2, 16, 64)
    a = C.attend_args()
    assert attend_holds(a, C.pools()) == attend_long(a, C.pools()) == (3, 2, 16, 64)


@pytest.mark.parametrize("change,kw", cases_of(C.test_append_refuses))
def test_append_refuses(on_a_device, change, kw):
    args, four = C.append_args()
    assert append_holds(dict(args, **change), four, **kw) is None
    with pytest.raises(ops.KernelError):
        C.call_append(dict(args, **change), four, **kw)


@pytest.mark.parametrize("change,kw", [c for c in cases_of(C.test_attention_refuses) if not c[1]])
def test_attention_refuses(on_a_device, change, kw):
    a = dict(C.attend_args(), **change)
    assert attend_holds(a, C.pools()) is None
    with pytest.raises(ops.KernelError):
        C.call_attend(a)


@pytest.mark.parametrize("i", range(9))
def test_both_refuse_pools(on_a_device, i):
    what, four = C.bad_pools()[i]
    assert append_holds(C.append_args()[0], four) is None and attend_holds(C.attend_args(), four) is None
    with pytest.raises(ops.KernelError, match=what):
        C.call_append(C.append_args()[0], four)


def test_tables_in_another_form(on_a_device):
    args, four = C.append_args()
    turn = dict(positions=C.i32(0, 1, 2, 3), freq=torch.ones(32))
    for change, kw in (({}, dict(turn, positions=turn["positions"][None])), (dict(slot_map=args["slot_map"][None]), {})):
        assert append_holds(dict(args, **change), four, **kw) is None
        with pytest.raises(ops.KernelError):
            C.call_append(dict(args, **change), four, **kw)


def forms(rng, shape, dtype):
    """A tensor of this shape, or of one near it, whole or a view, in this dtype or another."""
    shape = list(shape)
    if rng.random() < 0.15:
        i = rng.randrange(len(shape))
        shape[i] = max(0, shape[i] + rng.choice([-1, 1, shape[i]]))
    if rng.random() < 0.05:
        shape = shape + [1] if rng.random() < 0.5 else [1] + shape
    if rng.random() < 0.1:
        dtype = rng.choice([torch.float32, torch.bfloat16, torch.int32, torch.int64, FP8])
    if rng.random() < 0.05:
        return None
    way = rng.random()
    if way < 0.7:
        return torch.zeros(shape).to(dtype)
    if way < 0.85:      # rows further apart
        return torch.zeros(shape[:-1] + [shape[-1] + 8]).to(dtype)[..., :shape[-1]]
    if way < 0.93:
        return torch.zeros(shape[::-1]).to(dtype).permute(*range(len(shape) - 1, -1, -1))
    return torch.zeros(shape[:-1] + [2 * shape[-1]]).to(dtype)[..., ::2]


def refused(f, *a, **kw):
    try:
        f(*a, **kw)
        return None
    except ops.KernelError as e:
        return str(e)


@pytest.mark.parametrize("seed", range(8))
def test_what_the_short_checks_let_pass_the_long_ones_do(on_a_device, seed):
    rng, passed, failed = random.Random(seed), 0, 0
    for _ in range(1500):
        T, H, hkv, dh, ps = rng.choice([0, 1, 4]), 4, 2, rng.choice([16, 63, 64]), 16
        w = (H + 2 * hkv) * dh
        src = forms(rng, (T, w), rng.choice([torch.float32, torch.bfloat16]))
        four = [forms(rng, (3, hkv, ps, dh), FP8), forms(rng, (3, hkv, dh, ps), FP8), forms(rng, (3, hkv), torch.float32), forms(rng, (3, hkv), torch.float32)]
        if rng.random() < 0.7:      # (all right, so that the other arguments are looked at)
            four = C.pools(dh=dh)
        args = dict(src=src, k_col=H * dh + rng.choice([0, 0, 0, 1, -1, -dh]), v_col=(H + hkv) * dh + rng.choice([0, 0, 0, 1, -1]),
                    slot_map=forms(rng, (T,), torch.int32))
        kw = {}
        if rng.random() < 0.7:
            kw.update(freq=forms(rng, (rng.choice([1, dh // 2, dh // 2 + 1]),), torch.float32), positions=forms(rng, (T,), torch.int32))
        if rng.random() < 0.5:
            q = forms(rng, (T, H * dh), torch.bfloat16 if src is None else src.dtype)
            if src is not None and src.dim() == 2 and src.shape[1] >= H * dh and rng.random() < 0.5:
                c = rng.choice([0, 0, 1, dh])
                q = src[:, c:c + H * dh]
            kw.update(q_out=q, q_col=rng.choice([0, 0, 1, dh]), n_heads=rng.choice([H, H, H - 1, 0]))
        shape = append_holds(args, four, **kw)
        if shape is not None:
            passed += 1
            assert refused(append_long, args, four, **kw) is None, (args, kw)
        else:
            failed += 1
        q = forms(rng, (T, H * dh), torch.bfloat16)
        a = dict(q=q, out=forms(rng, (T, H * dh), torch.bfloat16), block_tables=forms(rng, (1, 3), torch.int32), tiles=forms(rng, (4, 1), torch.int32),
                 n_heads=rng.choice([H, H, H, 3, 0, -2]))
        if attend_holds(a, four) is not None:
            passed += 1
            assert refused(attend_long, a, four) is None, a
    assert passed > 100 and failed > 100
