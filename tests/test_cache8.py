"""The cache in 8 bits without a GPU: what its functions refuse, what its C entries refuse before they launch anything, and the
definitions that the GPU tests compare with."""
import contextlib
import ctypes
import math

import pytest
import torch

import cache8_refs as R
from denno_beta_amd.kernels import ops

FP8 = torch.float8_e4m3fn


class Launched(Exception):
    pass


@contextlib.contextmanager
def host_checks_only(monkeypatch):
    """The host's checks on CPU tensors; a launch raises Launched.  (cuda:0 stands for the CPU: where a tensor lies is not checked here.)"""
    real = ops._dev

    def dev(t, name, dtypes=None, dims=None):
        if isinstance(t, torch.Tensor) and not t.is_cuda:
            if dtypes is not None and t.dtype not in dtypes:
                raise ops.KernelError(f"{name}: dtype {t.dtype}, wanted one of {dtypes}")
            if dims is not None and t.dim() != dims:
                raise ops.KernelError(f"{name}: {t.dim()} dimensions, wanted {dims}")
            return t
        return real(t, name, dtypes, dims)

    def launch(name):
        raise Launched(name)
    monkeypatch.setattr(ops, "_dev", dev)
    monkeypatch.setattr(ops, "_lib", launch)
    monkeypatch.setattr(ops, "_lib_quiet", launch)
    monkeypatch.setattr(ops, "_one_device", lambda *a: None)
    yield


def pools(n_pages=3, hkv=2, ps=16, dh=64, dtype=FP8):
    return [torch.zeros(n_pages, hkv, ps, dh).to(dtype), torch.zeros(n_pages, hkv, dh, ps).to(dtype), torch.zeros(n_pages, hkv),
            torch.zeros(n_pages, hkv)]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def append_args(T=4, H=4, hkv=2, dh=64):
    src = torch.zeros(T, (H + 2 * hkv) * dh, dtype=torch.bfloat16)
    return dict(src=src, k_col=H * dh, v_col=(H + hkv) * dh, slot_map=i32(*range(T))), pools()


def call_append(args, four, **kw):
    a = dict(args)
    return ops.kv_append8(a.pop("src"), a.pop("k_col"), a.pop("v_col"), a.pop("slot_map"), *four, **dict(a, **kw))


def test_append_takes_what_it_documents(monkeypatch):
    args, four = append_args()
    freq, pos = torch.ones(32), i32(0, 1, 2, 3)
    with host_checks_only(monkeypatch):
        for kw in (dict(), dict(positions=pos, freq=freq), dict(positions=pos, freq=freq, halves=True, mag=2.0),
                   dict(positions=pos, freq=freq, q_out=args["src"][:, :256], q_col=0, n_heads=4),
                   dict(positions=pos, freq=freq, q_out=torch.zeros(4, 256, dtype=torch.bfloat16), q_col=0, n_heads=4)):
            with pytest.raises(Launched):
                call_append(args, four, **kw)
        none = dict(args, src=args["src"][:0], slot_map=args["slot_map"][:0])
        assert call_append(none, four) is None       # no rows: nothing to launch


@pytest.mark.parametrize("change,kw", [
    (dict(src=torch.zeros(4, 512, dtype=torch.float16)), {}),
    (dict(src=torch.zeros(512)), {}),
    (dict(src=torch.zeros(512, 4, dtype=torch.bfloat16).t()), {}),
    (dict(slot_map=i32(0, 1, 2)), {}),
    (dict(slot_map=torch.arange(4)), {}),
    (dict(slot_map=i32(*range(8))[::2]), {}),
    (dict(k_col=512 - 127), {}),
    (dict(v_col=-1), {}),
    ({}, dict(freq=torch.ones(33), positions=i32(0, 1, 2, 3))),
    ({}, dict(freq=torch.ones(0), positions=i32(0, 1, 2, 3))),
    ({}, dict(freq=torch.ones(32, dtype=torch.float64), positions=i32(0, 1, 2, 3))),
    ({}, dict(freq=torch.ones(32))),
    ({}, dict(freq=torch.ones(32), positions=i32(0, 1, 2))),
    ({}, dict(freq=torch.ones(32), positions=torch.arange(4))),
    ({}, dict(q_out=torch.zeros(4, 256, dtype=torch.bfloat16), n_heads=4)),
    ({}, dict(n_heads=4)),
    ({}, dict(freq=torch.ones(32), positions=i32(0, 1, 2, 3), q_out=torch.zeros(4, 256), n_heads=4)),
    ({}, dict(freq=torch.ones(32), positions=i32(0, 1, 2, 3), q_out=torch.zeros(4, 256, dtype=torch.bfloat16), n_heads=3)),
    ({}, dict(freq=torch.ones(32), positions=i32(0, 1, 2, 3), q_out=torch.zeros(4, 256, dtype=torch.bfloat16), n_heads=4, q_col=1)),
    ({}, dict(freq=torch.ones(32), positions=i32(0, 1, 2, 3), q_out=torch.zeros(3, 256, dtype=torch.bfloat16), n_heads=4)),
])
def test_append_refuses(monkeypatch, change, kw):
    args, four = append_args()
    with host_checks_only(monkeypatch), pytest.raises(ops.KernelError):
        call_append(dict(args, **change), four, **kw)


def test_append_refuses_a_q_out_that_overlaps_its_source(monkeypatch):
    args, four = append_args()
    turn = dict(freq=torch.ones(32), positions=i32(0, 1, 2, 3), n_heads=4, q_col=0)
    with host_checks_only(monkeypatch):
        for bad in (args["src"][:, 1:257], args["src"][:, 256:512], args["src"].view(-1)[:1024].view(4, 256)):
            with pytest.raises(ops.KernelError, match="q_out"):
                call_append(args, four, q_out=bad, **turn)


def bad_pools():
    p = pools()
    return [("dtype", [p[0].float()] + p[1:]), ("dtype", [p[0], p[1].to(torch.float8_e5m2)] + p[2:]), ("wanted", [p[0], p[0]] + p[2:]),
            ("wanted", [p[0].transpose(0, 1).contiguous().transpose(0, 1)] + p[1:]), ("scale", p[:2] + [p[2][:2], p[3]]),
            ("dtype", p[:3] + [p[3].double()]), ("scale", p[:3] + [torch.zeros(2, 3).t()]), ("empty", pools(n_pages=0)),
            ("head size", pools(dh=257))]


@pytest.mark.parametrize("i", range(9))
def test_both_refuse_pools(monkeypatch, i):
    what, four = bad_pools()[i]
    args, _ = append_args()
    q = torch.zeros(4, 256, dtype=torch.bfloat16)
    with host_checks_only(monkeypatch):
        with pytest.raises(ops.KernelError, match=what):
            call_append(args, four)
        with pytest.raises(ops.KernelError, match=what):
            ops.attention8(q, torch.zeros_like(q), *four, torch.zeros(1, 3, dtype=torch.int32), i32([0], [0], [4], [3]), 4, 0.125)


def attend_args():
    q = torch.zeros(4, 256, dtype=torch.bfloat16)
    return dict(q=q, out=torch.zeros_like(q), block_tables=torch.zeros(1, 3, dtype=torch.int32), tiles=i32([0], [0], [4], [3]), n_heads=4)


def call_attend(a, **kw):
    return ops.attention8(a["q"], a["out"], *pools(), a["block_tables"], a["tiles"], a["n_heads"], 0.125, **kw)


def test_attention_takes_what_it_documents(monkeypatch):
    a = attend_args()
    with host_checks_only(monkeypatch):
        for kw in (dict(), dict(window=5, keep_first=3), dict(sink=True), dict(sink=torch.zeros(4)), dict(softcap=3.0),
                   dict(tiles_wide=a["tiles"])):
            with pytest.raises(Launched):
                call_attend(a, **kw)
        none = dict(a, tiles=torch.zeros(4, 0, dtype=torch.int32))
        assert call_attend(none) is none["out"]


@pytest.mark.parametrize("change,kw", [
    (dict(q=torch.zeros(4, 256, dtype=torch.float16)), {}),
    (dict(out=torch.zeros(4, 256)), {}),
    (dict(out=torch.zeros(4, 128, dtype=torch.bfloat16)), {}),
    (dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)), {}),
    (dict(q=torch.zeros(4, 255, dtype=torch.bfloat16)), {}),
    (dict(q=torch.zeros(256, 4, dtype=torch.bfloat16).t()), {}),
    (dict(n_heads=3), {}),
    (dict(n_heads=0), {}),
    (dict(block_tables=torch.zeros(1, 3, dtype=torch.int64)), {}),
    (dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).t()), {}),
    (dict(tiles=torch.zeros(3, 1, dtype=torch.int32)), {}),
    (dict(tiles=torch.zeros(2, 4, dtype=torch.int32).t()), {}),
    ({}, dict(sink=torch.zeros(3))),
    ({}, dict(sink=torch.zeros(4, dtype=torch.bfloat16))),
    ({}, dict(window=-1)),
    ({}, dict(window=4, keep_first=-1)),
    ({}, dict(softcap=-1.0)),
    ({}, dict(softcap=math.inf)),
    ({}, dict(softcap=math.nan)),
])
def test_attention_refuses(monkeypatch, change, kw):
    with host_checks_only(monkeypatch), pytest.raises(ops.KernelError):
        call_attend(dict(attend_args(), **change), **kw)


def test_no_cpu_path():
    args, four = append_args()
    with pytest.raises(ops.KernelError, match="GPU"):
        call_append(args, four)
    with pytest.raises(ops.KernelError, match="GPU"):
        call_attend(attend_args())


# -- the C entries --------------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def library():
    if torch.cuda.is_available():
        pytest.skip("a launch is an error only where there is no GPU")
    from denno_beta_amd.build import load_library
    lib = load_library("cache8")
    ops._declare("cache8", lib)
    return lib


def c_append(lib, dims=64, n_heads=0, T=4, hkv=2, dh=64, ps=16, dtype=1, n_pages=3):
    p = ctypes.addressof((ctypes.c_float * 64)())
    return lib.dn_kv_append8(p, 512, 256, 384, p, p, p, p, p, n_pages, p, p, dims, 0, 1.0, 0, n_heads, p, 256, T, hkv, dh, ps, dtype, None)


def test_append_entry_refuses_before_it_launches(library):
    assert c_append(library, T=0) == 0
    for kw in (dict(dims=3), dict(dims=66), dict(dims=-2), dict(dh=0, dims=0), dict(dh=257), dict(ps=0), dict(hkv=0), dict(n_heads=-1), dict(n_pages=0),
               dict(n_heads=1, dims=0)):
        assert c_append(library, **kw) == -2, kw
    assert c_append(library, dtype=2) == -1
    assert c_append(library) > 0      # (no GPU here: the launch itself)


def c_attend(lib, n_tiles=1, H=4, hkv=2, dh=64, ps=16, window=0, keep=0, cap=0.0, dtype=1):
    p = ctypes.addressof((ctypes.c_float * 64)())
    return lib.dn_attention8(p, 256, p, 256, p, p, p, p, 3, p, 3, p, p, p, p, n_tiles, H, hkv, dh, ps, 0.125, window, keep, 0, None, cap, dtype, None)


def test_attention_entry_refuses_before_it_launches(library):
    assert c_attend(library, n_tiles=0) == 0
    for kw in (dict(dh=0), dict(dh=257), dict(hkv=0), dict(hkv=3), dict(ps=0), dict(window=-1), dict(keep=1), dict(keep=-1, window=4),
               dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf)):
        assert c_attend(library, **kw) == -2, kw
    assert c_attend(library, dtype=2) == -1
    assert c_attend(library) > 0


# -- the definitions ------------------------------------------------------------------------------------------------------------

def test_nearest_numbers_are_the_formats_own():
    """Every e4m3 number is its own nearest; between two neighbours the middle goes to the even one, and what is just off it does not."""
    numbers = torch.arange(127, dtype=torch.uint8).view(FP8).double()
    assert torch.equal(R.nearest(numbers).double(), numbers) and torch.equal(R.nearest(-numbers).double(), -numbers)
    middle, code = (numbers[1:] + numbers[:-1]) / 2, torch.arange(126)
    even = numbers[torch.where(code % 2 == 0, code, code + 1)]
    assert torch.equal(R.nearest(middle).double(), even)
    assert torch.equal(R.nearest(middle * (1 + 1e-14)).double(), numbers[1:]) and torch.equal(R.nearest(middle * (1 - 1e-14)).double(), numbers[:-1])


def test_a_pages_scale_never_shrinks_and_begins_anew():
    k, v, ks, vs = pools(hkv=1, dh=2)
    for t, x in enumerate((1.0, 1000.0, 1e-6, 0.0)):
        src = torch.full((1, 4), x)
        R.kv_append8(src, 0, 2, i32(t), k, v, ks, vs)
    assert float(ks[0, 0]) == 4.0                       # 1000 / 448 = 2.2
    assert (k[0, 0, :4, 0].float() * 4).tolist() == [1.0, 1024.0, 0.0, 0.0]      # (the nearest of 960 and 1024)
    R.kv_append8(torch.full((1, 4), 0.5), 0, 2, i32(0), k, v, ks, vs)
    assert float(ks[0, 0]) == 2.0 ** -9 and not bool(k[0, 0, 1:].float().any())      # 0.5 / 2^-9 = 256
