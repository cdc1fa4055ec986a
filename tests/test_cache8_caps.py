"""Soft caps of any size over the cache in 8 bits: a score is off by some units of its own last place, however large the cap is."""
import pytest
import torch

import cache8_refs as R
from test_cache8_gpu import BF16, DEV, F32, HALF, attention_case, ops

pytestmark = pytest.mark.gpu


def check(case, H, dh, dtype, cap, what, **how):
    """As `test_cache8_gpu.check_attention`, but for what a cap costs: cap * tanh(s / cap) is no larger than |s|, its slope no larger than 1, and it
    is made with some roundings (the quotient, its square, five terms and the product near 0; elsewhere the power, the reciprocal, 1 minus
    twice that, and the product): 16 half units of its own last place hold them, 16 * 2^-24 of scale * sum |q||k| at most."""
    q, pools, bt, tiles, wide = case
    want, mass, most = R.attention_exact(q, *pools, bt, tiles, H, dh ** -0.5, softcap=cap)
    got = torch.full((q.shape[0], H * dh), 9.0, dtype=dtype, device=DEV)
    ops().attention8(q.contiguous().to(DEV), got, *[p.to(DEV) for p in pools], bt.to(DEV), tiles.to(DEV), H, dh ** -0.5, tiles_wide=wide.to(DEV),
                     softcap=cap, **how)
    n = int(pools[0].shape[2] * bt.shape[1])
    loss = (2.0 ** -8 if dtype == BF16 else 2.0 ** -23) + 2 * (dh + 8 + 8) * 2.0 ** -23 * most.repeat_interleave(dh, 1) + 2 * n * 2.0 ** -24
    bound = HALF[dtype] * want.abs() + loss * mass * 1.01 + 1e-30
    off = (got.cpu().double() - want).abs() / bound
    assert bool((off <= 1).all()), (what, float(off.max()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh,ps", [(4, 4, 64, 16), (8, 2, 128, 32), (3, 1, 160, 16), (4, 2, 20, 8)])
@pytest.mark.parametrize("cap", [1e-39, 0.5, 5.0, 50.0, 1e4, 1e6, 1e30, 3e38])
def test_caps(dtype, H, hkv, dh, ps, cap):
    for lens, new, how in (([140, 33, 90], [1, 33, 40], {}), ([140, 1, 64], [1] * 3, dict(single_rows=True, max_context=140))):
        case = attention_case(lens, new, H, hkv, dh, ps, dtype, seed=21, q_scale=2.0)
        check(case, H, dh, dtype, cap, (lens, new), **how)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh", [(4, 4, 64), (8, 2, 128), (3, 1, 160)])
def test_a_rows_bits_do_not_depend_on_the_rows_beside_it(dtype, H, hkv, dh):
    """Tiles of scores that are all small beside the cap go another way than those with larger ones among them: the same bits."""
    for lens, new, how in (([140], [140], {}), ([140, 90, 33], [1] * 3, dict(single_rows=True, max_context=140))):
        q, pools, bt, tiles, wide = attention_case(lens, new, H, hkv, dh, 16, dtype, seed=22, q_scale=0.5)
        on = [p.to(DEV) for p in pools]

        def run(x):
            x = x.contiguous().to(DEV)
            return ops().attention8(x, torch.empty_like(x), *on, bt.to(DEV), tiles.to(DEV), H, dh ** -0.5, tiles_wide=wide.to(DEV), softcap=10.0, **how)
        loud = q.clone()
        loud[::2] *= 40
        loud[1:, :dh] *= 40 if how else 1      # (single rows: a wave has a row's heads)
        a, b = run(q)[1::2], run(loud)[1::2]
        assert torch.equal(a[:, dh:], b[:, dh:])
