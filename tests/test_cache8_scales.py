"""Scales that are no finite numbers, of pages that are in a request's table: the rows that read such a page have no finite number, all others
are as if the page were not there."""
import math

import pytest
import torch

import cache8_refs as R
from test_cache8_gpu import BF16, DEV, F32, attention_case, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh", [(4, 2, 64), (4, 2, 96), (2, 1, 160), (4, 2, 20)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("splits", [1, 3])
def test_rows_that_do_not_read_a_page(monkeypatch, dtype, H, hkv, dh, bad, splits):
    """A window of 24 in portions: a page that all rows of a tile have passed, one that the earlier rows of a tile still read, and one that only
    the later rows read."""
    o = ops()
    monkeypatch.setattr(o, "_portions8_splits", lambda *a: splits)
    for lens, new, page_at in (([140], [21], 5), ([140], [140], 2), ([140], [140], 7), ([140, 60], [140, 3], 6)):
        q, pools, bt, tiles, wide = attention_case(lens, new, H, hkv, dh, 16, dtype, seed=31)
        on = dict(tiles_wide=wide.to(DEV), window=24)
        tables, q_on = (bt.to(DEV), tiles.to(DEV), H, dh ** -0.5), q.contiguous().to(DEV)

        def attend(four):
            return o.attention8(q_on, torch.full_like(q_on, 9.0), *[p.to(DEV) for p in four], *tables, **on).cpu().double()
        clean = attend(pools)
        for which in (2, 3):      # the keys' scale, the values'
            changed = [p.clone() for p in pools]
            changed[which][int(bt[0, page_at]), 0] = bad
            got = attend(changed).view(q.shape[0], H, dh)
            for s, (n, m) in enumerate(zip(lens, new)):
                for r in range(m):
                    row, pos = sum(new[:s]) + r, n - m + r
                    reads = s == 0 and pos >= 16 * page_at and pos - 23 <= 16 * page_at + 15
                    mine, its = got[row, :H // hkv], clean.view(q.shape[0], H, dh)[row, :H // hkv]
                    if not reads:
                        assert torch.equal(mine, its), (which, page_at, s, pos)
                    elif which == 3:
                        assert not bool(mine.isfinite().any()), (which, page_at, s, pos)
                    # (the other key heads have scales of their own)
                    assert torch.equal(got[row, H // hkv:], clean.view(q.shape[0], H, dh)[row, H // hkv:])
