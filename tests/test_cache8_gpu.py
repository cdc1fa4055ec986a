"""The cache in 8 bits on the GPU: rows into the pages and attention over them, against the definition in 64 bits."""
import math

import pytest
import torch

import cache8_refs as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP8 = torch.float8_e4m3fn
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}      # half a step, relative


def ops():
    from denno_beta_amd.kernels import ops as o
    return o


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def random_pools(n_pages, hkv, ps, dh, gen):
    """Pages that other steps left: any finite numbers, scales of many sizes."""
    def numbers(*shape):
        b = torch.randint(0, 256, shape, generator=gen, dtype=torch.int64)
        return torch.where(b % 128 == 127, b - 1, b).to(torch.uint8).view(FP8)
    scales = [2.0 ** torch.randint(-12, -4, (n_pages, hkv), generator=gen).float() for _ in range(2)]
    return [numbers(n_pages, hkv, ps, dh), numbers(n_pages, hkv, dh, ps)] + scales


def same(a, b):
    """Equal numbers, NaN in the same places."""
    a, b = a.cpu().double(), b.cpu().double()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def slots_for(requests, ps, gen):
    """requests: [(tokens there, new tokens)] on shuffled pages -> slots, positions, pages in all."""
    blocks = [-(-(h + n) // ps) for h, n in requests]
    order = torch.randperm(sum(blocks) + 2, generator=gen).tolist()
    slots, positions, at = [], [], 0
    for (h, n), b in zip(requests, blocks):
        pages = order[at:at + b]
        at += b
        slots += [pages[p // ps] * ps + p % ps for p in range(h, h + n)]
        positions += range(h, h + n)
    return slots, positions, sum(blocks) + 2


DECODE, PORTIONS = [(0, 1), (17, 1), (15, 1), (16, 1), (300, 1)], [(0, 1), (0, 70), (13, 21), (31, 1), (16, 33)]


def append_both(dtype, H, hkv, dh, ps, requests, turn, dims, mag=1.0, in_place=True, loud=1.0, seed=0, edit=None):
    gen = torch.Generator().manual_seed(seed)
    slots, positions, n_pages = slots_for(requests, ps, gen)
    T = len(slots)
    extra = 3 if dh % 2 else 8          # rows are longer than what is read of them
    src = (torch.randn(T, (H + 2 * hkv) * dh + extra, generator=gen) * loud * torch.exp(torch.randn(T, 1, generator=gen))).to(dtype)
    pools = random_pools(n_pages, hkv, ps, dh, gen)
    if edit:
        edit(src, slots, pools)
    slot_map, pos = i32(slots), i32(positions)
    kw = {}
    if turn != "none":
        freq = (10000.0 ** (-torch.arange(dims // 2, dtype=torch.float64) * 2 / dims)).float()
        kw = dict(positions=pos, freq=freq, halves=turn == "halves", mag=mag, q_col=0, n_heads=H)
    want = [p.clone() for p in pools]
    q_want = torch.zeros(T, H * dh, dtype=dtype)
    R.kv_append8(src, H * dh, (H + hkv) * dh, slot_map, *want, **dict(kw, **({"q_out": q_want} if kw else {})))
    got, there = [p.to(DEV) for p in pools], src.to(DEV)
    q_got = None
    if kw:
        q_got = there[:, :H * dh] if in_place else torch.full((T, H * dh + 5), 7.0, dtype=dtype, device=DEV)[:, :H * dh]
    ops().kv_append8(there, H * dh, (H + hkv) * dh, slot_map.to(DEV), *got,
                     **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}, **({"q_out": q_got} if kw else {}))
    return src, there, want, got, q_want, q_got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh,ps,turn,dims", [
    (4, 4, 64, 16, "none", 0), (8, 2, 128, 16, "pairs", 128), (8, 2, 128, 16, "halves", 128), (5, 5, 80, 32, "halves", 40),
    (6, 3, 48, 8, "pairs", 20), (2, 1, 256, 64, "halves", 256), (3, 3, 15, 16, "pairs", 14), (3, 3, 15, 16, "halves", 6),
    (1, 1, 1, 5, "none", 0), (2, 2, 100, 5, "pairs", 100), (4, 2, 96, 1, "halves", 64), (12, 4, 112, 16, "pairs", 64),
    (3, 1, 176, 48, "none", 0), (25, 25, 64, 16, "none", 0), (4, 2, 128, 64, "pairs", 128), (3, 1, 64, 128, "halves", 64)])
@pytest.mark.parametrize("requests", [DECODE, PORTIONS, [(17, 1)]], ids=["decode", "portions", "one row"])
def test_append(dtype, H, hkv, dh, ps, turn, dims, requests):
    """Numbers and scales are the definition's exactly (both round 64-bit values once); everything outside the rows' pages stays."""
    for in_place in (True, False):
        src, there, want, got, q_want, q_got = append_both(dtype, H, hkv, dh, ps, requests, turn, dims, in_place=in_place, seed=dh + ps)
        for name, a, b in zip(("keys", "values", "key scales", "value scales"), got, want):
            assert same(a, b), name
        if q_got is not None:
            # one rounding to the type, and the 32-bit one before it
            bound = (HALF[dtype] + 2.0 ** -24) * q_want.double().abs() + 1e-300
            assert bool(((q_got.cpu().double() - q_want.double()).abs() <= 2 * bound).all())
            keep = there[:, H * dh:] if in_place else there
            assert torch.equal(keep.cpu(), src[:, H * dh:] if in_place else src)
        else:
            assert torch.equal(there.cpu(), src)


@pytest.mark.parametrize("H,hkv,dh,ps,turn,dims", [(4, 4, 64, 16, "none", 0), (4, 2, 128, 16, "pairs", 64), (2, 2, 40, 32, "halves", 40)])
def test_append_infinities_zeros_and_extremes(H, hkv, dh, ps, turn, dims):
    """Values that are not finite become NaN and do not count for a scale; rows of zeros, rows so small that the scale's exponent is at
    its end, rows as large as the type has them, and rows so small that all their numbers are zero beside what the page holds."""
    for dtype in (F32, BF16):
        def edit(src, slots, pools):
            w = src.shape[1]
            src[0] = 0
            src[1, ::7] = math.inf
            src[1, 3::11] = -math.inf
            src[2, 5::13] = math.nan
            src[3] *= 1e-38
            src[4] = torch.finfo(dtype).max * torch.linspace(-0.5, 0.5, w).sign().to(dtype) * 0.5
            src[5] = math.nan
            src[6] *= 1e-30
            pools[0].view(torch.uint8)[slots[6] // ps, :, -1] = 0x7f       # a page that holds NaN keeps it
        _, _, want, got, _, _ = append_both(dtype, H, hkv, dh, ps, [(0, 2), (5, 1), (0, 1), (7, 1), (3, 1), (9, 1), (0, 5)], turn, dims,
                                            in_place=False, edit=edit, seed=3)
        for name, a, b in zip(("keys", "values", "key scales", "value scales"), got, want):
            assert same(a, b), (name, dtype)


@pytest.mark.parametrize("turn,mag", [("pairs", 1.25), ("halves", 0.7)])
def test_append_far_positions_and_a_factor(turn, mag):
    """Positions up to the largest int32: the angle is the 64-bit product, and so are its sine and cosine."""
    gen = torch.Generator().manual_seed(1)
    T, dh, ps = 6, 64, 16
    positions = i32([0, 1, 131071, 4194304, 1 << 30, (1 << 31) - 1])
    slots = i32([0, 17, 34, 51, 68, 85])
    freq = (500000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float()
    src = torch.randn(T, 3 * dh, generator=gen)
    pools = random_pools(7, 1, ps, dh, gen)
    want, q_want = [p.clone() for p in pools], torch.zeros(T, dh)
    kw = dict(halves=turn == "halves", mag=mag, q_col=0, n_heads=1)
    R.kv_append8(src, dh, 2 * dh, slots, *want, positions=positions, freq=freq, q_out=q_want, **kw)
    got, q_got = [p.to(DEV) for p in pools], torch.empty(T, dh, device=DEV)
    ops().kv_append8(src.to(DEV), dh, 2 * dh, slots.to(DEV), *got, positions=positions.to(DEV), freq=freq.to(DEV), q_out=q_got, **kw)
    assert all(same(a, b) for a, b in zip(got, want))
    assert torch.allclose(q_got.cpu(), q_want, atol=0, rtol=2.0 ** -23)


@pytest.mark.parametrize("requests", [[(0, 700), (5, 650), (40, 300)], [(0, 2600)],
                                      [(17, 1)] * 40 + [(0, 700), (7, 1), (5, 650)] + [(31, 1)] * 30 + [(6, 500), (32, 1)], [(3, 1), (0, 1)] * 300,
                                      [(15, 2), (14, 3), (16, 1)] * 120], ids=["portions", "a prompt", "mixed", "single rows", "ends of pages"])
def test_append_many_rows(requests):
    """More rows than there are workgroups for one by one: runs of rows that begin and end inside pages, single ones beside them."""
    for H, hkv, dh, ps, turn, dims in ((33, 33, 16, 16, "none", 0), (2, 9, 16, 64, "halves", 8), (2, 5, 24, 16, "pairs", 24)):
        _, _, want, got, q_want, q_got = append_both(BF16, H, hkv, dh, ps, requests, turn, dims, seed=len(requests))
        for name, a, b in zip(("keys", "values", "key scales", "value scales"), got, want):
            assert same(a, b), name
        if q_got is not None:
            assert bool(((q_got.cpu().double() - q_want.double()).abs() <= 2 * (2.0 ** -8 + 2.0 ** -24) * q_want.double().abs() + 1e-300).all())


def test_append_leaves_rows_without_a_slot_and_bad_pages():
    """Rows of padding (slot -1) and rows whose page is outside the pools write nothing; their queries are turned like the others'."""
    gen = torch.Generator().manual_seed(2)
    H, hkv, dh, ps = 2, 1, 64, 16
    slots = [-1, 5, 6, -1, 16 * 4 + 1, -7, 16 * 3 + 15, -1]
    src = torch.randn(8, 4 * dh, generator=gen).to(BF16)
    pools = random_pools(4, hkv, ps, dh, gen)
    freq = torch.ones(4)
    kw = dict(positions=i32(range(8)), freq=freq, q_col=0, n_heads=H)
    want, q_want = [p.clone() for p in pools], torch.zeros(8, H * dh, dtype=BF16)
    R.kv_append8(src, 2 * dh, 3 * dh, i32(slots), *want, q_out=q_want, **kw)
    got, q_got = [p.to(DEV) for p in pools], torch.zeros(8, H * dh, dtype=BF16, device=DEV)
    ops().kv_append8(src.to(DEV), 2 * dh, 3 * dh, i32(slots).to(DEV), *got, positions=kw["positions"].to(DEV), freq=freq.to(DEV), q_out=q_got,
                     q_col=0, n_heads=H)
    assert all(same(a, b) for a, b in zip(got, want))
    assert torch.allclose(q_got.cpu().float(), q_want.float(), atol=0, rtol=2.0 ** -7)


def test_append_token_by_token_and_at_once():
    """A page filled token by token holds the same scales as one filled at once, and numbers within the roundings that its growing scale
    made: those of a normal size are the same, the others are off by at most a step of the least ones, 2^-9 of the scale."""
    gen = torch.Generator().manual_seed(4)
    hkv, dh, ps, T = 3, 64, 16, 40
    src = (torch.randn(T, 2 * hkv * dh, generator=gen) * torch.exp(torch.randn(T, 1, generator=gen))).to(BF16).to(DEV)
    slots = i32(range(T)).to(DEV)
    pools = [[p.to(DEV) for p in random_pools(3, hkv, ps, dh, gen)] for _ in range(2)]
    ops().kv_append8(src, 0, hkv * dh, slots, *pools[0])
    for t in range(T):
        ops().kv_append8(src[t:t + 1], 0, hkv * dh, slots[t:t + 1], *pools[1])
    (k, v, ks, vs), (k1, v1, ks1, vs1) = pools
    assert torch.equal(ks, ks1) and torch.equal(vs, vs1)
    for a, b in ((k, k1), (v, v1)):
        a, b = a.float(), b.float()
        assert bool(((a - b).abs() <= 2.0 ** -9).all()) and bool((a == b)[a.abs() >= 2.0 ** -5].all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dh,ps,turn,dims", [(64, 16, "pairs", 64), (128, 32, "halves", 96), (48, 16, "none", 0)])
def test_append_rows_of_a_page_in_any_order(dtype, dh, ps, turn, dims):
    """The rows of a page stand side by side, but not in the order of their places; the pages before and behind are in order."""
    gen = torch.Generator().manual_seed(6)
    H, hkv = 10, 5
    slots = [3 * ps + i for i in range(ps)] + [ps + i for i in (5, 4, 9, 0, 2)] + [2 * ps + 7 - i for i in range(4)] + [i for i in range(1, 9)]
    T = len(slots)
    src = (torch.randn(T, (H + 2 * hkv) * dh, generator=gen) * torch.exp(torch.randn(T, 1, generator=gen))).to(dtype)
    pools = random_pools(5, hkv, ps, dh, gen)
    kw = {}
    if dims:
        kw = dict(positions=i32(range(100, 100 + T)), freq=(10000.0 ** (-torch.arange(dims // 2).double() * 2 / dims)).float(), halves=turn == "halves",
                  q_col=0, n_heads=H)
    want, q_want = [p.clone() for p in pools], torch.zeros(T, H * dh, dtype=dtype)
    R.kv_append8(src, H * dh, (H + hkv) * dh, i32(slots), *want, **dict(kw, **({"q_out": q_want} if kw else {})))
    got, q_got = [p.to(DEV) for p in pools], torch.zeros(T, H * dh, dtype=dtype, device=DEV)
    ops().kv_append8(src.to(DEV), H * dh, (H + hkv) * dh, i32(slots).to(DEV), *got,
                     **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}, **({"q_out": q_got} if kw else {}))
    for name, a, b in zip(("keys", "values", "key scales", "value scales"), got, want):
        assert same(a, b), name
    if kw:
        assert bool(((q_got.cpu().double() - q_want.double()).abs() <= 2 * (HALF[dtype] + 2.0 ** -24) * q_want.double().abs() + 1e-300).all())


# -- attention -----------------------------------------------------------------------------------------------------------------

def attention_case(seq_lens, new_rows, H, hkv, dh, ps, dtype, seed=0, q_scale=1.0, window=0, keep=0):
    """A cache for requests of the given lengths on shuffled pages, of which request s's last new_rows[s] tokens are this step's rows.
    Places behind a request's last token and pages of nobody hold NaN; pages in front of the window are given back, but for those kept."""
    gen = torch.Generator().manual_seed(seed)
    blocks = [-(-n // ps) for n in seq_lens]
    n_pages = sum(blocks) + 3
    order = torch.randperm(n_pages, generator=gen).tolist()
    k = torch.randn(n_pages, hkv, ps, dh, generator=gen) * torch.exp(0.5 * torch.randn(n_pages, hkv, 1, 1, generator=gen))
    v = torch.randn(n_pages, hkv, dh, ps, generator=gen) * torch.exp(0.5 * torch.randn(n_pages, hkv, 1, 1, generator=gen))
    pools, scales = [], []
    for x in (k, v):
        m, e = torch.frexp(x.abs().amax(dim=(2, 3)))
        s = R.power(torch.where(2 * m <= 1.75, e - 9, e - 8)).float()
        pools.append((x / s[:, :, None, None]).to(FP8))
        scales.append(s)
    kb, vb = pools[0].view(torch.uint8), pools[1].view(torch.uint8)
    used = set()
    bt = torch.full((len(seq_lens), max(blocks) + 1), -1, dtype=torch.int32)
    tiles, wide, row = [], [], 0
    for s, (n, new) in enumerate(zip(seq_lens, new_rows)):
        for b in range(blocks[s]):
            page = order.pop()
            used.add(page)
            first_read = n - new - window + 1 if window else 0
            if (b + 1) * ps > first_read or b * ps < keep:
                bt[s, b] = page
            if n < (b + 1) * ps:
                kb[page, :, n - b * ps:] = 0x7f
                vb[page, :, :, n - b * ps:] = 0xff
        for size, got in ((16, tiles), (128, wide)):
            got += [(s, row + i, min(size, new - i), n - new + i) for i in range(0, new, size)]
        row += new
    for page in set(range(n_pages)) - used:
        kb[page], vb[page] = 0xff, 0x7f
    q = (torch.randn(row, H * dh + 8, generator=gen) * q_scale).to(dtype)[:, :H * dh]
    return q, pools + scales, bt, i32(tiles).t().contiguous(), i32(wide).t().contiguous()


def check_attention(q, pools, bt, tiles, wide, H, scale, dtype, single=False, longest=0, what="", **extras):
    want, mass, most = R.attention_exact(q, *pools, bt, tiles, H, scale, **extras)
    T, dh = q.shape[0], pools[0].shape[3]
    where = dict(extras, sink=extras["sink"].to(DEV)) if isinstance(extras.get("sink"), torch.Tensor) else extras
    on = [p.to(DEV) for p in pools]
    got = torch.full((T, H * dh + 8), 9.0, dtype=dtype, device=DEV)
    big = torch.empty(T, q.stride(0), dtype=dtype, device=DEV)
    qd = big[:, :H * dh].copy_(q)
    ops().attention8(qd, got[:, :H * dh], *on, bt.to(DEV), tiles.to(DEV), H, scale, tiles_wide=wide.to(DEV), single_rows=single,
                     max_context=longest, **where)
    assert bool((got[:, H * dh:] == 9.0).all()), what
    rows = got[:, :H * dh].cpu().double()
    assert torch.equal(rows.isnan(), want.isnan()), what
    # The bound: half a step of the result's type; of the weights as the matrix instructions take them (bfloat16 rows: rounded to bfloat16,
    # 2^-8 of each; 32-bit ones stay 32-bit), and what 32-bit sums lose: a score off by d moves a weight by d of itself, numerator and
    # denominator, d = (dh + 8) 2^-23 of scale * sum |q||k|, and sums over n keys lose n 2^-24.
    n = int(pools[0].shape[2] * bt.shape[1])
    loss = (2.0 ** -8 if dtype == BF16 else 2.0 ** -23) + 2 * (dh + 8) * 2.0 ** -23 * most.repeat_interleave(dh, 1) + 2 * n * 2.0 ** -24
    if extras.get("softcap"):
        loss = loss + 4 * extras["softcap"] * 2.0 ** -22
    bound = HALF[dtype] * want.abs() + loss * mass * 1.01 + 1e-30
    off = ((rows - want).abs() > bound) & ~want.isnan()
    assert not bool(off.any()), (what, float(((rows - want).abs() / bound)[~want.isnan()].max()))
    return got[:, :H * dh]


SHAPES = [(4, 4, 16, 16), (25, 25, 64, 16), (6, 2, 48, 8), (2, 1, 128, 64), (3, 3, 256, 16), (8, 2, 32, 16), (5, 5, 80, 32), (4, 2, 15, 16),
          (3, 3, 100, 5), (2, 1, 250, 16), (5, 5, 1, 16), (32, 8, 128, 16), (40, 2, 64, 16), (8, 8, 112, 48), (4, 2, 192, 32), (17, 1, 96, 16)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh,ps", SHAPES)
def test_attention_portions(dtype, H, hkv, dh, ps):
    # a decoded token far into a context, a whole prompt, a portion, a first token
    case = attention_case([300, 70, 133, 1], [1, 70, 21, 1], H, hkv, dh, ps, dtype, seed=H + dh)
    check_attention(*case, H, dh ** -0.5, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh,ps", SHAPES)
def test_attention_single_rows(dtype, H, hkv, dh, ps):
    lens = [300, 1, 64, 65, 17, 128]
    case = attention_case(lens, [1] * len(lens), H, hkv, dh, ps, dtype, seed=H + dh)
    check_attention(*case, H, dh ** -0.5, dtype, single=True, longest=300)


EXTRAS = [dict(window=20), dict(window=64, keep_first=4), dict(window=1), dict(window=33, keep_first=70, sink=True), dict(softcap=5.0),
          dict(sink=True), dict(softcap=20.0, sink=True, window=100, keep_first=1)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh,ps", [(4, 4, 64, 16), (8, 2, 128, 32), (6, 3, 80, 16), (4, 2, 20, 8)])
@pytest.mark.parametrize("extras", EXTRAS, ids=str)
def test_attention_extras(dtype, H, hkv, dh, ps, extras):
    kw = dict(extras)
    if kw.get("sink") and kw.get("window") != 33:
        kw["sink"] = torch.linspace(-2, 3, H)
    for lens, new, single in (([300, 70, 133, 1], [1, 70, 21, 1], False), ([300, 1, 64, 129], [1] * 4, True)):
        case = attention_case(lens, new, H, hkv, dh, ps, dtype, seed=7, q_scale=2.0, window=kw.get("window", 0), keep=kw.get("keep_first", 0))
        check_attention(*case, H, dh ** -0.5, dtype, single=single, longest=max(lens), what=(single,), **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_long_contexts(dtype):
    """Contexts that are split over workgroups, and portions behind them, with lengths around the places where tiles end."""
    for H, hkv, dh, ps in ((2, 2, 64, 16), (8, 2, 128, 16)):
        for lens in ([2500], [1023, 1025, 4097]):
            case = attention_case(lens, [1] * len(lens), H, hkv, dh, ps, dtype, seed=5)
            check_attention(*case, H, dh ** -0.5, dtype, single=True, longest=max(lens), what=("single", lens))
        case = attention_case([1500, 700], [130, 257], H, hkv, dh, ps, dtype, seed=6)
        check_attention(*case, H, dh ** -0.5, dtype, what="portions")
        case = attention_case([2500, 30], [40, 3], H, hkv, dh, ps, dtype, seed=7)
        assert ops()._portions8_splits(2 * H * 2, 2, dh, 2500, 0, 0) > 1
        check_attention(*case, H, dh ** -0.5, dtype, longest=2500, what="few rows")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 24])
def test_attention_nan_reaches_only_the_rows_that_read_it(dtype, window):
    """A key and a value that are NaN inside a portion: rows before them do not read them, nor do rows whose window has passed them."""
    H, hkv, dh, ps = 4, 2, 64, 16
    q, pools, bt, tiles, wide = attention_case([140], [140], H, hkv, dh, ps, dtype, seed=8)
    for pos, which in ((37, 0), (90, 1)):
        page = int(bt[0, pos // ps])
        if which == 0:
            pools[0].view(torch.uint8)[page, 0, pos % ps, 3] = 0x7f
        else:
            pools[1].view(torch.uint8)[page, 1, 5, pos % ps] = 0xff
    check_attention(q, pools, bt, tiles, wide, H, dh ** -0.5, dtype, window=window)
    lens = [140, 95, 90]
    q, pools, bt, tiles, wide = attention_case(lens, [1] * 3, H, hkv, dh, ps, dtype, seed=9)
    for s in range(3):
        page = int(bt[s, 5])
        pools[0].view(torch.uint8)[page, 0, 9, 3] = 0x7f      # position 89
        pools[1].view(torch.uint8)[page, 1, 5, 10] = 0x7f     # position 90: behind the last one's end
    check_attention(q, pools, bt, tiles, wide, H, dh ** -0.5, dtype, single=True, longest=140, window=window)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dh,bad", [(64, math.nan), (96, math.inf), (20, math.nan)])
@pytest.mark.parametrize("window", [0, 24])
def test_attention_scales_of_pages_that_nobody_reads(dtype, dh, bad, window):
    """Scales that are no numbers, of pages that no row has, the pools' first among them, and of a page behind the window."""
    for lens, new, single in (([140, 95, 20], [140, 21, 1], False), ([140, 95, 20], [1] * 3, True)):
        q, pools, bt, tiles, wide = attention_case(lens, new, 4, 2, dh, 16, dtype, seed=15, window=window)
        k, v = (torch.cat([p.view(torch.uint8)[:1], p.view(torch.uint8)]) for p in pools[:2])
        k[0] = v[0] = 0x55
        ks, vs = (torch.cat([torch.full((1, 2), bad), s]) for s in pools[2:])
        bt = torch.where(bt >= 0, bt + 1, bt)
        unread = sorted(set(range(k.shape[0])) - set(bt.flatten().tolist()))
        assert 0 in unread
        ks[unread] = vs[unread] = bad
        if window and single:      # the page is still in the table, in the tile of 64 keys that the window begins in
            bt[0, 4] = unread[-1]
        check_attention(q, [k.view(FP8), v.view(FP8), ks, vs], bt, tiles, wide, 4, dh ** -0.5, dtype, single=single, longest=140, window=window)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_values_at_the_end_of_the_range(dtype):
    """A value that has become 2^128 (256 times the scale 2^120) in a portion: the rows before it are as without it."""
    q, pools, bt, tiles, wide = attention_case([70], [70], 4, 2, 64, 16, dtype, seed=16)
    q, pools = q.contiguous().to(DEV), [p.to(DEV) for p in pools]
    bt, tiles, wide = bt.to(DEV), tiles.to(DEV), wide.to(DEV)
    clean = ops().attention8(q, torch.empty_like(q), *pools, bt, tiles, 4, 0.125, tiles_wide=wide)
    page = int(bt[0, 3])                                           # positions 48 to 63
    pools[3][page] = 2.0 ** 120
    pools[1].view(torch.uint8)[page] = 0x78 | 0x80
    got = ops().attention8(q, torch.empty_like(q), *pools, bt, tiles, 4, 0.125, tiles_wide=wide)
    assert torch.equal(got[:48], clean[:48])
    # one key of such a value, the others' are zeros: weight times 240 2^120, the value's rounding of up to 2^-4 taken off again
    assert bool((got[48].float() < -2.0 ** 100).all()) and bool(got[48].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_rows_that_read_nothing_and_padding(dtype):
    """A request all of whose pages are given back reads nothing: zeros; rows of padding tiles are left as they were."""
    H, hkv, dh, ps = 4, 2, 64, 16
    for new, single in (([1, 1, 1], True), ([20, 1, 30], False)):
        q, pools, bt, tiles, wide = attention_case([40, 50, 60], new, H, hkv, dh, ps, dtype, seed=10)
        bt[1] = -1
        row = sum(new[:2])
        tiles[0][tiles[1] >= row] = -1
        wide[0][wide[1] >= row] = -1
        T = q.shape[0]
        got = torch.full((T, H * dh), 9.0, dtype=dtype, device=DEV)
        want, _, _ = R.attention_exact(q, *pools, bt, tiles, H, dh ** -0.5)
        ops().attention8(q.to(DEV), got, *[p.to(DEV) for p in pools], bt.to(DEV), tiles.to(DEV), H, dh ** -0.5, tiles_wide=wide.to(DEV),
                         single_rows=single, max_context=60)
        assert bool((got[row:] == 9.0).all()) and bool((got[row - 1] == 0).all())
        assert torch.allclose(got[:row].cpu().double(), want[:row], atol=0.02, rtol=0.02)
        sunk = torch.full((T, H * dh), 9.0, dtype=dtype, device=DEV)
        ops().attention8(q.to(DEV), sunk, *[p.to(DEV) for p in pools], bt.to(DEV), tiles.to(DEV), H, dh ** -0.5, tiles_wide=wide.to(DEV),
                         single_rows=single, max_context=60, sink=True)
        assert bool((sunk[row - 1] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh", [(4, 2, 16), (2, 2, 64), (4, 1, 80), (3, 3, 96), (3, 3, 128)])
@pytest.mark.parametrize("shape", [(4, 1), (4, 2), (2, 2)], ids=str)
def test_attention_portions_in_every_shape(monkeypatch, dtype, H, hkv, dh, shape):
    """Every shape of workgroup of the portions' kernel, not only the one that its rule picks for this little work."""
    if dh > 96 and shape != (4, 1) and dtype == F32:
        pytest.skip("not a shape for these heads")
    o = ops()
    monkeypatch.setattr(o, "_portions8_shape", lambda *a: shape)
    kw = dict(window=150, keep_first=5, sink=True) if dh == 64 else dict(softcap=10.0) if dh == 80 else {}
    case = attention_case([300, 260, 133, 65], [1, 260, 21, 33], H, hkv, dh, 16, dtype, seed=dh, window=kw.get("window", 0), keep=kw.get("keep_first", 0))
    check_attention(*case, H, dh ** -0.5, dtype, what=shape, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh", [(4, 2, 16), (2, 2, 64), (4, 1, 80), (3, 3, 128), (2, 1, 208)])
@pytest.mark.parametrize("splits", [2, 3, 20])
def test_attention_portions_shared_out(monkeypatch, dtype, H, hkv, dh, splits):
    """A tile's keys shared out to several workgroups, more workgroups than steps among them."""
    o = ops()
    monkeypatch.setattr(o, "_portions8_splits", lambda *a: splits)
    kw = dict(window=150, keep_first=5, sink=True) if dh == 64 else dict(softcap=10.0, sink=torch.linspace(-2, 3, H)) if dh == 80 else {}
    case = attention_case([1100, 260, 133, 65], [1, 260, 21, 33], H, hkv, dh, 16, dtype, seed=dh, window=kw.get("window", 0), keep=kw.get("keep_first", 0))
    check_attention(*case, H, dh ** -0.5, dtype, what=splits, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 24])
def test_attention_portions_shared_out_nan_and_padding(monkeypatch, dtype, window):
    """Keys and values that are NaN in some workgroups' shares reach the rows that read them; a row that reads nothing; rows of no tile."""
    H, hkv, dh, ps = 4, 2, 64, 16
    o = ops()
    monkeypatch.setattr(o, "_portions8_splits", lambda *a: 3)
    q, pools, bt, tiles, wide = attention_case([600], [140], H, hkv, dh, ps, dtype, seed=8)
    for pos, which in ((37, 0), (490, 0), (470, 1), (90, 1)):
        pools[which].view(torch.uint8)[int(bt[0, pos // ps]), which, (pos % ps, 5)[which], (3, pos % ps)[which]] = 0x7f
    check_attention(q, pools, bt, tiles, wide, H, dh ** -0.5, dtype, window=window)
    q, pools, bt, tiles, wide = attention_case([400, 50, 600], [20, 1, 30], H, hkv, dh, ps, dtype, seed=10)
    bt[1] = -1
    wide[0, 2] = -1
    got = torch.full((51, H * dh), 9.0, dtype=dtype, device=DEV)
    want, _, _ = R.attention_exact(q, *pools, bt, tiles, H, dh ** -0.5)
    o.attention8(q.to(DEV), got, *[p.to(DEV) for p in pools], bt.to(DEV), tiles.to(DEV), H, dh ** -0.5, tiles_wide=wide.to(DEV), max_context=600)
    assert bool((got[21:] == 9.0).all()) and bool((got[20] == 0).all())
    assert torch.allclose(got[:20].cpu().double(), want[:20], atol=0.02, rtol=0.02)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,hkv,dh", [(4, 2, 16), (40, 2, 64), (3, 3, 128), (2, 1, 208)])
@pytest.mark.parametrize("splits", [1, 2, 3, 20])
def test_attention_single_rows_in_every_shape(monkeypatch, dtype, H, hkv, dh, splits):
    """Every number of workgroups that share a row's keys out, more workgroups than tiles of keys among them."""
    o = ops()
    monkeypatch.setattr(o, "_single8_splits", lambda *a: splits)
    kw = dict(window=150, keep_first=5, sink=True) if dh == 64 else {}
    lens = [700, 1, 64, 300]
    case = attention_case(lens, [1] * 4, H, hkv, dh, 16, dtype, seed=dh, window=kw.get("window", 0), keep=kw.get("keep_first", 0))
    check_attention(*case, H, dh ** -0.5, dtype, single=True, longest=700, what=splits, **kw)


def test_attention_shapes_are_refused_by_the_entries():
    o = ops()
    q = torch.zeros(1, 256, dtype=BF16, device=DEV)
    p = [t.to(DEV) for t in random_pools(2, 1, 16, 256, torch.Generator().manual_seed(0))]
    bt, tiles = torch.zeros(1, 1, dtype=torch.int32, device=DEV), i32([[0], [0], [1], [0]]).to(DEV)
    for name, shape, kw in (("_single8_splits", 0, dict(single_rows=True, max_context=1)), ("_portions8_shape", (2, 2), dict(tiles_wide=tiles)),
                            ("_portions8_splits", 0, dict(tiles_wide=tiles))):
        real = getattr(o, name)
        setattr(o, name, lambda *a: shape)
        try:
            with pytest.raises(o.KernelError, match="sizes"):
                o.attention8(q, torch.empty_like(q), *p, bt, tiles, 1, 1.0, **kw)
        finally:
            setattr(o, name, real)


def test_attention_scales_that_are_not_positive():
    """A scale below zero (the portions' kernel takes the largest product for the largest score: it goes the plain way) and zero."""
    case = attention_case([100, 70], [40, 70], 4, 2, 64, 16, BF16, seed=12)
    for scale in (-0.125, 0.0):
        q, pools, bt, tiles, wide = case
        want, mass, most = R.attention_exact(q, *pools, bt, tiles, 4, scale)
        got = torch.empty(q.shape[0], 256, dtype=BF16, device=DEV)
        ops().attention8(q.to(DEV), got, *[p.to(DEV) for p in pools], bt.to(DEV), tiles.to(DEV), 4, scale, tiles_wide=wide.to(DEV))
        loss = 2.0 ** -23 + 2 * 72 * 2.0 ** -23 * most.abs().repeat_interleave(64, 1) + 2 * 128 * 2.0 ** -24
        assert bool(((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + loss * mass * 1.01 + 1e-30).all())


def test_calls_on_another_stream_and_two_at_once():
    """Two streams that use the operators at once, each on tensors of its own, get what one after the other gives."""
    gen = torch.Generator().manual_seed(13)
    hkv, dh, ps, H = 4, 64, 16, 8
    lens = [900, 33, 517]

    def state(seed):
        q, pools, bt, tiles, wide = attention_case(lens, [1] * 3, H, hkv, dh, ps, BF16, seed=seed)
        src = torch.randn(3, 2 * hkv * dh, generator=gen).to(BF16).to(DEV)
        slots = i32([int(bt[s, (n - 1) // ps]) * ps + (n - 1) % ps for s, n in enumerate(lens)]).to(DEV)
        return [t.to(DEV) for t in (q, bt, tiles)], [p.to(DEV) for p in pools], src, slots

    def run(st):
        (q, bt, tiles), pools, src, slots = st
        out = []
        for _ in range(20):
            ops().kv_append8(src, 0, hkv * dh, slots, *pools)
            out.append(ops().attention8(q, torch.empty_like(q), *pools, bt, tiles, H, 0.125, single_rows=True, max_context=900))
        return out
    states = [state(20), state(21)]
    want = [run((s[0], [p.clone() for p in s[1]], *s[2:])) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = []
    for st, stream in zip(states, streams):
        with torch.cuda.stream(stream):
            got.append(run(st))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_two_captured_graphs_of_a_step():
    """Append and attention captured together, twice over different caches; the graphs are replayed in turn with eager work and
    synchronizations between them, and every replay gives the eager result (the split results' workspaces are the graphs' own)."""
    hkv, dh, ps, H = 2, 128, 16, 8

    def state(seed, n):
        q, pools, bt, tiles, wide = attention_case([n], [1], H, hkv, dh, ps, BF16, seed=seed)
        src = torch.randn(1, (H + 2 * hkv) * dh, generator=torch.Generator().manual_seed(seed)).to(BF16)
        slot = i32([int(bt[0, (n - 1) // ps]) * ps + (n - 1) % ps])
        freq = (10000.0 ** (-torch.arange(dh // 2).double() * 2 / dh)).float()
        return [t.to(DEV) for t in (src, slot, i32([n - 1]), freq, bt, tiles)], [p.to(DEV) for p in pools], n

    def step(st, pools):
        (src, slot, pos, freq, bt, tiles), _, n = st
        turned = torch.empty(1, H * dh, dtype=BF16, device=DEV)
        ops().kv_append8(src, H * dh, (H + hkv) * dh, slot, *pools, positions=pos, freq=freq, q_out=turned, q_col=0, n_heads=H)
        return ops().attention8(turned, torch.empty_like(turned), *pools, bt, tiles, H, dh ** -0.5, single_rows=True, max_context=n)
    states = [state(31, 6000), state(32, 4100)]
    want = [step(s, [p.clone() for p in s[1]]) for s in states]
    assert ops()._single8_splits(1, H, hkv, dh, 6000, 0, 0) > 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in states:
            step(s, [p.clone() for p in s[1]])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s, s[1]))
        graphs.append(g)
    for turn in range(4):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        x = torch.randn(256, 256, device=DEV)
        (x @ x).sum().item()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), turn


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("longest", [0, 2300])
def test_a_captured_portion(dtype, longest):
    """Portions whose tiles take more LDS than a workgroup has by itself, captured before they have run otherwise; replays with eager
    work between them.  With keys shared out the results to be joined are the graph's own memory."""
    H, hkv, dh, ps = 8, 2, 128, 32
    q, pools, bt, tiles, wide = [x if isinstance(x, list) else x.to(DEV) for x in attention_case([2300, 77], [130, 77], H, hkv, dh, ps, dtype, seed=33)]
    pools = [p.to(DEV) for p in pools]
    out = torch.zeros(q.shape[0], H * dh, dtype=dtype, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops().attention8(q, out, *pools, bt, tiles, H, 0.088, tiles_wide=wide, max_context=longest)
    want = ops().attention8(q, torch.zeros_like(out), *pools, bt, tiles, H, 0.088, tiles_wide=wide, max_context=longest)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        (pools[2].sum() + 1).item()


def test_long_caches_pass_32_bits():
    """Pools of more than 2^31 numbers, the pages at their end."""
    hkv, dh, ps, H = 2, 256, 16, 4
    n_pages = (1 << 31) // (hkv * ps * dh) + 40
    k = torch.zeros(n_pages, hkv, ps, dh, dtype=torch.uint8, device=DEV).view(FP8)
    v = torch.zeros(n_pages, hkv, dh, ps, dtype=torch.uint8, device=DEV).view(FP8)
    ks, vs = torch.ones(n_pages, hkv, device=DEV), torch.ones(n_pages, hkv, device=DEV)
    gen = torch.Generator().manual_seed(14)
    n = 40
    pages = [n_pages - 1, n_pages - 17, n_pages - 30]
    src = torch.randn(n, (H + 2 * hkv) * dh, generator=gen).to(BF16)
    slots = i32([pages[i // ps] * ps + i % ps for i in range(n)])
    ops().kv_append8(src.to(DEV), H * dh, (H + hkv) * dh, slots.to(DEV), k, v, ks, vs)
    small = [torch.zeros(3, hkv, ps, dh, dtype=FP8), torch.zeros(3, hkv, dh, ps, dtype=FP8), torch.zeros(3, hkv), torch.zeros(3, hkv)]
    R.kv_append8(src, H * dh, (H + hkv) * dh, i32(range(n)), *small)
    for big, want in zip((k, v, ks, vs), small):
        assert same(torch.stack([big[p] for p in pages]), want)
    bt, tiles = i32([pages]), i32([[0, 0, 0], [0, 16, 32], [16, 16, 8], [0, 16, 32]])
    wide = i32([[0], [0], [n], [0]])
    q = src[:, :H * dh].contiguous()
    want, _, _ = R.attention_exact(q, *small, i32([[0, 1, 2]]), tiles, H, 0.0625)
    for dtype in (BF16, F32):
        for kw in (dict(tiles_wide=wide.to(DEV)), dict()):
            got = ops().attention8(q.to(dtype).to(DEV), torch.empty(n, H * dh, dtype=dtype, device=DEV), k, v, ks, vs, bt.to(DEV), tiles.to(DEV), H, 0.0625, **kw)
            assert torch.allclose(got.cpu().double(), want, atol=0.03, rtol=0.02)
        one = i32([[0], [0], [1], [n - 1]]).to(DEV)
        got = ops().attention8(q[n - 1:].to(dtype).to(DEV), torch.empty(1, H * dh, dtype=dtype, device=DEV), k, v, ks, vs, bt.to(DEV), one, H, 0.0625,
                               single_rows=True, max_context=n)
        assert torch.allclose(got.cpu().double(), want[n - 1:], atol=0.03, rtol=0.02)
