"""The operators of a paged cache held in 8 bits, as a step of the engine calls them.

The cache: pages of `page` tokens, keys [pages, heads, page, dim] and values [pages, heads, dim, page], as e4m3 numbers, and for
every page and head one 32-bit scale, a power of two; what a number stands for is the number times its page's and head's scale.

* "append": a step's rows of projected queries, keys and values; queries and keys are turned by their positions (in pairs or in
  halves, or not at all), and keys and values are added to the pages.  In a page and head that gets rows:
      a row in the page's first place begins the page anew (nothing of what it held counts, its other places become zero);
      the scale 2^e is the smallest power of two with which the largest new magnitude is at most 448, and no smaller than
      the scale that the page has if it does not begin anew (and at least 2^-117);
      new numbers are the nearest e4m3 numbers to value / 2^e, ties to the even one; what the page holds already is rounded in
      the same way where its scale grew.
  Outputs: the turned queries, the pages and the scales.
* "attend": causal attention of the step's rows (single rows of many requests, or portions of prompts) over such a cache, with a
  window that may keep the first keys, a sink per head and a soft cap.  Query head h reads key head h // (heads / key heads).
      s = scale * q . k, capped to cap * tanh(s / cap) where a cap is set; softmax over the keys that the row reads (a sink adds
      exp(sink[h]) under the softmax); the sum of the values weighted so.
  Outputs: a row per query row.

Sizes come from the repository's GPT-2 shapes (heads of 64, 25 of them in the largest) and from a generic one with grouped key heads
(32 over 8, heads of 128).  Lengths of contexts and portions are spread between `low` and `high` and do not change with the seed.
"""
import random

import torch

own = False

GPT2 = dict(heads=25, kv=25, dim=64)
GROUPED = dict(heads=32, kv=8, dim=128)


def _append(name, **more):
    return dict(dict(name=name, op="append", dtype="bfloat16", page=16, turn="none", dims=0, base=10000.0, requests=1, low=0, high=0,
                     rows_low=1, rows_high=1), **more)


def _attend(name, **more):
    return dict(dict(name=name, op="attend", dtype="bfloat16", page=16, requests=1, low=0, high=0, rows_low=1, rows_high=1, window=0,
                     keep=0, sink=False, cap=0.0), **more)


def listed():
    return [
        # one user's next token, GPT-2 XL: nothing is turned, latency alone
        _append("append b1", **GPT2, low=517, high=517),
        # a loaded server's decode step: a row for each of 64 requests, pairs turned
        _append("append b64", **GROUPED, turn="pairs", dims=128, low=100, high=3000, requests=64),
        # three prompts' portions in one step, none of them a multiple of a page, one behind a context, halves turned in part
        _append("append portions", **GROUPED, turn="halves", dims=96, base=500000.0, low=0, high=1001, requests=3, rows_low=519, rows_high=905),
        # the 32-bit engine's prompt, pages of 32
        _append("append f32 prompt", **GPT2, dtype="float32", page=32, turn="pairs", dims=64, requests=1, rows_low=1023, rows_high=1023),
        # one user's next token, GPT-2 XL
        _attend("attend b1", **GPT2, low=517, high=517),
        # one user, a whole book in the cache: the context has to be shared out over the card
        _attend("attend b1 long", **GROUPED, low=131071, high=131071),
        # a loaded server with GPT-2 XL
        _attend("attend b64", **GPT2, requests=64, low=100, high=1020),
        # many users with long contexts in a window that keeps the first keys, a sink per head, a soft cap
        _attend("attend window b16", **GROUPED, requests=16, low=900, high=30000, window=4096, keep=4, sink=True, cap=30.0),
        # the 32-bit engine's decode step
        _attend("attend f32 b8", **GPT2, dtype="float32", requests=8, low=384, high=1000),
        # GPT-2 XL's prompt phase: two full prompts in one step
        _attend("attend 2x1024", **GPT2, requests=2, rows_low=1024, rows_high=1024),
        # portions of three long prompts behind what is there already
        _attend("attend portions", **GROUPED, requests=3, low=2001, high=8192, rows_low=300, rows_high=1024),
        # the 32-bit engine's prompt
        _attend("attend f32 prompt", **GPT2, dtype="float32", page=32, rows_low=1001, rows_high=1001),
    ]


def _log_int(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    """One more case of the same ranges: heads shared or not, head sizes, pages, numbers of requests, lengths, options."""
    append = rng.random() < 0.4
    kv = rng.choice([1, 2, 4, 5, 8, 8, 12, 16, 25])
    c = dict(kv=kv, heads=kv * rng.choice([1, 1, 2, 4, 5, 8]), dim=rng.choice([48, 64, 64, 80, 96, 128, 128, 256]), dtype=rng.choice(["bfloat16"] * 3 + ["float32"]),
             page=rng.choice([16, 16, 16, 32, 64]))
    if c["heads"] > 40:
        c["heads"] = c["kv"]
    portions = rng.random() < 0.4
    if append:
        c = _append("", **c, turn=rng.choice(["none", "pairs", "halves"]), requests=_log_int(rng, 1, 6 if portions else 128))
        c["dims"] = 0 if c["turn"] == "none" else c["dim"] // rng.choice([1, 1, 2])
        c["base"] = rng.choice([10000.0, 500000.0])
        a, b = _log_int(rng, 1, 6000), _log_int(rng, 1, 6000)
    else:
        c = _attend("", **c, requests=_log_int(rng, 1, 4 if portions else 100))
        if rng.random() < 0.4:
            c.update(window=_log_int(rng, 20, 4000), keep=rng.choice([0, 1, 4, 70]))
        c.update(sink=rng.random() < 0.4, cap=rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]))
        most = 4000 if portions else max(64, min(60000, 100000 // c["requests"]))
        a, b = _log_int(rng, 1, most), _log_int(rng, 1, most)
    c.update(low=min(a, b), high=max(a, b))
    if portions:
        a, b = _log_int(rng, 2, 900), _log_int(rng, 2, 900)
        c.update(rows_low=min(a, b), rows_high=max(a, b))
    del c["name"]
    same = [work(k) for k in listed() if k["op"] == c["op"] and k["dtype"] == c["dtype"]]
    most = {k: max(w[k] for w in same) for k in ("bytes", "flops")}
    while any(work(c)[k] > most[k] for k in most) and (c["requests"] > 1 or c["rows_high"] > 1 or c["high"] > 1):
        if c["requests"] > 1:
            c["requests"] = c["requests"] * 3 // 4
        else:
            c.update({k: max(1 if "high" in k or k.startswith("rows") else 0, c[k] * 3 // 4) for k in ("low", "high", "rows_low", "rows_high")})
    return c


def _lengths(case):
    """-> (tokens in the cache before the step, rows that the step brings) of every request."""
    n = case["requests"]

    def spread(low, high, order):
        got = [low + (high - low) * k // max(1, n - 1) for k in range(n)]
        random.Random(order).shuffle(got)
        return got
    return spread(case["low"], case["high"], 1), spread(case["rows_low"], case["rows_high"], 2)


def _bytes_of(dtype):
    return 2 if dtype == "bfloat16" else 4


def work(case):
    had, rows = _lengths(case)
    T, kv, dim, heads, size = sum(rows), case["kv"], case["dim"], case["heads"], _bytes_of(case["dtype"])
    if case["op"] == "append":
        turned = 2 * heads * dim * size if case["turn"] != "none" else 0      # queries: read and written
        pages = sum((h + n - 1) // case["page"] - h // case["page"] + 1 for h, n in zip(had, rows))
        return {"bytes": float(T * (2 * kv * dim * (size + 1) + turned + 8) + pages * kv * 16),
                "flops": float(T * (kv + (heads if case["turn"] != "none" else 0)) * case["dims"] * 3)}
    pairs = keys = 0
    w, keep = case["window"], case["keep"]
    for h, n in zip(had, rows):
        for p in (range(h, h + n) if w else ()):
            pairs += min(p + 1, w + min(keep, max(0, p + 1 - w)))
        if not w:
            pairs += n * h + n * (n + 1) // 2
        first = max(0, h - w + 1) if w else 0
        keys += h + n - first + min(keep if w else 0, first)
    return {"bytes": float(2 * keys * kv * dim + 8 * kv * keys // case["page"] + 2 * T * heads * dim * size),
            "flops": float(4 * pairs * heads * dim)}


# -- what a program has in hand ---------------------------------------------------------------------------------------------

def _power(e):
    """2^e as a 32-bit number from its bits (a power taken by the library is not always exact)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pages(values):
    """values [pages, heads, ...] in 32 bits as e4m3 numbers and scales by page and head, as pages that were full when they were
    written."""
    top = values.abs().amax(dim=(2, 3))
    m, e = torch.frexp(top)
    scale = _power(torch.where(2 * m <= 1.75, e - 9, e - 8).clamp(min=-117))
    return (values / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    """A step's rows and tables, and a cache whose pages lie in any order and hold what other steps left."""
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    heads, kv, dim, ps = case["heads"], case["kv"], case["dim"], case["page"]
    had, rows = _lengths(case)
    T, S = sum(rows), len(rows)
    blocks = [-(-(h + n) // ps) for h, n in zip(had, rows)]
    n_pages = sum(blocks) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(int(seed)))
    table = torch.full((S, max(blocks)), -1, dtype=torch.int64)
    slots, positions, at = [], [], 0
    for s in range(S):
        table[s, :blocks[s]] = order[at:at + blocks[s]]
        at += blocks[s]
        p = torch.arange(had[s], had[s] + rows[s])
        positions.append(p)
        slots.append(table[s, p // ps] * ps + p % ps)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)
    loud = torch.exp(0.5 * normal(kv, 1, dim))                # some dims of a key are larger than others, in all tokens
    keys = normal(n_pages, kv, ps, dim).mul_(loud).mul_(torch.exp(0.3 * normal(n_pages, kv, 1, 1)))
    k_pool, k_scale = _pages(keys)
    del keys
    values = normal(n_pages, kv, dim, ps).mul_(torch.exp(0.3 * normal(n_pages, kv, 1, 1)))
    v_pool, v_scale = _pages(values)
    del values
    state = dict(case=case, k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale, T=T,
                 positions=torch.cat(positions).to(torch.int32).to(dev), slots=torch.cat(slots).to(torch.int32).to(dev))
    if case["op"] == "append":
        # some rows are louder than what the page holds, so that its scale grows under them
        rows_in = normal(T, (heads + 2 * kv) * dim) * torch.exp(0.7 * normal(T, 1))
        i = torch.arange(case["dims"] // 2, dtype=torch.float64)
        state.update(src=rows_in.to(dtype), freq=(case["base"] ** (-2 * i / max(1, case["dims"]))).to(torch.float32).to(dev))
        return state
    tiles = {16: [], 128: []}
    at = 0
    for s in range(S):
        for size, got in tiles.items():
            got += [(s, at + i, min(size, rows[s] - i), had[s] + i) for i in range(0, rows[s], size)]
        at += rows[s]
    tiles[128].sort(key=lambda t: -(t[3] + t[2]))              # (the longest work first, as a step's tables have it)
    start = torch.tensor([0] + rows).cumsum(0)[:-1]
    seq = torch.repeat_interleave(torch.arange(S), torch.tensor(rows))
    spot = torch.arange(T) - start[seq]
    most = torch.arange(max(rows))
    state.update(
        q=(1.5 * normal(T, heads * dim)).to(dtype), sink=normal(heads) if case["sink"] else None,
        block_tables=table.to(torch.int32).to(dev), **{"tiles%d" % n: torch.tensor(t, dtype=torch.int32).t().contiguous().to(dev) for n, t in tiles.items()},
        # for the plain form: every request's rows side by side, padded with its last one, and where each row then stands
        padded=(start[:, None] + torch.minimum(most[None, :], torch.tensor(rows)[:, None] - 1)).to(dev), seq=seq.to(dev), spot=spot.to(dev),
        single=max(rows) == 1, longest=max(h + n for h, n in zip(had, rows)))
    return state


# -- the plain forms --------------------------------------------------------------------------------------------------------

def _nearest(x):
    """64-bit values up to 448 to the nearest e4m3 numbers, ties to even; what is not finite becomes NaN."""
    _, e = torch.frexp(x)
    step = _power((e - 1).clamp(min=-6) - 3).double()
    return torch.where(x.isfinite(), torch.round(x / step) * step, x - x).to(torch.float8_e4m3fn)


def _turned(x, s, halves):
    """x [T, heads, dim] in 64 bits, its first dims turned by the rows' positions."""
    freq, dims = s["freq"].double(), 2 * s["freq"].shape[0]
    angle = (s["positions"].double()[:, None] * freq)[:, None, :]
    c, n = angle.cos(), angle.sin()
    u, v = (x[..., :dims // 2], x[..., dims // 2:dims]) if halves else (x[..., 0:dims:2], x[..., 1:dims:2])
    a, b = u * c - v * n, v * c + u * n
    front = torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([front, x[..., dims:]], -1)


def _add_rows(new, pool, scale, page, place, tokens_last):
    """new [T, heads, dim] in 64 bits into the pages.  Every row makes its page's new numbers out of the page as it was, rows of one
    page the same ones; then the rows' own numbers go to their places."""
    n_pages, kv = scale.shape
    top = torch.zeros((n_pages, kv), dtype=torch.float64, device=new.device)
    top = top.index_reduce(0, page, torch.where(new.isfinite(), new.abs(), 0).amax(-1), "amax")[page]
    anew = torch.zeros(n_pages, dtype=torch.bool, device=new.device).index_put((page,), place == 0, accumulate=True)[page][:, None]
    m, e = torch.frexp(top)
    need = torch.where(top > 0, torch.where(2 * m <= 1.75, e - 9, e - 8), -117).clamp(min=-117)
    was = scale[page].double()
    now = torch.maximum(_power(need).double(), torch.where(anew, 0, was))
    numbers = pool.view(torch.uint8)
    held = pool.view(torch.uint8)[page].view(torch.float8_e4m3fn).double() * (was / now)[:, :, None, None]
    numbers[page] = torch.where(anew[:, :, None, None], 0, _nearest(held).view(torch.uint8))
    mine = _nearest(new / now[:, :, None]).view(torch.uint8)
    if tokens_last:
        numbers[page, :, :, place] = mine
    else:
        numbers[page, :, place, :] = mine
    scale[page] = now.float()


def _plain_append(s):
    c = s["case"]
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    x = s["src"].double().view(s["T"], heads + 2 * kv, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    page, place = s["slots"].long() // c["page"], s["slots"].long() % c["page"]
    q_out = None
    if c["turn"] != "none":
        k = _turned(k, s, c["turn"] == "halves")
        q_out = _turned(q, s, c["turn"] == "halves").to(s["src"].dtype).view(s["T"], heads * dim)
    _add_rows(k, s["k_pool"], s["k_scale"], page, place, False)
    _add_rows(v, s["v_pool"], s["v_scale"], page, place, True)
    return [q_out, s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"]]


def _plain_attend(s):
    c = s["case"]
    heads, kv, dim, ps, w = c["heads"], c["kv"], c["dim"], c["page"], c["window"]
    table = s["block_tables"].long()
    S, blocks = table.shape
    pages = table.clamp(min=0)
    k = s["k_pool"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["k_scale"][pages][..., None, None]
    v = s["v_pool"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["v_scale"][pages][..., None, None]
    k = k.transpose(1, 2).reshape(S, kv, blocks * ps, dim)                           # [S, blocks, kv, page, dim]
    v = v.permute(0, 2, 1, 4, 3).reshape(S, kv, blocks * ps, dim)                    # [S, blocks, kv, dim, page]
    rows = s["padded"]
    n = rows.shape[1]
    q = s["q"].float()[rows].view(S, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(S, kv, heads // kv * n, dim)
    score = (torch.matmul(q, k.transpose(2, 3).contiguous()) * dim ** -0.5).view(S, kv, heads // kv, n, blocks * ps)
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    key, pos = torch.arange(blocks * ps, device=rows.device), s["positions"].long()[rows][..., None]
    reads = (key <= pos) & ((key > pos - w) | (key < c["keep"]) if w else key >= 0)
    score = torch.where(reads[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].view(1, kv, heads // kv, 1, 1) - top)
    out = torch.matmul(weight.view(S, kv, heads // kv * n, blocks * ps), v).view(S, kv, heads // kv, n, dim) / total
    return out.permute(0, 3, 1, 2, 4).reshape(S, n, heads * dim)[s["seq"], s["spot"]].to(s["q"].dtype)


def run(s):
    """One pass: the operator's call."""
    c = s["case"]
    if not own:
        return _plain_append(s) if c["op"] == "append" else _plain_attend(s)
    from denno_beta_amd.kernels import ops
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    pools = (s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"])
    if c["op"] == "append":
        turn, q_out = {}, None
        if c["turn"] != "none":
            q_out = torch.empty((s["T"], heads * dim), dtype=s["src"].dtype, device=s["src"].device)
            turn = dict(positions=s["positions"], freq=s["freq"], halves=c["turn"] == "halves", q_out=q_out, q_col=0, n_heads=heads)
        ops.kv_append8(s["src"], heads * dim, (heads + kv) * dim, s["slots"], *pools, **turn)
        return [q_out, *pools]
    out = torch.empty_like(s["q"])
    return ops.attention8(s["q"], out, *pools, s["block_tables"], s["tiles16"], heads, dim ** -0.5, window=c["window"],
                          tiles_wide=s["tiles128"], single_rows=s["single"], max_context=s["longest"],
                          sink=s["sink"] if s["sink"] is not None else False, keep_first=c["keep"], softcap=c["cap"])


# -- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _e4m3_numbers(dev):
    """What the 256 bytes stand for, from the format: a sign, four bits of exponent with bias 7, three of fraction; 0x7f: NaN."""
    code = torch.arange(256, dtype=torch.float64)
    low, sign = code % 128, torch.where(code >= 128, -1.0, 1.0)
    e, f = torch.floor(low / 8), low % 8
    power = torch.tensor([2.0 ** (i - 7) for i in range(16)], dtype=torch.float64)[e.long()]
    x = torch.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * power)
    return (sign * torch.where(low == 127, float("nan"), x)).to(dev)


def _exact_round(x, number):
    """By looking the two neighbours up among the numbers."""
    grid = number[:127].contiguous()
    a = x.abs()
    below = (torch.bucketize(a, grid, right=True) - 1).clamp(0, 126)
    above = (below + 1).clamp(max=126)
    d0, d1 = a - grid[below], grid[above] - a
    up = (d1 < d0) | ((d1 == d0) & (below % 2 == 1))
    return torch.copysign(grid[torch.where(up, above, below)], x)


def exact(case, seed):
    s = prepare(case, seed)
    dev = s["src"].device if case["op"] == "append" else s["q"].device
    number = _e4m3_numbers(dev)
    heads, kv, dim, ps = case["heads"], case["kv"], case["dim"], case["page"]
    k, v = number[s["k_pool"].view(torch.uint8).long()], number[s["v_pool"].view(torch.uint8).long()].transpose(2, 3)
    ks, vs = s["k_scale"].double(), s["v_scale"].double()
    had, rows = _lengths(case)
    if case["op"] == "append":
        v = v.contiguous()
        x = s["src"].double()
        parts = {"q": x[:, :heads * dim].clone().view(-1, heads, dim), "k": x[:, heads * dim:(heads + kv) * dim].clone().view(-1, kv, dim),
                 "v": x[:, (heads + kv) * dim:].view(-1, kv, dim)}
        half = case["dims"] // 2
        if case["turn"] != "none":
            first = torch.arange(half, device=dev) if case["turn"] == "halves" else 2 * torch.arange(half, device=dev)
            second = first + (half if case["turn"] == "halves" else 1)
            turn = torch.polar(torch.ones((s["T"], half), dtype=torch.float64, device=dev), s["positions"].double()[:, None] * s["freq"].double())
            for name in ("q", "k"):
                z = torch.complex(parts[name][:, :, first], parts[name][:, :, second]) * turn[:, None, :]
                parts[name][:, :, first], parts[name][:, :, second] = z.real, z.imag
        powers = torch.tensor([2.0 ** i for i in range(-200, 200)], dtype=torch.float64).to(dev)
        slots, at = s["slots"].tolist(), 0
        while at < len(slots):
            end = at
            while end < len(slots) and slots[end] // ps == slots[at] // ps:
                end += 1
            page, a, b = slots[at] // ps, slots[at] % ps, slots[at] % ps + end - at
            for held, scale, new in ((k, ks, parts["k"][at:end]), (v, vs, parts["v"][at:end])):
                e = torch.ceil(torch.log2(new.abs().amax(dim=(0, 2)) / 448)).clamp(min=-117)
                size = powers[e.long() + 200]
                if a > 0:
                    size = torch.maximum(size, scale[page])
                    held[page] = _exact_round(held[page] * (scale[page] / size)[:, None, None], number)
                else:
                    held[page] = 0
                held[page, :, a:b] = _exact_round(new / size[None, :, None], number).transpose(0, 1)
                scale[page] = size
            at = end
        return [parts["q"].reshape(-1, heads * dim) if case["turn"] != "none" else None, k, v.transpose(2, 3).contiguous(), ks, vs]
    table = s["block_tables"].long()
    out, at = torch.empty((s["T"], heads, dim), dtype=torch.float64, device=dev), 0
    for r, (h, n) in enumerate(zip(had, rows)):
        pages = table[r][:-(-(h + n) // ps)]
        pos = torch.arange(h, h + n, device=dev)[:, None]
        key = torch.arange(h + n, device=dev)[None, :]
        hidden = key > pos
        if case["window"]:
            hidden |= (key <= pos - case["window"]) & (key >= case["keep"])
        for g in range(kv):
            kk = (k[pages, g] * ks[pages, g][:, None, None]).reshape(-1, dim)[:h + n]
            vv = (v[pages, g] * vs[pages, g][:, None, None]).reshape(-1, dim)[:h + n]
            for head in range(g * heads // kv, (g + 1) * heads // kv):
                z = s["q"][at:at + n, head * dim:(head + 1) * dim].double() @ kk.t() / dim ** 0.5
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                z = z.masked_fill(hidden, float("-inf"))
                if s["sink"] is not None:
                    z = torch.cat([z, s["sink"][head].double().expand(n, 1)], 1)
                out[at:at + n, head] = torch.softmax(z, 1)[:, :h + n] @ vv
        at += n
    return out.view(-1, heads * dim)
