"""The cache in 8 bits from its definition, in 64 bits on the CPU: what `ops.kv_append8` and `ops.attention8` are compared with, and, under
the same names and arguments, what stands in their place where the engine runs without a GPU (`emulated`)."""
from __future__ import annotations

import contextlib
import math

import torch

FP8 = torch.float8_e4m3fn
POWERS = torch.tensor([2.0 ** i for i in range(-300, 300)], dtype=torch.float64)


def power(e):
    return POWERS[e.long() + 300]


def nearest(x):
    """64-bit values up to 448 in magnitude to the nearest e4m3 numbers, ties to even; not finite: NaN."""
    _, e = torch.frexp(x)
    step = power((e - 1).clamp(min=-6) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, torch.full_like(x, math.nan)).float().to(FP8)


def turned(x, positions, freq, halves, mag):
    """x [T, heads, dh] 64-bit."""
    dims = 2 * freq.numel()
    a = positions.double()[:, None] * freq.double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    u, v = (x[..., :dims // 2], x[..., dims // 2:dims]) if halves else (x[..., 0:dims:2], x[..., 1:dims:2])
    p, q = (u * c - v * s) * mag, (v * c + u * s) * mag
    front = torch.cat([p, q], -1) if halves else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([front, x[..., dims:]], -1)


def store(new, slots, pool, scale, ps, tokens_last):
    """new [T, heads, dh] 64-bit into pool (e4m3, on the CPU) and scale, run of rows by run of rows."""
    t = 0
    while t < len(slots):
        page = slots[t] // ps
        if slots[t] < 0 or page >= pool.shape[0]:
            t += 1
            continue
        end = t
        while end < len(slots) and slots[end] >= 0 and slots[end] // ps == page:
            end += 1
        places = [s % ps for s in slots[t:end]]
        x = new[t:end]
        held = pool[page].double()
        held = held.transpose(1, 2).clone() if tokens_last else held.clone()        # [heads, ps, dh]
        for h in range(x.shape[1]):
            fine = x[:, h][x[:, h].isfinite()].abs()
            top = float(fine.max()) if fine.numel() else 0.0
            e = -117
            if top > 0:
                m, k = math.frexp(top)
                e = max(-117, k - 9 if 2 * m <= 1.75 else k - 8)
            was = 0.0 if 0 in places else float(scale[page, h])
            now = max(2.0 ** e, was)
            if 0 in places:
                held[h] = 0
            elif now != was:
                held[h] = nearest(held[h] * (was / now)).double()
            for r, place in enumerate(places):
                held[h, place] = nearest(x[r, h] / now).double()
            scale[page, h] = now
        pool[page] = (held.transpose(1, 2) if tokens_last else held).float().to(FP8)
        t = end


def kv_append8(src, k_col, v_col, slot_map, k_pool, v_pool, k_scale, v_scale, positions=None, freq=None, halves=False, mag=1.0,
               q_out=None, q_col=0, n_heads=0):
    _, hkv, ps, dh = k_pool.shape
    T, w, slots = src.shape[0], hkv * dh, slot_map.tolist()
    x = src.detach().cpu().double()
    k, v = x[:, k_col:k_col + w].view(T, hkv, dh), x[:, v_col:v_col + w].view(T, hkv, dh)
    if freq is not None:
        pos, f = positions.cpu(), freq.cpu()
        k = turned(k, pos, f, halves, float(torch.tensor(mag, dtype=torch.float32)))
        if q_out is not None:
            q = turned(x[:, q_col:q_col + n_heads * dh].view(T, n_heads, dh), pos, f, halves, float(torch.tensor(mag, dtype=torch.float32)))
            q_out.copy_(q.reshape(T, n_heads * dh))
    for new, pool, scale, last in ((k, k_pool, k_scale, False), (v, v_pool, v_scale, True)):
        p, s = pool.cpu().clone(), scale.cpu().clone()
        store(new, slots, p, s, ps, last)
        pool.copy_(p), scale.copy_(s)


def attention_exact(q, k_pool, v_pool, k_scale, v_scale, block_tables, tiles, n_heads, scale, window=0, sink=False, keep_first=0,
                    softcap=0.0):
    """-> (rows [T, H dh] 64-bit, NaN where no tile has the row; for every entry the sum of weight * |value|, and for every row and head the
    largest scale * sum |q| |k|), all on the CPU."""
    n_pages, hkv, ps, dh = k_pool.shape
    group, T = n_heads // hkv, q.shape[0]
    kf = k_pool.cpu().double() * k_scale.cpu().double()[:, :, None, None]
    vf = v_pool.cpu().double() * v_scale.cpu().double()[:, :, None, None]
    x, bt = q.cpu().double(), block_tables.cpu()
    out = torch.full((T, n_heads, dh), math.nan, dtype=torch.float64)
    mass, most = torch.zeros_like(out), torch.zeros((T, n_heads), dtype=torch.float64)
    at = sink.cpu().double() if isinstance(sink, torch.Tensor) else torch.zeros(n_heads, dtype=torch.float64) if sink else None
    for seq, row0, nrows, pos0 in zip(*tiles.cpu().tolist()):
        for r in range(nrows if seq >= 0 else 0):
            pos = pos0 + r
            key = torch.arange(pos + 1)
            if window > 0:
                key = key[(key > pos - window) | (key < keep_first)]
            key = key[key // ps < bt.shape[1]]
            pages = bt[seq][key // ps].long()
            key, pages = key[pages >= 0], pages[pages >= 0]
            for h in range(n_heads):
                g = h // group
                k, v = kf[pages, g, key % ps], vf[pages, g, :, key % ps]
                qv = x[row0 + r, h * dh:(h + 1) * dh]
                s = (k @ qv) * scale
                if softcap > 0:
                    s = softcap * torch.tanh(s / softcap)
                if key.numel() == 0:
                    out[row0 + r, h] = 0
                    continue
                e = torch.exp(s - s.max())
                total = e.sum() + (torch.exp(at[h] - s.max()) if at is not None else 0)
                out[row0 + r, h] = (e @ v) / total
                mass[row0 + r, h] = (e @ v.abs()) / total
                most[row0 + r, h] = (k.abs() @ qv.abs()).max() * scale
    return out.view(T, -1), mass.view(T, -1), most


def attention8(q, out, k_pool, v_pool, k_scale, v_scale, block_tables, tiles, n_heads, scale, window=0, tiles_wide=None,
               single_rows=False, max_context=0, sink=False, keep_first=0, softcap=0.0):
    got, _, _ = attention_exact(q, k_pool, v_pool, k_scale, v_scale, block_tables, tiles, n_heads, scale, window, sink, keep_first, softcap)
    for seq, row0, nrows, _ in zip(*tiles.cpu().tolist()):
        if seq >= 0:
            out[row0:row0 + nrows] = got[row0:row0 + nrows].to(out)
    return out


@contextlib.contextmanager
def emulated():
    """`emulation.emulated_kernels` with the cache in 8 bits as well."""
    from denno_beta_amd.kernels import ops
    from emulation import emulated_kernels
    names = ("kv_append8", "attention8")
    saved = {n: getattr(ops, n) for n in names}
    try:
        for n in names:
            setattr(ops, n, globals()[n])
        with emulated_kernels():
            yield
    finally:
        for n, f in saved.items():
            setattr(ops, n, f)
