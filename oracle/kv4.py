"""CPU oracle of the paged 4-bit key/value cache — TEST INFRASTRUCTURE, as oracle.py.

Restates, from their definitions in include/cek.h, the page plan (plain
Python), the quantiser (IEEE fp32 steps, bit for bit), the decoding and the
attention (float64).  Parity is pinned to these definitions only.
"""
from __future__ import annotations

import math

import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _e4m3_table() -> np.ndarray:
    t = np.empty(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        t[b] = (math.nan if (b & 127) == 127 else v) * (-1 if b & 128 else 1)
    return t


E4M3 = _e4m3_table()


def nearest_even(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the grid number nearest to x >= 0 (ties to the even index; beyond the last: the last)."""
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    lo = hi - 1
    x = np.minimum(x.astype(np.float64), grid[-1])
    dl, dh = x - grid[lo], grid[hi] - x  # exact: few bits apart
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def quantize(x: torch.Tensor, g: torch.Tensor):
    """x [T, H, D] (16-bit), g [H] fp32 -> (packed codes uint8 [T, H, D/2], scale bytes uint8 [T, H, D/16])."""
    v = x.float().numpy().reshape(x.shape[0], x.shape[1], x.shape[2] // 16, 16)
    gg = g.float().numpy()[None, :, None]
    with np.errstate(all="ignore"):
        a = np.abs(v).max(-1)  # NaN stays NaN
        ratio = (a / (np.float32(6.0) * gg)).astype(np.float32)
        byte = np.where(np.isnan(ratio), 127, nearest_even(np.nan_to_num(ratio, nan=0.0, posinf=448.0), E4M3[:127]))
        unit = (E4M3[byte].astype(np.float32) * gg).astype(np.float32)[..., None]
        y = np.where(unit == 0, np.float32(0), v / unit).astype(np.float32)
        code = nearest_even(np.nan_to_num(np.abs(y), nan=6.0, posinf=6.0), E2M1)
        code = code | np.where(np.signbit(y) & ~np.isnan(y), 8, 0)
    code = code.reshape(x.shape).astype(np.uint8)
    return (torch.from_numpy(code[..., 0::2] | (code[..., 1::2] << 4)), torch.from_numpy(byte.astype(np.uint8)))


def offsets(page_size: int, d: int):
    """Byte offsets of K codes, K scales, V codes, V scales in a block, and its size."""
    code, scale = page_size * d // 2, page_size * d // 16
    return 0, code, code + scale, 2 * code + scale, 2 * (code + scale)


def append(cache: torch.Tensor, page_size: int, key, value, scales, slots) -> torch.Tensor:
    """The cache [pages, H, bytes] (CPU) after the append."""
    cache = cache.clone()
    d = key.shape[2]
    off = offsets(page_size, d)
    for part, x in ((0, key), (1, value)):
        code, scale = quantize(x, scales[part])
        for t, slot in enumerate(slots.tolist()):
            if not 0 <= slot < cache.shape[0] * page_size:
                continue
            p, r = divmod(slot, page_size)
            c0, s0 = off[2 * part] + r * d // 2, off[2 * part + 1] + r * d // 16
            cache[p, :, c0:c0 + d // 2] = code[t]
            cache[p, :, s0:s0 + d // 16] = scale[t]
    return cache


def decode(cache: torch.Tensor, page_size: int, d: int, slots, part: int, scales) -> np.ndarray:
    """float64 [len(slots), H, D] of keys (part 0) or values (part 1)."""
    off = offsets(page_size, d)
    slots = np.asarray(slots, dtype=np.int64)
    p, r = slots // page_size, slots % page_size
    c = cache.numpy()
    n, h = c.shape[:2]
    code = c[:, :, off[2 * part]:off[2 * part] + page_size * d // 2].reshape(n, h, page_size, d // 2)
    scale = c[:, :, off[2 * part + 1]:off[2 * part + 1] + page_size * d // 16].reshape(n, h, page_size, d // 16)
    code, scale = code[p, :, r], scale[p, :, r]
    nib = np.stack((code & 15, code >> 4), -1).reshape(len(slots), h, d)
    val = np.where(nib & 8, -1.0, 1.0) * E2M1[nib & 7]
    return val * np.repeat(E4M3[scale], 16, axis=-1) * scales[part].double().numpy()[None, :, None]


def attention(q, cache, page_size, scales, table, query_start, seq_lens, softmax_scale, window=0):
    """float64 (out [T, Hq, D], bound [T, Hq]): the result, and the largest |value| that each row and head sees."""
    T, hq, d = q.shape
    hkv = cache.shape[1]
    out, vmax = np.zeros((T, hq, d)), np.zeros((T, hq))
    x = q.double().numpy()
    for i, n_seq in enumerate(seq_lens.tolist()):
        a, b = query_start[i].item(), query_start[i + 1].item()
        n_seq = max(n_seq, 0)
        if a == b or n_seq == 0:
            continue
        keys = np.arange(n_seq)
        slots = table[i].numpy().astype(np.int64)[keys // page_size] * page_size + keys % page_size
        k, v = (decode(cache, page_size, d, slots, part, scales) for part in (0, 1))
        for r in range(a, b):
            pos = n_seq - (b - a) + (r - a)
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            for h in range(hq):
                kk, vv = k[lo:pos + 1, h * hkv // hq], v[lo:pos + 1, h * hkv // hq]
                with np.errstate(all="ignore"):
                    s = kk @ x[r, h] * softmax_scale
                    top = s.max()
                    p = np.exp(s - (0.0 if top == -np.inf else top))
                    out[r, h] = p @ vv / p.sum() if p.sum() != 0 else 0.0
                vmax[r, h] = np.abs(vv).max()
    return torch.from_numpy(out), torch.from_numpy(vmax)


def plan(query_lens, context_lens, table, free_pages, free_count, page_size, tokens):
    """Plain lists in and out: (table, query_start, seq_lens, free count, positions, slots)."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    start, seq, pos, slots = [0], [], [], []
    asked = taken = 0
    for i, (n, c) in enumerate(zip(query_lens, context_lens)):
        n = max(n, 0)
        start.append(start[-1] + n)
        here = ~c if c < 0 else c
        have, total = -(-here // page_size), -(-(here + n) // page_size)
        need = total - have if c >= 0 and total <= width else 0
        ok = c >= 0 and total <= width and (need == 0 or asked + need <= free_count)
        if ok:
            for j in range(need):
                table[i][have + j] = free_pages[free_count - 1 - asked - j]
            taken = max(taken, asked + need if need else 0)
        asked += need
        seq.append(c + n if ok else ~here)
        for r in range(n):
            pos.append(here + r)
            slots.append(table[i][(here + r) // page_size] * page_size + (here + r) % page_size if ok else -1)
    pos, slots = (pos + [0] * tokens)[:tokens], (slots + [-1] * tokens)[:tokens]
    return table, start, seq, free_count - taken, pos, slots
