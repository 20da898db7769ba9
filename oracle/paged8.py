"""The 8-bit paged cache and windowed attention over paged caches in float64.

quantise_rows        codes (float8_e4m3fn) and scale exponents of rows, by search
                     over all 254 scales and all 127 magnitudes of e4m3
append_reference     kv_cache_append on copies of the caches
read_reference       kv_cache_read
window_reference     attention with window and sinks, with what an error bound needs
"""
import math

import torch

E4M3 = torch.float8_e4m3fn


def e4m3_magnitudes():
    """The 127 magnitudes of e4m3 in ascending order: code i's value at index i (7 is 7/512; 8 is 2^-6)."""
    return torch.tensor([(i & 7) * 2.0 ** -9 if i < 8 else (8 + (i & 7)) * 2.0 ** ((i >> 3) - 10) for i in range(127)],
                        dtype=torch.float64)


def quantise_rows(x):
    """x [..., D] -> codes uint8 (bits of float8_e4m3fn) [..., D], exponents uint8 [...]."""
    y = x.double()
    fin = torch.isfinite(y)
    amax = torch.where(fin, y.abs(), 0.0).amax(-1)
    scales = torch.tensor([2.0 ** (e - 127) for e in range(1, 255)], dtype=torch.float64)
    e = (amax[..., None] > 448 * scales).sum(-1) + 1  # the first scale that holds amax
    s = scales[e - 1][..., None]
    z = torch.where(fin, y / s, 0.0)
    held = 256 * s > torch.finfo(x.dtype).max
    z = torch.where(held, z.clamp(-240, 240), z)
    mags = e4m3_magnitudes()
    up = torch.searchsorted(mags, z.abs().contiguous()).clamp(max=126)  # the first magnitude >= |z|
    down = (up - 1).clamp(min=0)
    to_up, to_down = mags[up] - z.abs(), z.abs() - mags[down]
    code = torch.where((to_up < to_down) | ((to_up == to_down) & (up % 2 == 0)), up, down)
    code = torch.where(torch.signbit(x), code + 128, code)
    return torch.where(fin, code, 127).to(torch.uint8), e.to(torch.uint8)


def values(codes, exponents):
    """float64 values of codes (uint8 [..., D]) under exponents [...]."""
    mags = torch.cat([e4m3_magnitudes(), torch.tensor([math.nan], dtype=torch.float64)])
    v = mags[(codes & 127).long()] * torch.where(codes >= 128, -1.0, 1.0)
    return v * torch.pow(torch.tensor(2.0, dtype=torch.float64), exponents.double() - 127)[..., None]


def _place(table, num_blocks, bs, b, pos):
    i = pos // bs
    if pos < 0 or i >= table.shape[1] or not 0 <= int(table[b, i]) < num_blocks:
        return None
    return int(table[b, i]), pos % bs


def append_reference(k, v, k_codes, v_codes, scales, table, seq_lens, cu=None):
    """Codes as uint8; returns new (k_codes, v_codes, scales)."""
    k_codes, v_codes, scales = k_codes.clone(), v_codes.clone(), scales.clone()
    n, bs = k_codes.shape[:2]
    kq, ke = quantise_rows(k)
    vq, ve = quantise_rows(v)
    for b in range(table.shape[0]):
        lo, hi = (b, b + 1) if cu is None else (int(cu[b]), int(cu[b + 1]))
        for t in range(lo, hi):
            at = _place(table, n, bs, b, int(seq_lens[b]) - (hi - t))
            if at is None:
                continue
            blk, slot = at
            k_codes[blk, slot], v_codes[blk, slot] = kq[t], vq[t]
            scales[blk, :, slot, 0], scales[blk, :, slot, 1] = ke[t], ve[t]
    return k_codes, v_codes, scales


def cache_values(k_codes, v_codes, scales):
    """float64 K and V of 8-bit caches [num_blocks, block_size, heads_kv, head_dim]."""
    return (values(k_codes, scales[..., 0].transpose(1, 2)), values(v_codes, scales[..., 1].transpose(1, 2)))


def rows_of(cache, table, b, n):
    """The first n rows of sequence b, zeros where no block holds them."""
    num_blocks, bs = cache.shape[:2]
    rows = torch.zeros(n, *cache.shape[2:], dtype=torch.float64)
    for i in range(-(-n // bs)):
        at = _place(table, num_blocks, bs, b, i * bs)
        if at is not None:
            m = min(bs, n - i * bs)
            rows[i * bs:i * bs + m] = cache[at[0], :m].double()
    return rows


def read_reference(k_codes, v_codes, scales, table, cu, total):
    out = [torch.zeros(total, *k_codes.shape[2:], dtype=torch.float64) for _ in range(2)]
    for rows, cache in zip(out, cache_values(k_codes, v_codes, scales)):
        for b in range(table.shape[0]):
            lo, hi = int(cu[b]), min(int(cu[b + 1]), total)
            if hi > lo:
                rows[lo:hi] = rows_of(cache, table, b, hi - lo)
    return out


def window_reference(q, k_cache, v_cache, table, cu, seq_lens, window=None, sinks=0, causal=True, sm_scale=None):
    """q [T, Hq, D]; caches of any type (8-bit ones as cache_values gives them). Returns o [T, Hq, D], lse [T, Hq], and for
    error bounds the weighted magnitudes a = sum w |v| [T, Hq, D] and the largest sum |q k| |scale| of a row [T, Hq]; rows of no
    sequence are zeros."""
    T, Hq, D = q.shape
    group = Hq // k_cache.shape[2]
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    most = table.shape[1] * k_cache.shape[1]
    o, a = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    lse, big = torch.full((T, Hq), -math.inf, dtype=torch.float64), torch.zeros(T, Hq, dtype=torch.float64)
    for b in range(table.shape[0]):
        lo, hi = (b, b + 1) if cu is None else (int(cu[b]), int(cu[b + 1]))
        nk = min(max(int(seq_lens[b]), 0), most)
        if hi <= lo or nk == 0:
            continue
        # Keys that no query sees are not read: their rows may hold anything.
        j = torch.arange(nk)
        p = torch.arange(nk - (hi - lo), nk)[:, None] if causal else torch.full((hi - lo, 1), nk - 1)
        seen = j <= p
        if window is not None:
            seen &= (j > p - window) | (j < sinks)
        any_seen = seen.any(0)
        kb, vb = (rows_of(c, table, b, nk).repeat_interleave(group, 1).transpose(0, 1) for c in (k_cache, v_cache))
        kb, vb = (torch.where(any_seen[None, :, None], x, 0.0) for x in (kb, vb))
        qb = q[lo:hi].double().transpose(0, 1)
        s = torch.where(seen, qb @ kb.transpose(1, 2) * scale, -math.inf)
        w = torch.softmax(s, -1)
        w = torch.where(seen.any(-1, keepdim=True), w, 0.0)
        o[lo:hi] = (w @ vb).transpose(0, 1)
        a[lo:hi] = (w @ vb.abs()).transpose(0, 1)
        lse[lo:hi] = s.logsumexp(-1).T
        big[lo:hi] = torch.where(seen, qb.abs() @ kb.abs().transpose(1, 2) * abs(scale), 0.0).amax(-1).T
    return o, lse, a, big
