"""Paged attention over 8-bit caches and under a sliding window with sinks, against the float64 oracle.

Bounds are elementwise, from arithmetic: with u half a step of q's type, the weights that multiply V are p rounded to that type
and normalised by the sum of the rounded ones, so o is off by at most 2u a (a = sum w |v|), and rounding o adds u |o|. A score is
a sum of D products that are exact in fp32: each addition is off by half a step of a partial sum of at most big = sum |q k|
|scale|, and the scalings, the exponent and the split of a row over waves and workgroups add a few steps: e = (D + 16) 2^-24 big
+ 2^-19, which moves weights by a factor of exp(+-2e). Sums over n keys add n 2^-24 a. The lse is off by e, n 2^-24 and two steps
of itself. fp16 operands of V round below 2^-14 to 2^-25. Second orders are covered by a factor of 1.05.
"""
import math

import pytest
import torch

from lightserve_amd import _lib
from lightserve_amd.kernels.paged_attention import paged_attention_decode, paged_prefill
from lightserve_amd.kernels.quantized_kv_cache import kv_cache_append, quantized_kv_cache
from oracle import paged8
from tests.paged8_cases import cache8, offsets, tables

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _cache(kind, dtype, pool, bs, hkv, d, seed):
    """Device caches and scales, and float64 values for the oracle."""
    if kind == "e4m3":
        kc, vc, sc = cache8(pool, bs, hkv, d, seed)
        return (kc.cuda().view(E4M3), vc.cuda().view(E4M3), sc.cuda()), paged8.cache_values(kc, vc, sc)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(pool, bs, hkv, d, generator=g).to(dtype) for _ in range(2))
    return (k.cuda(), v.cuda(), None), (k.double(), v.double())


def _q(t, hq, d, dtype, seed):
    return torch.randn(t, hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _assert_close(got, lse, ref, n, what):
    o, want_lse, a, big = ref
    got, lse = got.cpu(), lse.cpu().double()
    u, d = torch.finfo(got.dtype).eps / 2, got.shape[-1]
    e = (d + 16) * 2.0 ** -24 * big + 2.0 ** -19
    tol = 1.05 * ((2 * u + 2 * e[..., None] + n * 2.0 ** -24) * a + u * o.abs()) + 2.0 ** -24
    off = (got.double() - o).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert worst <= 1, f"{what}: {worst:.2f} of the bound at {(off / tol).argmax().item()}"
    none = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, none), f"{what}: rows that see nothing"
    lse_tol = e + n * 2.0 ** -24 + want_lse.abs() * 2.0 ** -22
    lse_off = ((lse - want_lse).abs() / lse_tol)[~none]
    assert lse_off.numel() == 0 or lse_off.max() <= 1, f"{what}: lse {lse_off.max():.2f} of the bound"
    print(f"[bound] {what}: o {worst:.2f}, lse {lse_off.max().item() if lse_off.numel() else 0:.2f}", flush=True)


def _decode(kind, dtype, lens, hq, hkv, d, bs, seed, window=None, sinks=0, max_seq_len=None, sm_scale=None, what=""):
    table, pool = tables(lens, bs, seed)
    cache, vals = _cache(kind, dtype, pool, bs, hkv, d, seed + 1)
    q = _q(len(lens), hq, d, dtype, seed + 2)
    o, lse = paged_attention_decode(q.cuda(), *cache[:2], table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                    max_seq_len=max_seq_len, sm_scale=sm_scale, return_lse=True, kv_scales=cache[2],
                                    window=window, sinks=sinks)
    torch.cuda.synchronize()
    ref = paged8.window_reference(q, *vals, table, None, lens, window, sinks, sm_scale=sm_scale)
    _assert_close(o, lse, ref, max(lens + [1]), what)


def _chunk(kind, dtype, new, had, hq, hkv, d, bs, seed, window=None, sinks=0, causal=True, sm_scale=None, what=""):
    lens = [a + b for a, b in zip(new, had)]
    table, pool = tables(lens, bs, seed)
    cache, vals = _cache(kind, dtype, pool, bs, hkv, d, seed + 1)
    q = _q(sum(new), hq, d, dtype, seed + 2)
    o, lse = paged_prefill(q.cuda(), *cache[:2], table.cuda(), offsets(new).cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), causal=causal, sm_scale=sm_scale, return_lse=True,
                           kv_scales=cache[2], window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert lse.shape == (hq, sum(new))
    ref = paged8.window_reference(q, *vals, table, offsets(new), lens, window, sinks, causal, sm_scale)
    _assert_close(o, lse.t(), ref, max(lens + [1]), what)


KINDS = [("e4m3", torch.bfloat16), ("e4m3", torch.float16), ("16 bit", torch.bfloat16), ("16 bit", torch.float16)]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (32, 8, 128), (14, 2, 64), (6, 2, 80), (20, 1, 128), (3, 3, 16)])
def test_decode(gpu, kind, dtype, hq, hkv, d):
    """Group sizes 1 to 20 (more than a row tile), head dims with and without padding; lengths around pieces and tiles."""
    print(f"case decode {kind} {dtype} hq={hq} hkv={hkv} d={d}", flush=True)
    lens = [1, 15, 16, 17, 31, 32, 33, 0, 100, 333]
    for window, sinks in ((None, 0), (20, 3)):
        if window is not None or kind == "e4m3":
            _decode(kind, dtype, lens, hq, hkv, d, 16, hq + d, window, sinks, what=f"decode w={window}")


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 32, 33, 100, 5000])
@pytest.mark.parametrize("sinks", [0, 1, 16, 33, 5000])
def test_decode_windows(gpu, window, sinks):
    """Windows and sinks that end inside pieces and tiles, meet, overlap, and pass the sequence."""
    print(f"case decode window={window} sinks={sinks}", flush=True)
    _decode("e4m3", torch.bfloat16, [1, 16, 40, 64, 65, 130, 500], 8, 2, 64, 16, 7, window, sinks, what="window")


@pytest.mark.parametrize("bs", [16, 32, 64, 256])
def test_decode_block_sizes(gpu, bs):
    print(f"case decode bs={bs}", flush=True)
    _decode("e4m3", torch.bfloat16, [3, 300, 77], 8, 2, 96, bs, bs, 50, 2, sm_scale=0.3, what=f"bs={bs}")
    _decode("16 bit", torch.float16, [3, 300, 77], 8, 2, 72, bs, bs, 50, 2, sm_scale=-0.2, what=f"bs={bs}")


@pytest.mark.parametrize("lens", [[9000], [4096, 1, 3000], [12000, 700, 0, 5]])
def test_decode_shared_out(gpu, lens):
    """Sequences that lie in several runs, and runs that hold several sequences."""
    print(f"case decode runs lens={lens}", flush=True)
    _decode("e4m3", torch.bfloat16, lens, 8, 1, 128, 16, 11, what="runs")
    _decode("e4m3", torch.float16, lens, 4, 2, 64, 16, 12, max_seq_len=16384, what="runs, wide limit")
    _decode("16 bit", torch.bfloat16, lens, 8, 1, 128, 16, 13, 3000, 4, what="runs, window")


@pytest.mark.parametrize("batch", [63, 64, 65, 200])
def test_decode_many_sequences(gpu, batch):
    print(f"case decode batch={batch}", flush=True)
    lens = [(37 * b * b) % 300 for b in range(batch)]
    lens[batch // 2], lens[-1] = 2500, 1200
    _decode("e4m3", torch.bfloat16, lens, 8, 2, 64, 16, batch, what="batch")
    _decode("16 bit", torch.float16, lens, 8, 2, 64, 16, batch, 64, 1, what="batch, window")


def test_decode_limit(gpu):
    """seq_lens past max_seq_len are clamped."""
    print("case decode limit", flush=True)
    lens, limit = [40, 64, 90], 64
    table, pool = tables(lens, 16, 14)
    cache, vals = _cache("e4m3", torch.bfloat16, pool, 16, 2, 64, 15)
    q = _q(3, 4, 64, torch.bfloat16, 16)
    sl = torch.tensor(lens, dtype=torch.int32)
    o, lse = paged_attention_decode(q.cuda(), *cache[:2], table.cuda(), sl.cuda(), max_seq_len=limit, return_lse=True,
                                    kv_scales=cache[2])
    _assert_close(o, lse, paged8.window_reference(q, *vals, table, None, sl.clamp(max=limit)), 64, "limit")


@pytest.mark.parametrize("kind", ["e4m3", "16 bit"])
@pytest.mark.parametrize("n", [1, 3])
def test_what_no_query_sees_is_not_read(gpu, kind, n):
    """NaN codes and scales, infinities and wild table entries wherever no query of the call looks: left of the window, behind
    the sequence in its last block, in blocks of nobody."""
    print(f"case unseen rows {kind} n={n}", flush=True)
    lens, bs, window, sinks, dtype = [200, 37, 90], 16, 40, 5, torch.bfloat16
    table, pool = tables(lens, bs, 17)
    q = _q(3 * n, 4, 64, dtype, 18)
    clean = cache8(pool, bs, 2, 64, 19)
    if kind == "e4m3":
        kc, vc, sc = (t.clone() for t in clean)
        vals = paged8.cache_values(*clean)
        bad = 127
    else:
        kc, vc = (t.to(dtype) for t in paged8.cache_values(*clean))
        vals, sc, bad = (kc.double(), vc.double()), None, math.nan
        kc, vc = kc.clone(), vc.clone()
    seen = torch.zeros(pool, bs, dtype=torch.bool)
    dirty = table.clone()
    for b, length in enumerate(lens):
        used = set()
        for p in range(length):
            if p < sinks or p > length - n - window:
                seen[table[b, p // bs], p % bs] = True
                used.add(p // bs)
        for i in range(table.shape[1]):
            if i not in used:
                dirty[b, i] = [-5, 1 << 30, pool, int(table[0, 0])][i % 4]
    kc[~seen], vc[~seen] = bad, bad
    if sc is not None:
        sc.transpose(1, 2)[~seen] = 255
    elif n == 1:
        vc[~seen] = math.inf
    cache = (kc.cuda().view(E4M3), vc.cuda().view(E4M3)) if sc is not None else (kc.cuda(), vc.cuda())
    how = dict(return_lse=True, kv_scales=sc.cuda() if sc is not None else None, window=window, sinks=sinks)
    sl = torch.tensor(lens, dtype=torch.int32).cuda()
    cu = offsets([n] * 3)
    ref = paged8.window_reference(q, *vals, table, cu, lens, window, sinks)
    o, lse = paged_prefill(q.cuda(), *cache, dirty.cuda(), cu.cuda(), sl, **how)
    _assert_close(o, lse.t(), ref, 200, "chunk")
    if n == 1:
        o, lse = paged_attention_decode(q.cuda(), *cache, dirty.cuda(), sl, **how)
        _assert_close(o, lse, ref, 200, "decode")


def test_blocks_outside_the_cache_read_as_zeros(gpu):
    print("case blocks outside", flush=True)
    lens = [100, 20]
    table, pool = tables(lens, 16, 20)
    table[0, 2], table[1, 0] = pool, -1
    cache, vals = _cache("e4m3", torch.bfloat16, pool, 16, 2, 64, 21)
    q = _q(2, 4, 64, torch.bfloat16, 22)
    o, lse = paged_attention_decode(q.cuda(), *cache[:2], table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                    return_lse=True, kv_scales=cache[2])
    _assert_close(o, lse, paged8.window_reference(q, *vals, table, None, lens), 100, "zeros")


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (16, 4, 128), (14, 2, 64), (6, 2, 80), (16, 1, 112)])
def test_chunks(gpu, kind, dtype, hq, hkv, d):
    """Ragged and empty chunks, one of a single token, one without a prefix."""
    print(f"case chunks {kind} {dtype} hq={hq} hkv={hkv} d={d}", flush=True)
    new, had = [128, 17, 1, 0, 64, 3, 150], [172, 0, 999, 64, 65, 29, 0]
    for window, sinks in ((None, 0), (70, 5)):
        if window is not None or kind == "e4m3":
            _chunk(kind, dtype, new, had, hq, hkv, d, 16, hq + d, window, sinks, what=f"chunks w={window}")


@pytest.mark.parametrize("window", [1, 31, 64, 65, 127, 1000])
@pytest.mark.parametrize("sinks", [0, 4, 70, 1000])
def test_chunk_windows(gpu, window, sinks):
    print(f"case chunk window={window} sinks={sinks}", flush=True)
    _chunk("e4m3", torch.bfloat16, [300, 40, 7], [0, 300, 130], 4, 2, 64, 32, 23, window, sinks, what="window")
    _chunk("16 bit", torch.float16, [129, 257], [600, 0], 4, 4, 128, 16, 24, window, sinks, sm_scale=-0.1, what="window 16")


@pytest.mark.parametrize("new", [2, 4, 5, 16, 33])
def test_short_chunks(gpu, new):
    """Chunks of a few tokens, as a step that checks drafted ones has them."""
    print(f"case short chunks n={new}", flush=True)
    _chunk("e4m3", torch.bfloat16, [new, 1, new], [1000, 33, 5000], 8, 2, 128, 16, 25, what="short")
    _chunk("e4m3", torch.float16, [new, new - 1], [70, 2000], 7, 1, 64, 64, 26, 300, 10, what="short, window")


def test_chunks_without_a_mask(gpu):
    print("case chunks not causal", flush=True)
    _chunk("e4m3", torch.bfloat16, [100, 5], [30, 200], 4, 2, 64, 16, 27, causal=False, what="not causal")


def test_queries_before_the_first_key(gpu):
    """Chunks longer than what is cached: the first queries see nothing."""
    print("case queries before the first key", flush=True)
    new, lens = [40, 9, 5], [10, 9, 0]
    table, pool = tables([40, 9, 5], 16, 28)
    cache, vals = _cache("e4m3", torch.bfloat16, pool, 16, 2, 64, 29)
    q = _q(54, 4, 64, torch.bfloat16, 30)
    sl = torch.tensor(lens, dtype=torch.int32)
    for window in (None, 4):
        o, lse = paged_prefill(q.cuda(), *cache[:2], table.cuda(), offsets(new).cuda(), sl.cuda(), return_lse=True,
                               kv_scales=cache[2], window=window)
        _assert_close(o, lse.t(), paged8.window_reference(q, *vals, table, offsets(new), lens, window), 54, f"w={window}")


def test_rows_behind_the_last_sequence(gpu):
    """A padded batch: the rows of its sequences, whatever lies behind; offsets past q's rows reach nothing outside."""
    print("case padded batch", flush=True)
    new, had = [30, 50], [10, 100]
    lens = [a + b for a, b in zip(new, had)]
    table, pool = tables(lens, 16, 31)
    cache, vals = _cache("e4m3", torch.bfloat16, pool, 16, 2, 64, 32)
    q = _q(100, 4, 64, torch.bfloat16, 33)
    q[80:] = math.nan
    ref = paged8.window_reference(q[:80], *vals, table, offsets(new), lens, 64, 2)
    o, lse = paged_prefill(q.cuda(), *cache[:2], table.cuda(), offsets(new).cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True, kv_scales=cache[2], window=64, sinks=2)
    _assert_close(o[:80], lse.t()[:80], tuple(t[:80] for t in ref), 150, "padded")


def test_large_scores(gpu):
    """Rows whose scores differ by hundreds: the running offset is raised again and again, and falls short of none."""
    print("case large scores", flush=True)
    lens = [700, 130]
    table, pool = tables(lens, 16, 34)
    kc, vc, sc = cache8(pool, 16, 1, 64, 35)
    g = torch.Generator().manual_seed(36)
    sc[..., 0] = torch.randint(112, 126, sc[..., 0].shape, generator=g, dtype=torch.uint8)
    vals = paged8.cache_values(kc, vc, sc)
    q = _q(2, 4, 64, torch.float16, 37)
    o, lse = paged_attention_decode(q.cuda(), kc.cuda().view(E4M3), vc.cuda().view(E4M3), table.cuda(),
                                    torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True, kv_scales=sc.cuda())
    _assert_close(o, lse, paged8.window_reference(q, *vals, table, None, lens), 700, "large decode")
    q = _q(60, 4, 64, torch.bfloat16, 38)
    o, lse = paged_prefill(q.cuda(), kc.cuda().view(E4M3), vc.cuda().view(E4M3), table.cuda(), offsets([40, 20]).cuda(),
                           torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True, kv_scales=sc.cuda())
    _assert_close(o, lse.t(), paged8.window_reference(q, *vals, table, offsets([40, 20]), lens), 700, "large chunk")


def test_nan_of_a_key_reaches_the_rows_that_see_it(gpu):
    print("case NaN keys", flush=True)
    lens = [64, 64]
    table, pool = tables(lens, 16, 39)
    kc, vc, sc = cache8(pool, 16, 1, 64, 40)
    vc[table[0, 1], 3, 0, 5] = 127
    kc[table[1, 2], 0, 0, 9] = 255
    q = _q(2, 4, 64, torch.bfloat16, 41)
    o = paged_attention_decode(q.cuda(), kc.cuda().view(E4M3), vc.cuda().view(E4M3), table.cuda(),
                               torch.tensor(lens, dtype=torch.int32).cuda(), kv_scales=sc.cuda()).cpu()
    assert torch.isnan(o[0, :, 5]).all() and torch.isnan(o[1]).all()
    assert torch.isfinite(o[0, :, :5]).all() and torch.isfinite(o[0, :, 6:]).all()


@pytest.mark.parametrize("kind,bad", [("e4m3", math.nan), ("16 bit", math.nan), ("16 bit", math.inf), ("16 bit", -math.inf)])
@pytest.mark.parametrize("n,heads,d", [(3, 4, 64), (6, 4, 128), (8, 8, 80), (40, 4, 64), (100, 2, 128), (200, 16, 64), (600, 32, 72), (2048, 32, 64)])
def test_values_not_finite_reach_the_rows_that_see_them_alone(gpu, kind, bad, n, heads, d):
    """V of a key that a chunk's later (or, at the window's start, earlier) queries do not see, in both kernels."""
    print(f"case not finite {kind} {bad} n={n} heads={heads} d={d}", flush=True)
    if kind == "e4m3" and d % 16 != 0:
        d = 80
    length, bs, dtype = n + 150, 16, torch.float16 if n == 40 else torch.bfloat16
    table, pool = tables([length], bs, 54)
    codes = cache8(pool, bs, 2, d, 55)
    clean = paged8.cache_values(*codes)
    q = _q(n, heads, d, dtype, 56)
    at = [length - 2, length - n + 1, length - n - 40, 1, length - n - 58 + n // 2]
    p = torch.arange(length - n, length)
    for window, sinks in ((60, 2), (None, 0)):
        if window is None and kind != "e4m3":
            continue
        kc, vc, sc = (t.clone() for t in codes)
        if kind != "e4m3":
            kc, vc, sc = clean[0].to(dtype), clean[1].to(dtype), None
        for i, j in enumerate(at):
            vc[table[0, j // bs], j % bs, :, 7 * i] = 127 if kind == "e4m3" else bad
        dev = [t.cuda() if t is not None else None for t in (kc, vc, sc)]
        if kind == "e4m3":
            dev[:2] = [t.view(E4M3) for t in dev[:2]]
        o, lse = paged_prefill(q.cuda(), dev[0], dev[1], table.cuda(), offsets([n]).cuda(),
                               torch.tensor([length], dtype=torch.int32).cuda(), return_lse=True, kv_scales=dev[2],
                               window=window, sinks=sinks)
        alone = paged_prefill(q.cuda(), dev[0], dev[1], table.cuda(), offsets([n]).cuda(),
                              torch.tensor([length], dtype=torch.int32).cuda(), kv_scales=dev[2], window=window, sinks=sinks)
        assert torch.equal(torch.isfinite(alone), torch.isfinite(o)), "without the lse"
        o, ref = o.cpu(), paged8.window_reference(q, *clean, table, offsets([n]), [length], window, sinks)
        for i, j in enumerate(at):
            sees = (j <= p) & ((j > p - window) | (j < sinks) if window is not None else True)
            got = o[:, :, 7 * i]
            assert (torch.isnan(got[sees]).all() if math.isnan(bad) else (got[sees] == bad).all()), f"key {j}"
            assert torch.isfinite(got[~sees]).all(), f"key {j}"
            got[sees] = ref[0][:, :, 7 * i][sees].to(dtype)
        _assert_close(o, lse.t(), ref, length, f"the others w={window}")


# (kind, type, lengths from and to, sequences, heads, KV heads, head dim, queries, window, sinks): enough keys for every
# workgroup to have a long run, whose partial results a launch of their own merges; one, two and four KV heads a
# workgroup; one and two column blocks of rows; more sequences than lanes.
LONG = [("e4m3", torch.bfloat16, 0, 8000, 20, 32, 8, 128, 1, None, 0), ("e4m3", torch.float16, 1500, 3500, 70, 8, 2, 64, 1, None, 0),
        ("16 bit", torch.bfloat16, 15000, 25000, 6, 3, 3, 64, 1, 24000, 3), ("e4m3", torch.bfloat16, 2000, 3500, 70, 8, 4, 64, 1, 1500, 5),
        ("16 bit", torch.float16, 20000, 30000, 5, 64, 8, 64, 3, 29000, 0), ("e4m3", torch.bfloat16, 0, 60000, 2, 64, 16, 80, 2, None, 0),
        ("e4m3", torch.float16, 100, 20000, 9, 128, 16, 48, 4, 9000, 40)]


@pytest.mark.parametrize("case", range(len(LONG)))
def test_long_runs(gpu, case):
    kind, dtype, least, most, batch, hq, hkv, d, new, window, sinks = LONG[case]
    print(f"case long runs {LONG[case]}", flush=True)
    g = torch.Generator().manual_seed(60 + case)
    lens = torch.randint(least, most + 1, (batch,), generator=g).tolist()
    lens[0] = most
    if new == 1:
        _decode(kind, dtype, lens, hq, hkv, d, 16, 70 + case, window, sinks, what=f"long runs {case}")
    else:
        n = [min(new - b % 2, m) for b, m in enumerate(lens)]
        _chunk(kind, dtype, n, [m - k for m, k in zip(lens, n)], hq, hkv, d, 16, 70 + case, window, sinks, what=f"long runs {case}")


@pytest.mark.parametrize("window", [None, 100])
def test_chunks_of_many_sequences(gpu, window):
    """More sequences than a wave has lanes, some without queries, in the wide kernel."""
    print(f"case many chunks window={window}", flush=True)
    g = torch.Generator().manual_seed(63)
    new = [int(n) if b % 5 else 0 for b, n in enumerate(torch.randint(0, 90, (130,), generator=g))]
    had = torch.randint(0, 300, (130,), generator=g).tolist()
    _chunk("e4m3", torch.bfloat16, new, had, 8, 2, 64, 16, 64, window, 3 if window else 0, what=f"many chunks w={window}")


def test_window_past_every_position(gpu, monkeypatch):
    """The largest window that the C argument holds sees what a window of the sequence's length does."""
    print("case largest window", flush=True)
    lens = [90, 700]
    table, pool = tables(lens, 16, 68)
    cache, _ = _cache("e4m3", torch.bfloat16, pool, 16, 2, 64, 69)
    q = _q(120, 4, 64, torch.bfloat16, 70).cuda()
    launch, sizes = _lib.window, []

    def largest(args, stream):
        sizes.append(args.window)
        args.window = 2 ** 31 - 1
        launch(args, stream)

    def calls():
        sl = torch.tensor(lens, dtype=torch.int32).cuda()
        return [paged_prefill(q, *cache[:2], table.cuda(), offsets([n, 120 - n]).cuda(), sl, kv_scales=cache[2], window=800, sinks=0)
                for n in (2, 60)] + [paged_attention_decode(q[:2], *cache[:2], table.cuda(), sl, kv_scales=cache[2], window=800)]

    want = calls()
    monkeypatch.setattr(_lib, "window", largest)
    assert all(torch.equal(a, b) for a, b in zip(calls(), want)) and len(sizes) == 3


def test_graph_follows_the_lengths(gpu):
    """A captured step replayed after the lengths have changed: short runs, long ones, one sequence, none, and eager steps and
    calls on another stream between and beside the replays."""
    print("case graph lengths", flush=True)
    B, hq, hkv, d, bs, most = 24, 32, 8, 128, 16, 4096
    table, pool = tables([most] * B, bs, 65)
    cache, _ = _cache("e4m3", torch.bfloat16, pool, bs, hkv, d, 66)
    bt, q, sl = table.cuda(), _q(B, hq, d, torch.bfloat16, 67).cuda(), torch.full((B,), most, dtype=torch.int32).cuda()
    lens = [[most] * B, [33] * B, [most] + [0] * (B - 1), [0] * B, [most - 100 * b for b in range(B)], [1] * B]

    def step():
        return paged_attention_decode(q, *cache[:2], bt, sl, max_seq_len=most, return_lse=True, kv_scales=cache[2])

    want = []
    for n in lens:
        sl.copy_(torch.tensor(n, dtype=torch.int32))
        want.append(step())
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    sl2 = torch.tensor(lens[4], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    for turn in range(2):
        for i, n in enumerate(lens):
            sl.copy_(torch.tensor(n, dtype=torch.int32))
            with torch.cuda.stream(other):
                beside = paged_attention_decode(q, *cache[:2], bt, sl2, max_seq_len=most, return_lse=True, kv_scales=cache[2])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[i])), f"turn {turn}: lengths {i}"
            assert all(torch.equal(a, b) for a, b in zip(beside, want[4])), f"turn {turn}: beside lengths {i}"
            assert all(torch.equal(a, b) for a, b in zip(step(), want[i])), f"turn {turn}: eager, lengths {i}"
    for i, n in enumerate(lens[2:5]):
        o, lse = want[2 + i]
        none = torch.tensor(n) == 0
        assert (o.cpu()[none] == 0).all() and (lse.cpu()[none] == -math.inf).all()


def test_strided_inputs(gpu):
    """q inside a fused projection, caches of a wider allocation, a table with another column stride."""
    print("case strided", flush=True)
    lens = [77, 200]
    table, pool = tables(lens, 16, 42)
    (kc, vc, sc), vals = _cache("e4m3", torch.bfloat16, pool, 16, 2, 64, 43)
    both = torch.zeros(pool, 2, 16, 2, 64, dtype=torch.uint8, device="cuda")
    both[:, 0], both[:, 1] = kc.view(torch.uint8), vc.view(torch.uint8)
    wide = torch.full((2, table.shape[1] * 2), -3, dtype=torch.int32)
    wide[:, ::2] = table
    fused = _q(2, 9, 64, torch.bfloat16, 44)
    sl = torch.tensor([0] + lens, dtype=torch.int32).cuda()[1:]
    for q, dev in ((fused[:, 1:5], fused.cuda()[:, 1:5]), (fused.view(2, -1)[:, 3:259].reshape(2, 4, 64),
                                                           fused.cuda().view(2, -1)[:, 3:259].unflatten(1, (4, 64)))):
        o, lse = paged_attention_decode(dev, both[:, 0].view(E4M3), both[:, 1].view(E4M3), wide.cuda()[:, ::2], sl,
                                        return_lse=True, kv_scales=sc, window=90, sinks=1)
        _assert_close(o, lse, paged8.window_reference(q, *vals, table, None, lens, 90, 1), 200, "strided")


def test_same_results_every_time_and_in_graphs(gpu):
    """Bit for bit the same again, on another stream, and in two captured graphs replayed in turn beside eager calls."""
    print("case graphs", flush=True)
    lens = [3000, 40, 900]
    table, pool = tables(lens, 16, 45)
    cache, _ = _cache("e4m3", torch.bfloat16, pool, 16, 2, 128, 46)
    bt, sl = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    q, qc = _q(3, 8, 128, torch.bfloat16, 47).cuda(), _q(150, 8, 128, torch.bfloat16, 48).cuda()
    cu = offsets([100, 10, 40]).cuda()

    def decode():
        return paged_attention_decode(q, *cache[:2], bt, sl, max_seq_len=4096, return_lse=True, kv_scales=cache[2])

    def chunk():
        return paged_prefill(qc, *cache[:2], bt, cu, sl, max_seqlen_q=100, return_lse=True, kv_scales=cache[2], window=500, sinks=4)

    want = [f() for f in (decode, chunk)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        again = [f() for f in (decode, chunk)]
    stream.synchronize()
    graphs = []
    for f in (decode, chunk):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    for i in range(4):
        for g, out in graphs:
            for t in out:
                t.fill_(-1)
            g.replay()
        if i % 2:
            torch.cuda.synchronize()
            decode()
        torch.cuda.synchronize()
        for (_, out), w, s in zip(graphs, want, again):
            assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(out, w, s)), f"replay {i}"


def test_append_then_attend(gpu):
    """Together as they are used: prompts appended chunk by chunk under a window, then decode steps, against the oracle on the
    rows that the cache stands for."""
    print("case append then attend", flush=True)
    hq, hkv, d, bs, window, sinks = 8, 2, 64, 16, 48, 4
    total = [150, 61]
    table, pool = tables([n + 5 for n in total], bs, 49)
    bt = table.cuda()
    kc, vc, sc = quantized_kv_cache(pool, bs, hkv, d)
    g = torch.Generator().manual_seed(50)
    k, v, q = (torch.randn(2, 155, h, d, generator=g).to(torch.bfloat16) for h in (hkv, hkv, hq))
    done = [0, 0]
    for step in ([70, 61], [80, 0], [1, 1], [1, 1], [1, 1]):
        new = [slice(a, a + n) for a, n in zip(done, step)]
        kk, vv, qq = (torch.cat([x[b, s] for b, s in enumerate(new)]).cuda() for x in (k, v, q))
        done = [a + n for a, n in zip(done, step)]
        sl, cu = torch.tensor(done, dtype=torch.int32).cuda(), offsets(step).cuda()
        one = step == [1, 1]
        kv_cache_append(kk, vv, kc, vc, sc, bt, sl, None if one else cu)
        if one:
            o, lse = paged_attention_decode(qq, kc, vc, bt, sl, return_lse=True, kv_scales=sc, window=window, sinks=sinks)
        else:
            o, lse = paged_prefill(qq, kc, vc, bt, cu, sl, return_lse=True, kv_scales=sc, window=window, sinks=sinks)
            lse = lse.t()
        vals = paged8.cache_values(*(t.cpu().view(torch.uint8) for t in (kc, vc, sc)))
        ref = paged8.window_reference(qq.cpu(), *vals, table, cu.cpu(), done, window, sinks)
        _assert_close(o, lse, ref, 160, f"after {done}")
        for b in range(2):  # what the cache stands for is the rows themselves, rounded
            rows = paged8.rows_of(vals[0], table, b, done[b])
            assert torch.equal(rows, paged8.values(*paged8.quantise_rows(k[b, :done[b]])))


def _random_case(seed):
    import random
    r = random.Random(seed)
    kind, dtype = r.choice(KINDS)
    hkv, group, d = r.choice([1, 2, 3, 8]), r.choice([1, 2, 4, 7, 8, 12]), r.choice([16, 48, 64, 80, 96, 128])
    bs = r.choice([16, 32, 64])
    b = r.randint(1, 9)
    new = [r.choice([0, 1, r.randint(1, 8), r.randint(1, 200)]) for _ in range(b)]
    had = [r.choice([0, r.randint(0, 40), r.randint(0, 1500)]) for _ in range(b)]
    window = r.choice([None, r.randint(1, 40), r.randint(1, 700)]) if kind == "e4m3" else r.randint(1, 300)
    sinks = 0 if window is None else r.choice([0, 1, 4, r.randint(0, 90)])
    return kind, dtype, new, had, hkv * group, hkv, d, bs, window, sinks


@pytest.mark.parametrize("seed", range(24))
def test_random_chunks(gpu, seed):
    case = _random_case(seed)
    print(f"case random chunks seed={seed} {case}", flush=True)
    *how, window, sinks = case
    _chunk(*how, 600 + seed, window, sinks, what=f"seed {seed}")


@pytest.mark.parametrize("seed", range(24, 40))
def test_random_decode(gpu, seed):
    kind, dtype, new, had, hq, hkv, d, bs, window, sinks = _random_case(seed)
    print(f"case random decode seed={seed}", flush=True)
    _decode(kind, dtype, [5 * h for h in had], hq, hkv, d, bs, 700 + seed, window, sinks, what=f"seed {seed}")


def test_cache_past_32_bits(gpu):
    """A cache of more than 4 GiB: its last blocks."""
    print("case cache past 32 bits", flush=True)
    blocks = (1 << 32) // (16 * 8 * 128) + 10
    kc, vc = (torch.empty(blocks, 16, 8, 128, dtype=torch.uint8, device="cuda") for _ in range(2))
    sc = torch.empty(blocks, 8, 16, 2, dtype=torch.uint8, device="cuda")
    ids = [blocks - 1, blocks // 2, blocks - 7, 3]
    small = cache8(4, 16, 8, 128, 51)
    for i, blk in enumerate(ids):
        kc[blk], vc[blk], sc[blk] = (t[i].cuda() for t in small)
    q = _q(1, 16, 128, torch.bfloat16, 52)
    o, lse = paged_attention_decode(q.cuda(), kc.view(E4M3), vc.view(E4M3), torch.tensor([ids], dtype=torch.int32).cuda(),
                                    torch.tensor([60], dtype=torch.int32).cuda(), return_lse=True, kv_scales=sc)
    ref = paged8.window_reference(q, *paged8.cache_values(*small), torch.arange(4)[None], None, [60])
    _assert_close(o, lse, ref, 60, "far blocks")
    q = _q(50, 16, 128, torch.bfloat16, 53)
    o, lse = paged_prefill(q.cuda(), kc.view(E4M3), vc.view(E4M3), torch.tensor([ids], dtype=torch.int32).cuda(),
                           offsets([50]).cuda(), torch.tensor([60], dtype=torch.int32).cuda(), return_lse=True, kv_scales=sc)
    ref = paged8.window_reference(q, *paged8.cache_values(*small), torch.arange(4)[None], offsets([50]), [60])
    _assert_close(o, lse.t(), ref, 60, "far blocks, chunk")


def test_host_threads_on_one_stream(gpu):
    """Calls of two launches (key splits of a chunk, long runs of a decode step), calls of one and skinny products from three
    threads that all use the default stream: every result is the one that the call gives alone."""
    import threading

    from lightserve_amd.kernels.tiled_matmul import skinny_matmul
    print("case threads", flush=True)
    lens = [12000, 9000, 11000]
    table, pool = tables(lens, 16, 80)
    cache, _ = _cache("e4m3", torch.bfloat16, pool, 16, 8, 64, 81)
    bt, sl = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    q, cu = _q(90, 16, 64, torch.bfloat16, 82).cuda(), offsets([30, 20, 40]).cuda()
    x, w = (torch.randn(n, 4096, generator=torch.Generator().manual_seed(83)).to(torch.bfloat16).cuda() for n in (2, 4096))
    calls = [lambda: paged_prefill(q, *cache[:2], bt, cu, sl, max_seqlen_q=40, kv_scales=cache[2]),
             lambda: paged_attention_decode(q[:3], *cache[:2], bt, sl, max_seq_len=12000, kv_scales=cache[2]),
             lambda: paged_attention_decode(q[3:6], *cache[:2], bt, sl, max_seq_len=12000, kv_scales=cache[2]),
             lambda: paged_attention_decode(q[:3], *cache[:2], bt, sl, max_seq_len=300, kv_scales=cache[2]),
             lambda: skinny_matmul(x, w)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    got, start = [[], [], []], threading.Barrier(3)

    def run(i):
        start.wait(timeout=60)
        for turn in range(60):
            at = (turn + 2 * i) % len(calls)
            got[i].append((at, calls[at]()))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for results in got:
        assert len(results) == 60
        for at, out in results:
            assert torch.equal(out, want[at]), f"call {at}"


@pytest.mark.parametrize("kind", ["e4m3", "16 bit"])
@pytest.mark.parametrize("d", [64, 128])
def test_one_value_not_finite_after_a_long_prefix(gpu, kind, d):
    """A NaN in the diagonal tiles of a long item: the rows that see it alone, the other rows of their wave as without it, and
    no more than a few times the call's own time (a walk over the keys one by one takes 50 to 100 times as long)."""
    had, n, hq, hkv, dtype = 8192, 2048, 32, 8, torch.bfloat16
    print(f"case NaN after a long prefix {kind} d={d}", flush=True)
    length, at, channel = had + n, had + 700, 9
    table, pool = tables([length], 16, 84)
    cache, vals = _cache(kind, dtype, pool, 16, hkv, d, 85)
    how = dict(max_seqlen_q=n, return_lse=True, kv_scales=cache[2], **({} if kind == "e4m3" else dict(window=length)))
    q, sl = _q(n, hq, d, dtype, 86), torch.tensor([length], dtype=torch.int32).cuda()
    bt, cu, qd = table.cuda(), offsets([n]).cuda(), q.cuda()

    def timed():
        times = []
        for _ in range(4):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            out = paged_prefill(qd, *cache[:2], bt, cu, sl, **how)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return min(times), out

    clean, _ = timed()
    bits = cache[1].view(torch.uint8 if kind == "e4m3" else torch.int16)
    bits[table[0, at // 16], at % 16, :, channel] = 127 if kind == "e4m3" else 0x7fc0
    dirty, (o, lse) = timed()
    print(f"[time] clean {1e3 * clean:.0f} us, with a NaN {1e3 * dirty:.0f} us", flush=True)
    o, lse = o.cpu(), lse.t().cpu()
    assert torch.isfinite(o[:700]).all() and torch.isnan(o[700:, :, channel]).all()
    others = torch.arange(d) != channel
    assert torch.isfinite(o[:, :, others]).all()
    for first, last in ((0, 20), (680, 720)):  # (the row tile that the NaN cuts, and one before)
        ref = paged8.window_reference(q[first:last], *vals, table, offsets([last - first]), [had + last])
        got = o[first:last].clone()
        got[:, :, channel] = torch.where(torch.isnan(got[:, :, channel]), ref[0][:, :, channel].to(dtype), got[:, :, channel])
        _assert_close(got, lse[first:last], ref, length, f"rows {first} to {last}")
    assert dirty <= 25 * clean, "the other rows' sums cost too much"


# Chunks for the wide kernel: (queries a sequence, heads, KV heads, head dim): key splits, a head dim with padding, eight waves.
WIDE = [(40, 4, 2, 64), (200, 4, 2, 80), (64, 16, 8, 128), (1030, 32, 4, 64)]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("n,hq,hkv,d", WIDE)
def test_what_no_query_of_a_chunk_sees_is_not_read(gpu, kind, dtype, n, hq, hkv, d):
    """As test_what_no_query_sees_is_not_read, in the wide kernel: NaN codes, scales of 255, NaN and infinities in K and V and
    wild table entries between the sinks and the window, behind the sequences and in blocks of nobody."""
    print(f"case unseen rows of a chunk {kind} {dtype} n={n} hq={hq} d={d}", flush=True)
    lens, bs, window, sinks = [n + 300, n, n + 150], 16, 40, 5
    table, pool = tables(lens, bs, 90)
    q = _q(3 * n, hq, d, dtype, 91)
    clean = cache8(pool, bs, hkv, d, 92)
    vals = paged8.cache_values(*clean)
    if kind == "e4m3":
        kc, vc, sc = (t.clone() for t in clean)
        bad_k = bad_v = 127
    else:
        kc, vc, sc = vals[0].to(dtype), vals[1].to(dtype), None
        vals, bad_k, bad_v = (kc.double(), vc.double()), math.nan, math.inf
        kc, vc = kc.clone(), vc.clone()
    seen = torch.zeros(pool, bs, dtype=torch.bool)
    dirty = table.clone()
    for b, length in enumerate(lens):
        pos = torch.arange(length)
        pos = pos[(pos < sinks) | (pos > length - n - window)]
        seen[table[b, pos // bs].long(), pos % bs] = True
        for i in set(range(table.shape[1])) - set((pos // bs).tolist()):
            dirty[b, i] = [-5, 1 << 30, pool, int(table[0, 0])][i % 4]
    kc[~seen], vc[~seen] = bad_k, bad_v
    if sc is not None:
        sc.transpose(1, 2)[~seen] = 255
    cache = [t.cuda().view(E4M3) if sc is not None else t.cuda() for t in (kc, vc)]
    sl, cu = torch.tensor(lens, dtype=torch.int32).cuda(), offsets([n] * 3)
    o, lse = paged_prefill(q.cuda(), *cache, dirty.cuda(), cu.cuda(), sl, max_seqlen_q=n, return_lse=True,
                           kv_scales=sc.cuda() if sc is not None else None, window=window, sinks=sinks)
    _assert_close(o, lse.t(), paged8.window_reference(q, *vals, table, cu, lens, window, sinks), max(lens), "wide")


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("n,hq,hkv,d", WIDE)
def test_nan_of_a_key_and_blocks_outside_in_chunks(gpu, kind, dtype, n, hq, hkv, d):
    """A NaN in K reaches the rows that see its key, whole, and no other; blocks outside the cache read as zeros."""
    print(f"case NaN keys of a chunk {kind} {dtype} n={n} hq={hq} d={d}", flush=True)
    lens, window, sinks = [n + 100, n], 30, 2
    table, pool = tables(lens, 16, 93)
    cache, vals = _cache(kind, dtype, pool, 16, hkv, d, 94)
    at = 100 + n // 2
    bits = cache[0].view(torch.uint8 if kind == "e4m3" else torch.int16)
    bits[table[0, at // 16], at % 16, :, d - 3] = 255 if kind == "e4m3" else -1
    lost = table.clone()
    lost[0, 97 // 16], lost[1, 0] = pool, -1
    q = _q(2 * n, hq, d, dtype, 95)
    cu = offsets([n, n])
    p = torch.arange(100, 100 + n)
    for w, s in ((window, sinks), (None, 0)):
        if w is None and kind != "e4m3":
            continue
        o, lse = (t.cpu() for t in paged_prefill(q.cuda(), *cache[:2], lost.cuda(), cu.cuda(),
                                                 torch.tensor(lens, dtype=torch.int32).cuda(), max_seqlen_q=n, return_lse=True,
                                                 kv_scales=cache[2], window=w, sinks=s))
        lse = lse.t().contiguous()
        sees = (at <= p) & ((at > p - w) if w is not None else True)
        assert torch.isnan(o[:n][sees]).all() and torch.isnan(lse[:n][sees]).all() and sees.any() and not sees.all()
        ref = paged8.window_reference(q, *vals, lost, cu, lens, w, s)
        o[:n][sees], lse[:n][sees] = ref[0][:n][sees].to(dtype), ref[1][:n][sees].float()
        _assert_close(o, lse, ref, max(lens), f"the others w={w}")


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(64, 1, 64), (96, 2, 128), (66, 2, 80), (128, 1, 128)])
def test_decode_of_many_heads_on_one(gpu, kind, dtype, hq, hkv, d):
    """More than 32 query heads on a KV head, which go to the wide kernel without offsets: lengths around its tiles, long ones
    whose keys are split, more sequences than lanes."""
    print(f"case decode of many heads {kind} {dtype} hq={hq} hkv={hkv} d={d}", flush=True)
    for lens in ([1, 15, 63, 64, 65, 0, 129, 500], [9000, 3, 2500], [(29 * b * b) % 300 for b in range(70)]):
        for window, sinks in ((None, 0), (200, 3)):
            if window is not None or kind == "e4m3":
                _decode(kind, dtype, lens, hq, hkv, d, 16, hq + d, window, sinks, what=f"{len(lens)} sequences w={window}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,had,hq,hkv", [(40, 200, 4, 1), (40, 3000, 4, 1), (2048, 150, 32, 2)])
def test_scores_that_rise_in_chunks(gpu, dtype, n, had, hq, hkv):
    """Scores near zero in a row's first tile and far above the offset that it set later: the exponentials are taken again and
    the sums scaled; whole items of four and of eight waves, and splits."""
    print(f"case rising scores {dtype} n={n} had={had}", flush=True)
    length, d = n + had, 64
    table, pool = tables([length], 16, 96)
    kc, vc, sc = cache8(pool, 16, hkv, d, 97)
    g = torch.Generator().manual_seed(98)
    for i in range(-(-length // 16)):  # first tiles of 2^-12, then each 64 keys one of 2^-7 .. 2^-2 of the codes' values
        e = 115 if i < 4 else int(torch.randint(119, 125, (1,), generator=g))
        sc[table[0, i], ..., 0] = e
    vals = paged8.cache_values(kc, vc, sc)
    q = _q(n, hq, d, dtype, 99)
    scores = (q[-1, 0].double() @ paged8.rows_of(vals[0], table, 0, length)[:, 0].T) / 8 / math.log(2)
    assert scores[64:].max() - scores[:64].max() > 20  # past 2^15 of fp16 after the first tile
    o, lse = paged_prefill(q.cuda(), kc.cuda().view(E4M3), vc.cuda().view(E4M3), table.cuda(), offsets([n]).cuda(),
                           torch.tensor([length], dtype=torch.int32).cuda(), max_seqlen_q=n, return_lse=True, kv_scales=sc.cuda())
    want, want_lse, a, big = paged8.window_reference(q, *vals, table, offsets([n]), [length])
    if dtype == torch.float16:
        # Scores this far apart bring p into fp16's subnormals, which the bound leaves out: there a p (relative to the row's
        # offset) is off by at most half of 2^-24. The offset is the largest score of one of the row's tiles, so one p of the row
        # is at least 1 and their sum l too, and sums under a lower offset are scaled by less than 1 when it rises: o is off by
        # at most 2^-25 sum |v_j| / l <= 2^-25 sum |v_j| over the keys that the row sees. As 2u a = 2^-10 a, a takes that in as
        # 2^-15 sum |v_j|.
        v = paged8.rows_of(vals[1], table, 0, length).abs().cumsum(0)[had:].repeat_interleave(hq // hkv, 1)
        a = a + 2.0 ** -15 * v
    _assert_close(o, lse.t(), (want, want_lse, a, big), length, "rising")
