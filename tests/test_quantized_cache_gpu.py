"""The 8-bit paged cache on the GPU: quantise on write and read back, bit for bit against the float64 oracle.

Scales are powers of two, so codes, exponents and what is read back are exact numbers: there is no tolerance, but for rows read
into a 16-bit type that is coarser than the codes' values (fp16's subnormals), which are the oracle's values cast once.
"""
import math

import pytest
import torch

from lightserve_amd.kernels.flash_attention_varlen import flash_attention_varlen_forward
from lightserve_amd.kernels.paged_attention import paged_attention_decode, paged_prefill
from lightserve_amd.kernels.quantized_kv_cache import kv_cache_append, kv_cache_read, quantized_kv_cache
from oracle import paged8
from tests.paged8_cases import cache8, offsets, tables

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _same_codes(got, want, what):
    """Equal bits; any NaN stands for NaN."""
    got, want = got.cpu().view(torch.uint8), want
    nan = (want & 127) == 127
    assert torch.equal((got & 127) == 127, nan) and torch.equal(got[~nan], want[~nan]), what


def _rows(t, heads, d, dtype, seed, spread=12):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, heads, d, generator=g) * torch.exp2(torch.randint(-spread, spread, (t, heads, 1), generator=g).float())
    return x.to(dtype)


def _append(k, v, cache, table, seq_lens, cu, what):
    kc, vc, sc = cache
    want = paged8.append_reference(k, v, kc, vc, sc, table, seq_lens, cu)
    gk, gv, gs = kc.cuda().view(E4M3), vc.cuda().view(E4M3), sc.cuda()
    kv_cache_append(k.cuda(), v.cuda(), gk, gv, gs, table.cuda(), seq_lens.int().cuda(), cu.cuda() if cu is not None else None)
    torch.cuda.synchronize()
    _same_codes(gk, want[0], f"{what} k")
    _same_codes(gv, want[1], f"{what} v")
    assert torch.equal(gs.cpu(), want[2]), f"{what} scales"
    return gk, gv, gs


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,d,bs", [(8, 128, 16), (3, 80, 32), (1, 64, 64), (2, 16, 16), (5, 112, 16)])
def test_append_chunks(gpu, heads, d, bs, dtype):
    """Ragged chunks onto ragged prefixes, an empty one among them; everything else in the cache stays."""
    print(f"case append heads={heads} d={d} bs={bs} {dtype}", flush=True)
    new, had = [1, 17, 0, 40, 5], [0, 15, 9, 33, 100]
    total = [a + b for a, b in zip(new, had)]
    table, pool = tables(total, bs, 1)
    k, v = (_rows(sum(new), heads, d, dtype, s) for s in (2, 3))
    _append(k, v, cache8(pool, bs, heads, d, 4), table, torch.tensor(total), offsets(new), "chunks")


@pytest.mark.parametrize("batch", [1, 8, 70, 1030])
def test_append_one_row_each(gpu, batch):
    """A decode step; a sequence of no tokens stores nothing."""
    print(f"case append step batch={batch}", flush=True)
    lens = [(7 * b) % 50 for b in range(batch)]
    table, pool = tables(lens, 16, 5)
    k, v = (_rows(batch, 2, 64, torch.bfloat16, s) for s in (6, 7))
    _append(k, v, cache8(pool, 16, 2, 64, 8), table, torch.tensor(lens), None, "step")


@pytest.mark.parametrize("batch", [1, 64, 1023, 1024, 1025])
def test_append_many_sequences(gpu, batch):
    """Offsets searched in LDS (up to 1024 sequences) and in memory."""
    print(f"case append offsets batch={batch}", flush=True)
    new = [b % 3 for b in range(batch)]
    new[-1] += 1
    table, pool = tables(new, 16, 9)
    k, v = (_rows(sum(new), 1, 16, torch.float16, s) for s in (10, 11))
    _append(k, v, cache8(pool, 16, 1, 16, 12), table, torch.tensor(new), offsets(new), "offsets")


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_extreme_rows(gpu, dtype):
    """Zeros, the type's largest and smallest values, infinities, NaN, ties of the codes' rounding, and every binade's edges."""
    print(f"case append extremes {dtype}", flush=True)
    info, d = torch.finfo(dtype), 32
    special = [0.0, -0.0, info.max, -info.max, info.tiny, info.smallest_normal / 2, math.inf, -math.inf, math.nan, 448.0, 449.0,
               1.0, 336.0, -336.0, 0.9375, 208.0]
    rows = [[a, b] + [0.0] * (d - 2) for a in special for b in special]
    rows += [[448.0 * 2.0 ** e * f] + [2.0 ** e * (1 + i / 16) for i in range(d - 1)] for e in range(-14, 7) for f in (0.99, 1.0, 1.01)]
    rows += [[224.0 + 0.5] + [2.0 ** -9 * i / 2 for i in range(d - 1)], [math.inf] * d, [math.nan] * d, [-info.max] * d]
    k = torch.tensor(rows, dtype=torch.float64).to(dtype)[:, None]
    v = k.flip(0).contiguous()
    n = k.shape[0]
    table, pool = tables([n], 16, 13)
    gk, gv, gs = _append(k, v, cache8(pool, 16, 1, d, 14), table, torch.tensor([n]), offsets([n]), "extremes")
    back, _ = kv_cache_read(gk, gv, gs, table.cuda(), offsets([n]).cuda(), dtype=dtype)
    assert torch.equal(torch.isnan(back.cpu()), ~torch.isfinite(k)), "finite rows read back finite in their own type"
    assert torch.isfinite(back.cpu()[torch.isfinite(k)]).all()


def test_append_rows_that_have_no_place(gpu):
    """Rows behind the last sequence, before position 0, past the table, and in blocks that are not there."""
    print("case append without a place", flush=True)
    table = torch.tensor([[3, -1, 99], [1, 0, 2]], dtype=torch.int32)
    cu = torch.tensor([0, 40, 45], dtype=torch.int32)
    k, v = (_rows(50, 2, 32, torch.bfloat16, s) for s in (15, 16))
    for lens in ([40, 3], [48, 50], [0, 5], [-7, 60]):
        _append(k, v, cache8(4, 16, 2, 32, 17), table, torch.tensor(lens), cu, str(lens))


def test_append_strided(gpu):
    """Rows inside a fused projection, caches that are slices of larger ones, a table slice with another column stride."""
    print("case append strided", flush=True)
    new = [9, 20]
    table, pool = tables(new, 16, 18)
    qkv = _rows(29, 8, 64, torch.bfloat16, 19).cuda()
    k, v = qkv[:, 4:6], qkv[:, 6:8]
    kc, vc, sc = cache8(pool, 16, 2, 64, 20)
    want = paged8.append_reference(k.cpu(), v.cpu(), kc, vc, sc, table, torch.tensor(new), offsets(new))
    big = torch.zeros(2, pool, 16, 2, 2, 64, dtype=torch.uint8, device="cuda")
    big[0, :, :, 0], big[1, :, :, 1] = kc.cuda(), vc.cuda()
    wide = torch.zeros(2, table.shape[1] * 2, dtype=torch.int32)
    wide[:, ::2] = table
    gs = sc.cuda()
    kv_cache_append(k, v, big[0, :, :, 0].view(E4M3), big[1, :, :, 1].view(E4M3), gs, wide.cuda()[:, ::2],
                    torch.tensor(new, dtype=torch.int32).cuda(), offsets(new).cuda())
    torch.cuda.synchronize()
    _same_codes(big[0, :, :, 0].contiguous(), want[0], "k")
    _same_codes(big[1, :, :, 1].contiguous(), want[1], "v")
    assert torch.equal(gs.cpu(), want[2])
    assert (big[0, :, :, 1] == 0).all() and (big[1, :, :, 0] == 0).all()
    odd = _rows(29, 2, 68, torch.bfloat16, 19).cuda()[:, :, 2:66]  # rows that are not 16-byte aligned are copied
    kv_cache_append(odd, odd, big[0, :, :, 0].view(E4M3), big[1, :, :, 1].view(E4M3), gs, table.cuda(),
                    torch.tensor(new, dtype=torch.int32).cuda(), offsets(new).cuda())
    want = paged8.append_reference(odd.cpu(), odd.cpu(), kc, vc, sc, table, torch.tensor(new), offsets(new))
    _same_codes(big[0, :, :, 0].contiguous(), want[0], "unaligned k")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,d,bs", [(8, 128, 16), (3, 80, 32), (1, 64, 64), (2, 16, 16)])
def test_read(gpu, heads, d, bs, dtype):
    """Whole and partial sequences, empty ones, entries outside the cache, rows behind the last sequence."""
    print(f"case read heads={heads} d={d} bs={bs} {dtype}", flush=True)
    lens = [33, 0, 100, 1, 64]
    table, pool = tables(lens, bs, 21)
    table[2, 1] = pool + 5
    kc, vc, sc = cache8(pool, bs, heads, d, 22)
    sc[0] += 100
    cu, total = offsets(lens), sum(lens) + 7
    want = paged8.read_reference(kc, vc, sc, table, cu, total)
    got = kv_cache_read(kc.cuda().view(E4M3), vc.cuda().view(E4M3), sc.cuda(), table.cuda(), cu.cuda(), total=total, dtype=dtype)
    for g, w in zip(got, want):
        assert g.dtype == dtype and torch.equal(g.cpu(), w.float().to(dtype))
    short = kv_cache_read(kc.cuda().view(E4M3), vc.cuda().view(E4M3), sc.cuda(), table.cuda(), cu.cuda(), total=50, dtype=dtype)
    assert torch.equal(short[0].cpu(), want[0][:50].float().to(dtype))


def test_read_feeds_the_packed_attention(gpu):
    """Appended prefixes read back are what flash_attention_varlen_forward takes."""
    print("case read then packed attention", flush=True)
    lens = [130, 17, 64]
    table, pool = tables(lens, 16, 23)
    k, v = (_rows(sum(lens), 2, 64, torch.bfloat16, s, spread=1) for s in (24, 25))
    q = _rows(sum(lens), 4, 64, torch.bfloat16, 26, spread=1).cuda()
    kc, vc, sc = quantized_kv_cache(pool, 16, 2, 64)
    cu = offsets(lens).cuda()
    kv_cache_append(k.cuda(), v.cuda(), kc, vc, sc, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), cu)
    kr, vr = kv_cache_read(kc, vc, sc, table.cuda(), cu)
    for got, x in ((kr, k), (vr, v)):
        assert torch.equal(got.cpu().double(), paged8.values(*paged8.quantise_rows(x)))
    o, _ = flash_attention_varlen_forward(q, kr, vr, cu, cu, 130, 130, causal=True)
    assert torch.isfinite(o).all()


def test_captured_and_replayed(gpu):
    """A step captured in a graph appends what is in its inputs at each replay, beside eager calls."""
    print("case append in a graph", flush=True)
    lens = [20, 5, 31]
    table, pool = tables([40] * 3, 16, 27)
    codes, out = cache8(pool, 16, 2, 64, 28), None
    gk, gv, gs = codes[0].cuda().view(E4M3), codes[1].cuda().view(E4M3), codes[2].cuda()
    k, v = (_rows(3, 2, 64, torch.bfloat16, s).cuda() for s in (29, 30))
    sl, bt, cu = torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda(), offsets(lens).cuda()
    kv_cache_append(k, v, gk, gv, gs, bt, sl)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_cache_append(k, v, gk, gv, gs, bt, sl)
        out = kv_cache_read(gk, gv, gs, bt, cu, total=sum(lens))
    for i in range(4):
        k.copy_(_rows(3, 2, 64, torch.bfloat16, 31 + i))
        v.copy_(_rows(3, 2, 64, torch.bfloat16, 41 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = paged8.append_reference(k.cpu(), v.cpu(), *codes, table, torch.tensor(lens))
        codes = want
        _same_codes(gk, want[0], "k")
        assert torch.equal(gs.cpu(), want[2])
        eager = kv_cache_read(gk, gv, gs, bt, cu, total=sum(lens))
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_another_stream(gpu):
    print("case append on another stream", flush=True)
    table, pool = tables([64], 16, 32)
    kc, vc, sc = quantized_kv_cache(pool, 16, 2, 64)
    cu, sl, bt = offsets([64]).cuda(), torch.tensor([64], dtype=torch.int32).cuda(), table.cuda()
    src = _rows(64, 2, 64, torch.bfloat16, 33).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        k = src * 1.0
        kv_cache_append(k, k, kc, vc, sc, bt, sl, cu)
        got = kv_cache_read(kc, vc, sc, bt, cu, total=64)[0]
    stream.synchronize()
    assert torch.equal(got.cpu().double(), paged8.values(*paged8.quantise_rows(src.cpu())))


def test_offsets_past_32_bits(gpu):
    """A cache of more than 4 GiB: its last block."""
    print("case append past 32 bits", flush=True)
    blocks = (1 << 32) // (16 * 8 * 128) + 10
    kc, vc = (torch.empty(blocks, 16, 8, 128, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    sc = torch.ones(blocks, 8, 16, 2, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[blocks - 1, blocks // 2]], dtype=torch.int32)
    k, v = (_rows(20, 8, 128, torch.bfloat16, s) for s in (34, 35))
    cu = offsets([20]).cuda()
    kv_cache_append(k.cuda(), v.cuda(), kc, vc, sc, table.cuda(), torch.tensor([20], dtype=torch.int32).cuda(), cu)
    gk, gv = kv_cache_read(kc, vc, sc, table.cuda(), cu, total=20, dtype=torch.float32)
    assert torch.equal(gk.cpu().double(), paged8.values(*paged8.quantise_rows(k)))
    assert torch.equal(gv.cpu().double(), paged8.values(*paged8.quantise_rows(v)))


def test_rows_at_odd_addresses_and_shared_tables(gpu):
    """Packed rows that begin between two 16-byte pieces; a table that both sequences share; a column as one sequence's table."""
    print("case odd addresses", flush=True)

    def shifted(x):
        t = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
        assert t.data_ptr() % 16 != 0
        return t.copy_(x)

    kc, vc, sc = cache8(4, 16, 2, 64, 50)
    k, v = (_rows(2, 2, 64, torch.bfloat16, s) for s in (51, 52))
    q = _rows(2, 4, 64, torch.bfloat16, 53, spread=1)
    shared = torch.tensor([2, 0], dtype=torch.int32).expand(2, 2)
    column = torch.tensor([[3], [1]], dtype=torch.int32).t()
    for table, lens in ((shared, [18, 20]), (column, [25])):
        n = len(lens)
        sl = torch.tensor(lens, dtype=torch.int32)
        want = paged8.append_reference(k[:n], v[:n], kc, vc, sc, table, sl)
        gk, gv, gs = kc.cuda().view(E4M3), vc.cuda().view(E4M3), sc.cuda()
        dev = shared.cuda()[0].expand(2, 2) if table is shared else table.t().contiguous().cuda().t()
        kv_cache_append(shifted(k[:n]), shifted(v[:n]), gk, gv, gs, dev, sl.cuda())
        _same_codes(gk, want[0], "k")
        _same_codes(gv, want[1], "v")
        assert torch.equal(gs.cpu(), want[2])
        cu = offsets([1] * n).cuda()
        for call in (lambda x, t: paged_attention_decode(x, gk, gv, t, sl.cuda(), kv_scales=gs),
                     lambda x, t: paged_prefill(x, gk, gv, t, cu, sl.cuda(), kv_scales=gs, window=7)):
            assert torch.equal(call(shifted(q[:n]), dev), call(q[:n].cuda(), dev.contiguous().clone()))


@pytest.mark.parametrize("d,lanes", [(80, 16), (16, 8)])
def test_as_many_rows_as_a_launch_has_threads_for(gpu, d, lanes):
    """The largest append that is not refused, of one row over and over (a stride of 0): its last rows are stored."""
    rows = (1 << 32) // lanes - 64
    print(f"case append of {rows} rows d={d}", flush=True)
    kc, vc, sc = quantized_kv_cache(2, 16, 1, d)
    k, v = (_rows(1, 1, d, torch.bfloat16, s) for s in (60, 61))
    table, sl = torch.tensor([[1, 0]], dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    cu = torch.tensor([0, rows], dtype=torch.int32)
    kv_cache_append(k.cuda().expand(rows, 1, d), v.cuda().expand(rows, 1, d), kc, vc, sc, table.cuda(), sl.cuda(), cu.cuda())
    torch.cuda.synchronize()
    empty = (torch.zeros(2, 16, 1, d, dtype=torch.uint8), torch.zeros(2, 16, 1, d, dtype=torch.uint8), torch.ones_like(sc.cpu()))
    want = paged8.append_reference(k.expand(20, 1, d), v.expand(20, 1, d), *empty, table, sl, offsets([20]))
    _same_codes(kc, want[0], "k")
    _same_codes(vc, want[1], "v")
    assert torch.equal(sc.cpu(), want[2])


def test_the_packed_attention_over_rows_read_back(gpu):
    """Its output against the oracle's on what the cache stands for. u is half a step of bf16: the weights are rounded to it and
    their sum with them (2u of sum w |v|), o once more; the scores' fp32 sums add e = (64 + 16) 2^-24 big + 2^-19 twice."""
    print("case packed attention on rows read back", flush=True)
    lens = [130, 17, 64]
    table, pool = tables(lens, 16, 62)
    cu, sl = offsets(lens).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    k, v = (_rows(sum(lens), 2, 64, torch.bfloat16, s, spread=1).cuda() for s in (63, 64))
    q = _rows(sum(lens), 4, 64, torch.bfloat16, 65, spread=1)
    kc, vc, sc = quantized_kv_cache(pool, 16, 2, 64)
    kv_cache_append(k, v, kc, vc, sc, table.cuda(), sl, cu)
    o, _ = flash_attention_varlen_forward(q.cuda(), *kv_cache_read(kc, vc, sc, table.cuda(), cu), cu, cu, 130, 130, causal=True)
    vals = paged8.cache_values(*(t.cpu().view(torch.uint8) for t in (kc, vc, sc)))
    want, _, a, big = paged8.window_reference(q, *vals, table, offsets(lens), lens)
    u, e = torch.finfo(torch.bfloat16).eps / 2, 80 * 2.0 ** -24 * big + 2.0 ** -19
    tol = 1.05 * ((2 * u + 2 * e[..., None] + 130 * 2.0 ** -24) * a + u * want.abs()) + 2.0 ** -24
    assert ((o.cpu().double() - want).abs() <= tol).all()
