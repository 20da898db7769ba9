"""Beam search's selection and the reordering of the beams' caches, against the float64 oracle.

Which candidates are chosen is compared exactly: their scores differ by far more than the kernel's sums are off (checked for each
case), or are equal and go by index. A returned score is the 64-bit one rounded once, whose logarithm of a sum of
exponentials is off by less than 2^-23 (each exponential is, relatively): 2^-24 |score| + 2^-23.
"""
import math

import pytest
import torch

from lightserve_amd.kernels.beam_search import beam_search_select, kv_cache_reorder
from oracle import candidates
from tests.candidate_cases import E4M3, layer_caches, on_gpu, raw

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _select(logits, scores, num, what, dev=None, apart=True):
    got = beam_search_select(logits.cuda() if dev is None else dev, scores.cuda(), num)
    torch.cuda.synchronize()
    k, vocab = scores.shape[1], logits.shape[1]
    for b in range(scores.shape[0]):
        want = candidates.select_reference(logits[b * k:(b + 1) * k], scores[b:b + 1], num + 1)[0]
        if apart:
            gaps = [x[0] - y[0] for x, y in zip(want, want[1:]) if x[1] != y[1] and x[0] > y[0] and y[0] > -math.inf]
            assert not gaps or min(gaps) > 1e-6, f"{what}: the case leaves two candidates too near to each other"
        want = want[:num]
        assert got[1][b].tolist() == [w[1] for w in want], f"{what}: beams of {b}"
        assert got[2][b].tolist() == [w[2] for w in want], f"{what}: tokens of {b}"
        for x, w in zip(got[0][b].tolist(), want):
            assert x == w[0] or abs(x - w[0]) <= 2.0 ** -24 * abs(w[0]) + 2.0 ** -23, f"{what}: score {x} for {w[0]}"


def _logits(rows, vocab, dtype, seed, spread=2.5):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


def _scores(n, k, seed):
    return -torch.rand(n, k, generator=torch.Generator().manual_seed(seed + 1000)) * 6 - 3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 2048, 2049, 32000])
@pytest.mark.parametrize("n,k,num", [(1, 1, 1), (1, 4, 8), (3, 5, 5), (2, 2, 64)])
def test_select(gpu, dtype, vocab, n, k, num):
    print(f"case select {dtype} vocab={vocab} n={n} k={k} num={num}", flush=True)
    _select(_logits(n * k, vocab, dtype, vocab + num), _scores(n, k, vocab), num, "random")


@pytest.mark.parametrize("dtype", DTYPES)
def test_select_many_beams(gpu, dtype):
    print(f"case select beams {dtype}", flush=True)
    _select(_logits(64, 700, dtype, 1), _scores(1, 64, 1), 64, "64 beams")
    _select(_logits(34, 9000, dtype, 2), _scores(2, 17, 2), 34, "17 beams")
    _select(_logits(1, 120000, dtype, 3), _scores(1, 1, 3), 64, "one row")
    _select(_logits(200, 60, dtype, 4), _scores(100, 2, 4), 4, "100 sequences")


def test_select_the_most_chunks(gpu):
    """64 beams of a vocabulary of 2^18, most of it masked: the largest number of chunks that one sequence's beams have."""
    print("case select most", flush=True)
    x = torch.full((64, 2 ** 18), -math.inf, dtype=torch.bfloat16)
    at = torch.randint(0, 2 ** 18, (64, 40), generator=torch.Generator().manual_seed(9))
    x.scatter_(1, at, _logits(64, 40, torch.bfloat16, 10, 1.0))
    x[:, -1] = 3.0
    scores = torch.full((1, 64), -10.0) - torch.arange(64) / 8
    got = beam_search_select(x.cuda(), scores.cuda(), 64)
    # (the oracle's definition on the few finite logits)
    keep = [(float(scores[0, k]) + (x[k, v].double().item() - x[k].double().logsumexp(0).item()), k, v)
            for k in range(64) for v in sorted(set(at[k].tolist() + [2 ** 18 - 1]))]
    want = sorted(keep, key=lambda c: (-c[0], c[1], c[2]))[:64]
    gaps = [a[0] - b[0] for a, b in zip(want, want[1:]) if a[1] != b[1]]
    assert min(gaps) > 1e-6
    assert got[1][0].tolist() == [w[1] for w in want] and got[2][0].tolist() == [w[2] for w in want]


@pytest.mark.parametrize("dtype", DTYPES)
def test_select_ties(gpu, dtype):
    """Equal candidates go to the lower beam, then the lower token: equal logits, equal beams, and both."""
    print(f"case select ties {dtype}", flush=True)
    few = torch.randint(-2, 3, (8, 5000), generator=torch.Generator().manual_seed(1)).to(dtype)
    _select(few, _scores(2, 4, 1), 40, "few values")
    _select(torch.zeros(3, 20000, dtype=dtype), _scores(1, 3, 2), 64, "all equal")
    same = _logits(1, 3000, dtype, 3).repeat(4, 1)
    _select(same, torch.full((1, 4), -2.5), 12, "equal beams")
    _select(torch.zeros(4, 9000, dtype=dtype), torch.full((1, 4), -1.0), 64, "everything equal")
    _select(torch.tensor([[-0.0, 0.0, -0.0, -1.0]]).to(dtype), torch.zeros(1, 1), 3, "signed zeros")
    up = torch.arange(9000).float().div(700).to(dtype)[None]
    _select(up, torch.zeros(1, 1), 64, "rising")
    _select(up.flip(1), torch.zeros(1, 1), 64, "falling")


@pytest.mark.parametrize("dtype", DTYPES)
def test_select_what_offers_nothing(gpu, dtype):
    """Beams of no score, masked tokens, rows with NaN or infinities, fewer candidates than asked for."""
    print(f"case select masks {dtype}", flush=True)
    low = torch.finfo(dtype).min
    x = _logits(6, 3001, dtype, 1)
    first = torch.full((2, 3), -math.inf)
    first[:, 0] = 0.0
    _select(x, first, 6, "first step")
    _select(x, torch.tensor([[math.nan, -1.0, -math.inf], [-math.inf] * 3]), 5, "no beam at all")
    y = x.clone()
    y[0, 5], y[1, 3000], y[2] = math.nan, math.inf, -math.inf
    y[3, 7:], y[4, 2:], y[5] = -math.inf, low, low
    _select(y, _scores(2, 3, 1), 20, "rows")
    z = torch.full((2, 40000), -math.inf, dtype=dtype)
    z[0, 39999], z[1, 0], z[1, 20000] = 1.0, 2.0, 2.0
    _select(z, torch.tensor([[-1.0, -2.0]]), 7, "three candidates")
    _select(z * 1.0, torch.tensor([[-1.0, -2.0]]), 2, "two of three")


@pytest.mark.parametrize("dtype", DTYPES)
def test_select_peaked_and_large(gpu, dtype):
    """Distributions with one large logit, logits far from zero, scores far below."""
    print(f"case select large {dtype}", flush=True)
    x = _logits(4, 5000, dtype, 5)
    x[0, 17], x[1, 4000], x[2] = 60.0, 30.0, x[2] + 200
    _select(x, torch.tensor([[-1000.0, -1010.5, -990.25, -1003.0]]), 16, "peaked")
    _select(_logits(4, 5000, dtype, 6, 40.0), _scores(1, 4, 6), 16, "wide")


def test_select_near_scores(gpu):
    """Beams whose candidates differ by less than 32-bit sums tell are told apart."""
    print("case select near", flush=True)
    row = _logits(1, 4000, torch.float32, 7)
    x = row.repeat(2, 1)
    scores = torch.tensor([[-200.0, -200.0]])
    best = int(row.argmax())
    x[1, best] += 2.0 ** -18  # (below half a step of a score of 200; its row's sum grows by less)
    lse = x.double().logsumexp(1)
    gap = float((x[1, best].double() - lse[1]) - (x[0, best].double() - lse[0]))
    assert 1e-6 < gap < 2.0 ** -17
    got = beam_search_select(x.cuda(), scores.cuda(), 2)
    assert got[1].tolist() == [[1, 0]] and got[2].tolist() == [[best, best]]


@pytest.mark.parametrize("dtype", DTYPES)
def test_select_layouts(gpu, dtype):
    print(f"case select layouts {dtype}", flush=True)
    x = _logits(6, 2051, dtype, 3)
    wide = torch.full((6, 2100), 50.0, dtype=dtype)
    for shift in (0, 1, 2, 5, 8):
        wide.fill_(50.0)
        wide[:, shift:shift + 2051] = x
        _select(x, _scores(2, 3, 3), 6, f"shift {shift}", dev=wide.cuda()[:, shift:shift + 2051])
    _select(x, _scores(2, 3, 3), 6, "column-major", dev=x.t().contiguous().cuda().t())


def test_select_graph_and_streams(gpu):
    print("case select graph", flush=True)
    x, scores = _logits(8, 30000, torch.bfloat16, 3), _scores(2, 4, 3)
    dev, s = x.cuda(), scores.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam_search_select(dev, s, 8)
    for i in range(4):
        turned = x.roll(i * 11, 1)
        dev.copy_(turned)
        graph.replay()
        eager = beam_search_select(turned.cuda(), s, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), f"replay {i}"
    want = beam_search_select(x.cuda(), s, 8)
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    fixed = x.cuda()
    torch.cuda.synchronize()
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(beam_search_select(fixed, s, 8))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


# ----------------------------------------------------------------- reorder
def _beams(lens, k, bs, seed, extra=2):
    """Tables of k beams a sequence whose complete blocks are any of theirs."""
    g = torch.Generator().manual_seed(seed)
    most = max(n // bs for n in lens) + 1 + extra
    pool = len(lens) * k * most + 2
    own = torch.randperm(pool, generator=g)[:len(lens) * k * most].to(torch.int32).view(len(lens), k, most)
    table = own.clone()
    for b, n in enumerate(lens):
        table[b, :, :n // bs] = own[b].gather(0, torch.randint(0, k, (k, n // bs), generator=g))
    return table.view(len(lens) * k, most), pool


def _reorder(kind, lens, k, bs, heads, d, seed, parents=None, layers=2, what=""):
    table, pool = _beams(lens, k, bs, seed)
    ks, vs, scales = layer_caches(kind, layers, pool, bs, heads, d, seed)
    dev = on_gpu(kind, ks, vs, scales)
    if parents is None:
        parents = torch.randint(0, k, (len(lens), k), generator=torch.Generator().manual_seed(seed + 1), dtype=torch.int32)
    all_lens = torch.tensor([n for n in lens for _ in range(k)], dtype=torch.int32)
    on = table.cuda()
    kv_cache_reorder(dev[0], dev[1], on, all_lens.cuda(), parents.cuda(), kv_scales=dev[2])
    torch.cuda.synchronize()
    want, new = candidates.reorder_reference([c for c in (ks, vs, scales) if c is not None], table, all_lens, parents, (1, 1, 2))
    assert torch.equal(on.cpu(), new), f"{what}: tables"
    for got, w in zip((c for c in dev if c is not None), want):
        assert torch.equal(raw(got), raw(w)), f"{what}: rows"


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32, E4M3])
@pytest.mark.parametrize("heads,d,bs", [(1, 16, 16), (8, 128, 16), (3, 80, 64), (2, 256, 32)])
def test_reorder(gpu, kind, heads, d, bs):
    print(f"case reorder {kind} {heads} {d} {bs}", flush=True)
    _reorder(kind, [bs * 3 + 5, 0, bs - 1, bs, 1, bs * 2 + bs - 1], 4, bs, heads, d, bs + d, what="random")


@pytest.mark.parametrize("k", [1, 2, 15, 16, 17, 32, 64])
def test_reorder_beams(gpu, k):
    """Permutations, cycles and one parent of all; numbers that are no beam's."""
    print(f"case reorder k={k}", flush=True)
    for kind in (torch.bfloat16, E4M3):
        _reorder(kind, [37, 5], k, 16, 2, 64, k, what="random")
        cycle = torch.stack([torch.arange(k).roll(1), torch.arange(k).flip(0)]).int()
        _reorder(kind, [37, 5], k, 16, 2, 64, k + 1, cycle, what="permutations")
        odd = torch.full((2, k), k - 1, dtype=torch.int32)
        odd[1, :] = torch.tensor([-1, k, 2 ** 31 - 1, -2 ** 31] * 16, dtype=torch.int32)[:k]
        _reorder(kind, [37, 5], k, 16, 2, 64, k + 2, odd, what="one parent, none")


def test_reorder_long_tables(gpu):
    print("case reorder tables", flush=True)
    _reorder(torch.bfloat16, [16 * 700 + 3], 3, 16, 1, 16, 1, layers=1, what="700 blocks")
    _reorder(torch.bfloat16, [19, 40], 3, 16, 1, 64, 2, layers=9, what="layers")


def test_reorder_graph(gpu):
    """Captured with the selection that gives the parents, replayed on changing logits."""
    print("case reorder graph", flush=True)
    lens, k = [37, 60], 4
    table, pool = _beams(lens, k, 16, 1)
    ks, vs, _ = layer_caches(torch.bfloat16, 2, pool, 16, 2, 64, 2)
    kd, vd, on = ks.cuda(), vs.cuda(), table.cuda()
    all_lens = torch.tensor([n for n in lens for _ in range(k)], dtype=torch.int32)
    x, scores, ln = _logits(8, 9000, torch.bfloat16, 3), _scores(2, k, 3), all_lens.cuda()
    dev, s = x.cuda(), scores.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beam_search_select(dev, s)
        kv_cache_reorder(kd, vd, on, ln, out[1])
    for i in range(4):
        turned = x.roll(i, 0)
        dev.copy_(turned), kd.copy_(ks), vd.copy_(vs), on.copy_(table)
        graph.replay()
        torch.cuda.synchronize()
        parents = torch.tensor([[c[1] for c in row] for row in candidates.select_reference(turned, scores, k)], dtype=torch.int32)
        want, new = candidates.reorder_reference([ks, vs], table, all_lens, parents, (1, 1))
        assert torch.equal(out[1].cpu(), parents) and torch.equal(on.cpu(), new)
        assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])
