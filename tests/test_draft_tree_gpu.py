"""Draft trees over paged caches against the float64 oracle: attention, acceptance, and the rows that are kept.

Bounds of the attention are those of the windowed paged attention (tests/test_window_attention_gpu.py), whose kernels it runs: with u
half a step of q's type, o is off by at most 2u a (a = sum w |v|: the rounded weights, normalised by their sum) and u |o|; a score
by e = (D + 16) 2^-24 big + 2^-19 (big = the largest sum |q k| |scale| of the row), which moves weights by exp(+-2e); sums over n
keys add n 2^-24 a. The lse is off by e, n 2^-24 and two steps of itself. Second orders: a factor of 1.05. In fp16 a weight below
2^-14 (relative to an offset that is at most the row's largest score, so that the weights' sum is at least 1) is rounded by up to
2^-25 and not by u of itself: it moves the sum of w v by up to 2^-25 |v| and, by the normalising sum, again as much at most: 2^-24 sum |v|
in all. (With scores 50 apart, as under a scale of 3, most weights are that small.) Acceptance and moved rows are whole numbers and
bytes: equal.
"""
import math
import threading

import pytest
import torch

from lightserve_amd.kernels.beam_search import kv_cache_reorder
from lightserve_amd.kernels.draft_tree import accept_drafts, draft_tree, kv_cache_keep, paged_tree_attention
from lightserve_amd.kernels.paged_attention import paged_prefill
from oracle import candidates, paged8
from tests.candidate_cases import E4M3, forest, layer_caches, on_gpu, raw
from tests.paged8_cases import cache8, offsets, tables

pytestmark = pytest.mark.gpu
KINDS = [("e4m3", torch.bfloat16), ("e4m3", torch.float16), ("16 bit", torch.bfloat16), ("16 bit", torch.float16)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _cache(kind, dtype, pool, bs, hkv, d, seed):
    if kind == "e4m3":
        kc, vc, sc = cache8(pool, bs, hkv, d, seed)
        return (kc.cuda().view(E4M3), vc.cuda().view(E4M3), sc.cuda()), paged8.cache_values(kc, vc, sc)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(pool, bs, hkv, d, generator=g).to(dtype) for _ in range(2))
    return (k.cuda(), v.cuda(), None), (k.double(), v.double())


def _assert_close(got, lse, ref, n, what):
    o, want_lse, a, big, plain = ref
    got, lse = got.cpu(), lse.cpu().double()
    u, d = torch.finfo(got.dtype).eps / 2, got.shape[-1]
    e = (d + 16) * 2.0 ** -24 * big + 2.0 ** -19
    tol = 1.05 * ((2 * u + 2 * e[..., None] + n * 2.0 ** -24) * a + u * o.abs()) + 2.0 ** -24
    if got.dtype == torch.float16:
        tol += 2 * 2.0 ** -25 * plain
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = ((got.double() - o).abs() / tol).max().item() if o.numel() else 0.0
    none = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, none), f"{what}: rows that see nothing"
    lse_tol = e + n * 2.0 ** -24 + want_lse.abs() * 2.0 ** -22
    off = ((lse - want_lse).abs() / lse_tol)[~none]
    print(f"[bound] {what}: o {worst:.2f}, lse {off.max().item() if off.numel() else 0:.2f}", flush=True)
    assert worst <= 1, f"{what}: {worst:.2f} of the bound"
    assert off.numel() == 0 or off.max() <= 1, f"{what}: lse {off.max():.2f} of the bound"


def _attend(kind, dtype, nodes, had, hq, hkv, d, bs, seed, window=None, sinks=0, sm_scale=None, mask=None, words=None, what=""):
    lens = [a + b for a, b in zip(nodes, had)]
    table, pool = tables(lens, bs, seed)
    cache, vals = _cache(kind, dtype, pool, bs, hkv, d, seed + 1)
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(seed + 2)).to(dtype)
    _, tree, cu = forest(nodes, seed + 3, words)
    tree = tree if mask is None else mask
    o, lse = paged_tree_attention(q.cuda(), *cache[:2], table.cuda(), cu.cuda(), _i32(lens).cuda(), tree.cuda(), sm_scale=sm_scale,
                                  return_lse=True, kv_scales=cache[2], window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert lse.shape == (hq, sum(nodes))
    ref = candidates.tree_reference(q, *vals, table, cu, lens, tree, window, sinks, sm_scale)
    _assert_close(o, lse.t(), ref, max(lens + [1]), what)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (32, 8, 128), (14, 2, 64), (6, 2, 80), (20, 1, 128), (3, 3, 16)])
def test_tree_heads(gpu, kind, dtype, hq, hkv, d):
    """Groups of 1 to 20 heads, with few and many nodes: every kernel instance; drafts that begin inside tiles and blocks."""
    print(f"case tree {kind} {dtype} hq={hq} hkv={hkv} d={d}", flush=True)
    _attend(kind, dtype, [1, 2, 0, 4], [0, 31, 5, 100], hq, hkv, d, 16, hq + d, what="few")
    _attend(kind, dtype, [1, 16, 0, 33, 7], [300, 1, 40, 64, 0], hq, hkv, d, 16, hq + d + 1, what="many")
    _attend(kind, dtype, [12, 3], [333, 90], hq, hkv, d, 32, hq + d + 2, 20, 3, what="window")


@pytest.mark.parametrize("base", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100])
def test_tree_begins_anywhere(gpu, base):
    """The drafts' first key against the tiles' edges, with masks of one to four words."""
    print(f"case tree base={base}", flush=True)
    for n in (1, 5, 31, 32, 33, 64, 65, 129, 256):
        _attend("16 bit", torch.bfloat16, [n], [base], 2, 2, 64, 16, n + base, what=f"n={n}")
    _attend("e4m3", torch.bfloat16, [40, 70], [base, base + 7], 8, 1, 64, 16, base, what="rows of several waves")


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (17, 0), (33, 16), (100, 33), (5000, 0), (64, 5000)])
def test_tree_windows(gpu, window, sinks):
    """A window counts from each node's own depth; drafts stay visible whatever it is."""
    print(f"case tree window={window} sinks={sinks}", flush=True)
    _attend("e4m3", torch.bfloat16, [3, 8, 20, 1], [0, 40, 130, 500], 8, 2, 64, 16, 5, window, sinks, what="narrow")
    _attend("16 bit", torch.float16, [70, 20, 0, 100], [10, 140, 30, 500], 8, 2, 64, 32, 6, window, sinks, what="wide")


@pytest.mark.parametrize("lens", [[9000], [4096, 1, 3000], [12000, 700, 0, 5]])
@pytest.mark.parametrize("n", [4, 16, 60])
def test_tree_long(gpu, lens, n):
    """Sequences that several workgroups share."""
    print(f"case tree long {lens} n={n}", flush=True)
    _attend("e4m3", torch.bfloat16, [n] * len(lens), lens, 8, 1, 128, 16, 11, what="8 bits")
    _attend("16 bit", torch.float16, [max(0, n - 5 * i) for i in range(len(lens))], lens, 4, 2, 64, 16, 12, 3000, 4, what="window")


@pytest.mark.parametrize("batch", [63, 64, 65, 130])
def test_tree_many_sequences(gpu, batch):
    print(f"case tree batch={batch}", flush=True)
    had = [(37 * b * b) % 200 for b in range(batch)]
    _attend("16 bit", torch.bfloat16, [(b * 7) % 9 for b in range(batch)], had, 4, 2, 64, 16, batch, what="few nodes")
    _attend("e4m3", torch.float16, [(b * 7) % 40 for b in range(batch)], had, 4, 2, 64, 16, batch, what="many nodes")


def test_tree_any_mask(gpu):
    """Masks that are no tree's: nothing at all, everything, later nodes, bits past the nodes (not read)."""
    print("case tree masks", flush=True)
    g = torch.Generator().manual_seed(3)
    nodes, had = [9, 40, 3], [0, 70, 20]
    mask = torch.randint(-2 ** 62, 2 ** 62, (sum(nodes), 1), generator=g)
    mask[0], mask[1], mask[20] = 0, -1, 0
    for kind, dtype in KINDS:
        _attend(kind, dtype, nodes, had, 4, 2, 64, 16, 21, mask=mask, what="any")
        _attend(kind, dtype, nodes, had, 4, 2, 64, 16, 22, 30, 2, mask=mask, what="any, window")
    wide = torch.randint(-2 ** 62, 2 ** 62, (sum(nodes), 4), generator=g)
    _attend("16 bit", torch.bfloat16, nodes, had, 12, 2, 64, 16, 23, mask=wide, words=4, what="wider than needed")


def test_tree_of_more_nodes_than_keys(gpu):
    """Lengths below the number of nodes: the first nodes' own keys lie before the sequence, and nobody sees them."""
    print("case tree lengths below nodes", flush=True)
    for kind, dtype in KINDS:
        _attend(kind, dtype, [9, 12, 3, 2], [-4, -11, -3, 5], 4, 2, 64, 16, 31, what="few rows")
        _attend(kind, dtype, [40, 100, 70], [-7, -99, -70], 8, 2, 64, 16, 32, what="many rows")
        _attend(kind, dtype, [40, 100, 70], [-7, -99, 3], 8, 2, 64, 16, 33, 5, 2, what="window")


@pytest.mark.parametrize("kind", ["e4m3", "16 bit"])
@pytest.mark.parametrize("n", [3, 40])
def test_tree_far_blocks(gpu, kind, n):
    """Blocks whose offsets in the cache, in elements, pass 32 bits give what the same rows give near its beginning; and so do
    rows moved there."""
    print(f"case tree far {kind} n={n}", flush=True)
    nodes, had, hkv, d, bs = [n, n + 2], [50, 200], 2, 128, 16
    lens = [a + b for a, b in zip(nodes, had)]
    table, pool = tables(lens, bs, 3)
    (k, v, sc), _ = _cache(kind, torch.bfloat16, pool, bs, hkv, d, 4)
    blocks = 2 ** 32 // (bs * hkv * d) + pool + 5
    far = blocks - pool
    big = [torch.empty(blocks, *c.shape[1:], dtype=torch.uint8, device="cuda").view(c.dtype) if c.dtype == E4M3 else
           torch.empty(blocks, *c.shape[1:], dtype=c.dtype, device="cuda") for c in (k, v)]
    for c, small in zip(big, (k, v)):
        raw_bytes = c.view(torch.uint8) if c.dtype == E4M3 else c
        raw_bytes[far:] = small.view(torch.uint8) if c.dtype == E4M3 else small
    scales = None
    if sc is not None:
        scales = torch.zeros(blocks, hkv, bs, 2, dtype=torch.uint8, device="cuda")
        scales[far:] = sc
    q = torch.randn(sum(nodes), 8, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    _, mask, cu = forest(nodes, 6)
    near_table, far_table = table.cuda(), torch.where(table >= 0, table + far, -1).cuda()
    rest = (cu.cuda(), _i32(lens).cuda(), mask.cuda())
    a = paged_tree_attention(q, k, v, near_table, *rest, kv_scales=sc)
    b = paged_tree_attention(q, *big, far_table, *rest, kv_scales=scales)
    assert torch.equal(a, b)
    keep, counts = _i32([[0, 2, -1], [1, 4, 4]]).cuda(), _i32([2, 3]).cuda()
    kept = _i32([h + c for h, c in zip(had, [2, 3])]).cuda()
    kv_cache_keep(k, v, near_table, kept, keep, counts, kv_scales=sc)
    kv_cache_keep(*big, far_table, kept, keep, counts, kv_scales=scales)
    parents, two = _i32([[1, 0]]).cuda(), _i32([60, 60]).cuda()
    kv_cache_reorder(k, v, near_table, two, parents, kv_scales=sc)
    kv_cache_reorder(*big, far_table, two, parents, kv_scales=scales)
    torch.cuda.synchronize()
    assert torch.equal(torch.where(near_table >= 0, near_table + far, -1), far_table)
    for c, small in zip(big, (k, v)):
        assert torch.equal(raw(c[far:].contiguous()), raw(small))
    assert sc is None or torch.equal(scales[far:], sc)


@pytest.mark.parametrize("sm_scale", [0.0, -0.2, 3.0])
def test_tree_scales(gpu, sm_scale):
    print(f"case tree scale={sm_scale}", flush=True)
    _attend("16 bit", torch.bfloat16, [5, 50], [40, 90], 4, 2, 64, 16, 31, sm_scale=sm_scale, what="scale")
    _attend("e4m3", torch.float16, [5, 50], [40, 90], 4, 2, 64, 16, 32, sm_scale=sm_scale, what="scale")


def test_tree_of_a_chain_is_a_chunk(gpu):
    """A chain's mask is the causal one: the same as paged_prefill, window and all."""
    print("case tree chain", flush=True)
    n, had = [7, 60], [100, 333]
    lens = [a + b for a, b in zip(n, had)]
    table, pool = tables(lens, 16, 1)
    cache, _ = _cache("e4m3", torch.bfloat16, pool, 16, 2, 128, 2)
    q = torch.randn(sum(n), 8, 128, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    mask = torch.cat([draft_tree(range(-1, m - 1))[0] for m in n]).cuda()
    at = (table.cuda(), offsets(n).cuda(), _i32(lens).cuda())
    for window, sinks in ((None, 0), (90, 4)):
        a = paged_tree_attention(q, *cache[:2], *at, mask, kv_scales=cache[2], window=window, sinks=sinks)
        b = paged_prefill(q, *cache[:2], *at, kv_scales=cache[2], window=window, sinks=sinks)
        # (one rounding of bf16 apart: the two may sum in another order)
        assert (a.double() - b.double()).abs().max() <= 2.0 ** -8 * b.double().abs().max()


@pytest.mark.parametrize("kind", ["e4m3", "16 bit"])
@pytest.mark.parametrize("n", [6, 50])
def test_tree_values_not_finite(gpu, kind, n):
    """Infinities and NaN of a draft's K and V, and of a key under the window, reach only the nodes that see it."""
    print(f"case tree not finite {kind} n={n}", flush=True)
    hq, hkv, d, bs, had = 4, 2, 64, 16, 75
    lens = [had + n]
    table, pool = tables(lens, bs, 1)
    parents, mask, cu = forest([n], 3)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(n, hq, d, generator=g).bfloat16()
    bad = {"none": [], "draft": [had + 2, had + n - 1], "window": [3, 40]}
    outs = {}
    # Both are within 3u times the largest |v| of the exact (rounded weights and output; sums may be taken in another order).
    bound = 2 * 1.05 * 3 * 2.0 ** -8 * _cache(kind, torch.bfloat16, pool, bs, hkv, d, 5)[1][1].abs().max()
    for name, rows in bad.items():
        (kc, vc, sc), _ = _cache(kind, torch.bfloat16, pool, bs, hkv, d, 5)
        for r in rows:
            for c in (kc, vc):
                block, slot = int(table[0, r // bs]), r % bs
                if kind == "e4m3":
                    c.view(torch.uint8)[block, slot, 0, 5:9] = 127
                else:
                    c[block, slot, 0, 5], c[block, slot, 0, 7] = math.nan, math.inf
        outs[name] = paged_tree_attention(q.cuda(), kc, vc, table.cuda(), cu.cuda(), _i32(lens).cuda(), mask.cuda(), kv_scales=sc,
                                          window=20, sinks=2).cpu()
    for name, rows in bad.items():
        for i in range(n):
            m = candidates.bits_of(mask[i])
            pos = had + bin(m).count("1") - 1
            sees = any((r >= had and m >> (r - had) & 1) or (r < had and (r > pos - 20 or r < 2)) for r in rows)
            group = slice(0, hq // hkv)
            if sees:
                assert not torch.isfinite(outs[name][i, group]).all(), f"{name}: node {i} sees it"
            else:
                off = (outs[name][i, group].double() - outs["none"][i, group].double()).abs().max()
                assert off <= bound, f"{name}: node {i} does not see it"
            assert torch.equal(outs[name][i, hq // hkv:], outs["none"][i, hq // hkv:]), "another KV head"


def test_tree_strides_and_blocks_outside(gpu):
    """Strided q, caches, tables and masks, rows behind the last sequence, table entries outside the cache."""
    print("case tree strides", flush=True)
    nodes, had = [5, 20], [40, 100]
    lens = [a + b for a, b in zip(nodes, had)]
    table, pool = tables(lens, 16, 1)
    table[1, 2] = pool + 5
    g = torch.Generator().manual_seed(2)
    both = torch.randn(pool, 16, 2, 2, 64, generator=g).bfloat16()
    k, v = both.unbind(3)
    q = torch.randn(4, 30, 64, generator=g).bfloat16().transpose(0, 1)
    _, mask, cu = forest(nodes, 3)
    padded = torch.zeros(30, 3, dtype=torch.int64)
    padded[:25, 1:2] = mask
    wide = torch.full((2, 40), -1, dtype=torch.int32)
    wide[:, ::2][:, :table.shape[1]] = table
    dev = both.cuda()
    o, lse = paged_tree_attention(q.cuda(), *dev.unbind(3), wide.cuda()[:, ::2], cu.cuda(), _i32(lens).cuda(), padded.cuda()[:, 1:2],
                                  max_nodes=20, return_lse=True)
    ref = candidates.tree_reference(q[:25], k.double(), v.double(), table, cu, lens, mask)
    _assert_close(o[:25], lse.t()[:25], ref, max(lens), "strides")


def test_tree_refusals(gpu):
    """What is only found once the tensors are on a GPU."""
    print("case tree refusals", flush=True)
    table, pool = tables([20], 16, 1)
    (kc, vc, _), _ = _cache("16 bit", torch.bfloat16, pool, 16, 2, 64, 2)
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16).cuda()
    at = (table.cuda(), _i32([0, 4]).cuda(), _i32([20]).cuda())
    mask = torch.ones(4, 1, dtype=torch.int64).cuda()
    for kw in (dict(window=0), dict(sinks=2), dict(window=5, sinks=-1)):
        with pytest.raises(AssertionError):
            paged_tree_attention(q, kc, vc, *at, mask, **kw)
    with pytest.raises(AssertionError):
        paged_tree_attention(q, kc, vc, *at, mask.cpu())
    with pytest.raises(RuntimeError, match="lsfa_tree"):
        paged_tree_attention(q, kc.view(-1, 8, 2, 64), vc.view(-1, 8, 2, 64), *at, mask)


def test_tree_streams_and_graphs(gpu):
    """Calls on two streams at once, and replays of a captured one with eager calls between them."""
    print("case tree graphs", flush=True)
    nodes, had = [16, 40], [3000, 700]
    lens = [a + b for a, b in zip(nodes, had)]
    table, pool = tables(lens, 16, 1)
    cache, _ = _cache("16 bit", torch.bfloat16, pool, 16, 2, 128, 2)
    _, mask, cu = forest(nodes, 3)
    at = (table.cuda(), cu.cuda(), _i32(lens).cuda(), mask.cuda())
    qs = [torch.randn(sum(nodes), 8, 128, generator=torch.Generator().manual_seed(s)).bfloat16().cuda() for s in range(4)]
    want = [paged_tree_attention(q, *cache[:2], *at, max_nodes=40) for q in qs]
    torch.cuda.synchronize()
    got = [None] * 4
    streams = [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i] = paged_tree_attention(qs[i], *cache[:2], *at, max_nodes=40)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads], [t.join() for t in threads]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = qs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_tree_attention(static, *cache[:2], *at, max_nodes=40)
    for i in (1, 2, 3, 0):
        static.copy_(qs[i])
        graph.replay()
        assert torch.equal(paged_tree_attention(qs[3 - i], *cache[:2], *at, max_nodes=40), want[3 - i])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), f"replay {i}"


# ------------------------------------------------------------------ accept
def _drafts(nodes, vocab, dtype, seed, right=0.7, ties=False):
    """Logits and tokens of trees whose nodes are the greedy choice after their parents more often than not."""
    g = torch.Generator().manual_seed(seed)
    parents, mask, cu = forest(nodes, seed)
    x = torch.randn(sum(nodes), vocab, generator=g)
    logits = (torch.round(x) if ties else x * 2.5).to(dtype)
    tokens = torch.randint(0, vocab, (sum(nodes),), generator=g)
    for b, p in enumerate(parents):
        for i, parent in enumerate(p):
            if i and torch.rand((), generator=g) < right:
                tokens[int(cu[b]) + i] = candidates.first_largest(logits[int(cu[b]) + parent].double())
    return logits, tokens, mask, cu


def _accept(logits, tokens, mask, cu, what, max_nodes=None, seq_lens=True, dev=None):
    most = max([int(b - a) for a, b in zip(cu[:-1], cu[1:])] + [0]) if max_nodes is None else max_nodes
    lens = torch.arange(100, 100 + len(cu) - 1, dtype=torch.int32)
    on = lens.cuda() if seq_lens else None
    path, counts, following = accept_drafts(logits.cuda() if dev is None else dev, tokens.cuda(), mask.cuda(), cu.cuda(),
                                            max_nodes=max_nodes, seq_lens=on)
    want = candidates.accept_reference(logits, tokens, mask, cu, most)
    assert path.tolist() == want[0] and counts.tolist() == want[1] and following.tolist() == want[2], what
    if seq_lens:
        assert torch.equal(on.cpu(), lens + _i32(want[1]).view(-1)), what
    return want[1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 7, 1000, 4099, 32000])
def test_accept(gpu, dtype, vocab):
    print(f"case accept {dtype} {vocab}", flush=True)
    for nodes in ([1], [8], [0, 5, 0, 1, 33, 2]):
        counts = _accept(*_drafts(nodes, vocab, dtype, vocab + len(nodes)), f"{nodes}")
    assert max(counts) > 1
    _accept(*_drafts([9, 4], vocab, dtype, 5, ties=True), "ties", seq_lens=False)


@pytest.mark.parametrize("n", [63, 64, 65, 130, 256])
def test_accept_large_trees(gpu, n):
    print(f"case accept n={n}", flush=True)
    logits, tokens, mask, cu = _drafts([n, 3, n - 1], 300, torch.bfloat16, n, right=0.97)
    counts = _accept(logits, tokens, mask, cu, "large")
    assert max(counts) > 1  # (of the oracle; the chain below makes long paths)
    chain = draft_tree(range(-1, n - 1))[0]
    choice = [candidates.first_largest(r.double()) for r in logits[:n]]
    _accept(logits[:n], torch.tensor([0] + choice[:-1]), chain, _i32([0, n]), "a chain that is all right")


def test_accept_many_sequences(gpu):
    print("case accept batch", flush=True)
    _accept(*_drafts([(3 * b) % 5 for b in range(200)], 500, torch.float16, 1), "200 sequences")


def test_accept_special_values(gpu):
    """NaN beats every number, equal ones go to the first, -inf rows name token 0; two children of one token: the lower."""
    print("case accept special", flush=True)
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.full((6, 5000), -math.inf, dtype=dtype)
        logits[0, 4999], logits[0, 17], logits[0, 18] = math.inf, math.nan, math.nan
        logits[1, 40] = logits[1, 4000] = 3.0
        logits[2, 5], logits[2, 6] = -0.0, 0.0
        logits[4] = 1.0
        mask = draft_tree([-1, 0, 0, 1, 1, 3])[0]
        _accept(logits, torch.tensor([9, 17, 17, 40, 40, 0]), mask, _i32([0, 6]), "special")
        _accept(logits, torch.tensor([9, 1, 17, 5, 4, 5]), draft_tree([-1, 0, 0, 2, 2, 2])[0], _i32([0, 6]), "signed zeros")


def test_accept_layouts(gpu):
    """Rows at odd addresses and strides, rows behind the last sequence, fewer max_nodes than nodes."""
    print("case accept layouts", flush=True)
    for dtype in (torch.float32, torch.float16):
        logits, tokens, mask, cu = _drafts([4, 9], 2051, dtype, 3)
        wide = torch.full((15, 2100), 50.0, dtype=dtype)
        for shift in (0, 1, 3, 7):
            wide.fill_(50.0)
            wide[:13, shift:shift + 2051] = logits
            on = wide.cuda()[:, shift:shift + 2051]
            more = torch.cat([tokens, torch.zeros(2, dtype=torch.int64)])
            _accept(on.cpu(), more, torch.cat([mask, mask[:2]]), cu, f"shift {shift}", dev=on)
        _accept(logits, tokens, mask, cu, "max_nodes", max_nodes=4)
        turned = logits.t().contiguous().cuda().t()
        _accept(logits, tokens, mask, cu, "column-major", dev=turned)


def test_accept_graph(gpu):
    print("case accept graph", flush=True)
    logits, tokens, mask, cu = _drafts([8, 0, 20], 30000, torch.bfloat16, 3)
    dev, lens = logits.cuda(), torch.zeros(3, dtype=torch.int32, device="cuda")
    rest = tokens.cuda(), mask.cuda(), cu.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = accept_drafts(dev, *rest, max_nodes=20, seq_lens=lens)
    for i in range(4):
        turned = logits.roll(i * 7, 1)
        dev.copy_(turned)
        lens.zero_()
        graph.replay()
        accept_drafts(dev, *rest, max_nodes=20)
        torch.cuda.synchronize()
        want = candidates.accept_reference(turned, tokens, mask, cu, 20)
        assert [t.tolist() for t in out] == list(want) and lens.tolist() == want[1]


# -------------------------------------------------------------------- keep
def _keep(kind, keep, counts, lens, rows, bs, heads, d, seed, layers=2, what=""):
    table, pool = tables(rows, bs, seed)
    k, v, scales = layer_caches(kind, layers, pool, bs, heads, d, seed)
    dev = on_gpu(kind, k, v, scales)
    kv_cache_keep(dev[0], dev[1], table.cuda(), _i32(lens).cuda(), keep.cuda(), _i32(counts).cuda(), kv_scales=dev[2])
    torch.cuda.synchronize()
    want = candidates.keep_reference([c for c in (k, v, scales) if c is not None], table, lens, keep, counts, (1, 1, 2))
    for got, w in zip((c for c in dev if c is not None), want):
        assert torch.equal(raw(got), raw(w)), what


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32, E4M3])
@pytest.mark.parametrize("heads,d", [(1, 16), (8, 128), (3, 80), (2, 256)])
def test_keep(gpu, kind, heads, d):
    print(f"case keep {kind} {heads} {d}", flush=True)
    keep = torch.full((4, 9), -1, dtype=torch.int32)
    keep[0, :4], keep[1, :2], keep[2, :9] = _i32([0, 3, 4, 30]), _i32([5, 6]), _i32([0, 1, 2, 4, 5, 9, 10, 11, 39])
    _keep(kind, keep, [4, 2, 9, 0], [104, 2, 24, 7], [140, 9, 60, 8], 16, heads, d, 1, what="paths")


@pytest.mark.parametrize("kind", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("n,kept", [(33, 33), (65, 40), (700, 350), (700, 699), (2000, 64)])
def test_keep_many(gpu, kind, n, kept):
    """Widths above 32: dense and sparse ones, entries at most their own place among them."""
    print(f"case keep n={n} kept={kept}", flush=True)
    g = torch.Generator().manual_seed(n)
    keep = torch.stack([torch.randperm(n, generator=g)[:kept].sort().values for _ in range(2)]).int()
    keep[1, 5:9] = _i32([5, 0, -3, 8])
    _keep(kind, keep, [kept, kept - 3], [kept + 50, kept], [n + 60, n + 5], 32, 2, 64, 3, what="many")
    double = (torch.arange(kept, dtype=torch.int32) // 2 * 2 + 3).repeat(2, 1)
    _keep(kind, double, [kept, 10], [kept, 10], [kept + 5, 20], 16, 2, 64, 4, what="the same row twice")


def test_keep_wide_launches(gpu):
    """Many layers (a wave by itself goes through long lists), and few (16 waves together, at both widths of columns)."""
    print("case keep launches", flush=True)
    g = torch.Generator().manual_seed(2)
    for layers, sequences, n, kept in ((300, 2, 90, 60), (2, 1, 90, 60), (1, 2, 1200, 600), (2, 1, 600, 513)):
        keep = torch.stack([torch.randperm(n, generator=g)[:kept].sort().values for _ in range(sequences)]).int()
        _keep(torch.bfloat16, keep, [kept] * sequences, [kept + 5] * sequences, [n + 9] * sequences, 16, 2, 64, 7, layers=layers,
              what=f"{layers} layers, {kept} of {n}")


def test_keep_outside(gpu):
    """Rows that the table, the cache or the sequence does not have are not moved; counts past the width are held to it."""
    print("case keep outside", flush=True)
    keep = _i32([[2, 3, 1000, 2 ** 31 - 1], [7, 8, 9, 40]])
    _keep(torch.bfloat16, keep, [4, 4], [14, 4], [20, 16], 16, 2, 64, 5, what="past the table")
    _keep(torch.bfloat16, keep, [4, 4], [-100, 2], [20, 16], 16, 2, 64, 6, what="before the sequence")


def test_keep_one_layer_and_strides(gpu):
    """One layer's caches, as views of a pool that holds K beside V."""
    print("case keep layouts", flush=True)
    g = torch.Generator().manual_seed(1)
    table, pool = tables([40], 16, 2)
    both = torch.randn(pool, 16, 2, 2, 64, generator=g).half()
    dev = both.cuda()
    keep, counts, lens = _i32([[0, 5, 9]]), [3], [23]
    kv_cache_keep(dev[:, :, :, 0], dev[:, :, :, 1], table.cuda(), _i32(lens).cuda(), keep.cuda(), _i32(counts).cuda())
    want = candidates.keep_reference([both[None, :, :, :, 0], both[None, :, :, :, 1]], table, lens, keep, counts, (1, 1))
    assert torch.equal(dev[:, :, :, 0].cpu(), want[0][0]) and torch.equal(dev[:, :, :, 1].cpu(), want[1][0])


def test_a_step_together(gpu):
    """Attention, acceptance and the move, captured as one graph and replayed: afterwards the cache holds the path's rows as
    if its tokens had been decoded one by one."""
    print("case step", flush=True)
    nodes, had, hkv, d, bs = [6, 11, 1], [30, 100, 16], 2, 64, 16
    lens = [a + b for a, b in zip(nodes, had)]
    table, pool = tables(lens, bs, 1)
    k, v, _ = layer_caches(torch.bfloat16, 3, pool, bs, hkv, d, 2)
    logits, tokens, mask, cu = _drafts(nodes, 900, torch.bfloat16, 7, right=0.9)
    kd, vd, start = k.cuda(), v.cuda(), _i32(had).cuda()
    at, seq = (table.cuda(), cu.cuda()), start.clone()
    q = torch.randn(sum(nodes), 4, d, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    lg, tk, mk = logits.cuda(), tokens.cuda(), mask.cuda()
    n_dev = _i32(nodes).cuda()

    def step():
        o = paged_tree_attention(q, kd[0], vd[0], *at, seq + n_dev, mk, max_nodes=11)
        path, counts, following = accept_drafts(lg, tk, mk, at[1], max_nodes=11, seq_lens=seq)
        kv_cache_keep(kd, vd, at[0], seq, path, counts)
        return o, path, counts, following
    want_o = step()[0].clone()
    paths, counts, following = candidates.accept_reference(logits, tokens, mask, cu, 11)
    final = [a + c for a, c in zip(had, counts)]
    want = candidates.keep_reference([k, v], table, final, _i32(paths), counts, (1, 1))
    assert max(counts) > 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        kd.copy_(k), vd.copy_(v), seq.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want_o) and out[1].tolist() == paths and out[3].tolist() == following
        assert seq.tolist() == final and torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])
