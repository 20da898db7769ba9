"""Decoding with several candidates per sequence over a paged KV cache, as cases that a measuring program can time and compare.

Five operators, each reached through a public entry point. Two candidates' forms: a tree of drafted tokens that one step
verifies, and beams.

  tree     paged_tree_attention: the drafted tokens of each sequence against its cached ones and their own ancestors
  accept   accept_drafts: the path of a tree whose tokens are the model's own choices, and the token that follows it
  keep     kv_cache_keep: the accepted rows of the caches moved up to where the next step expects them, in all layers
  select   beam_search_select: the best continuations over a sequence's beams and the vocabulary
  reorder  kv_cache_reorder: the beams' caches after their parents', in all layers

A tree's node i has a mask of 64-bit words, bit j of which says that it sees node j (its ancestors and itself); node 0 is the last
token that is certain, whose K and V are cached with the drafts'. A sequence's drafts are the last of its cached tokens.

listed() names twelve cases; draw() gives others of the same ranges. Sizes are those of this repository's workloads
(lightserve_amd/workloads.py, model/minimal_llama.py) and tests, or generic ones. Lengths are spread evenly from the shortest
to the longest, so that a case's work is known without its inputs.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One request's step with a small tree of drafts at LLaMA-3-8B's layer shape: latency.
        dict(name="tree_single_bf16", op="tree", dtype="bf16", cache="16 bit", sequences=1, nodes_shortest=8, nodes_longest=8,
             shortest=1500, longest=1500, heads=32, kv_heads=8, dim=128, block=16, window=0, sinks=0, lse=False),
        # A batch of requests, 16 drafts or fewer each.
        dict(name="tree_batch_bf16", op="tree", dtype="bf16", cache="16 bit", sequences=16, nodes_shortest=5, nodes_longest=16,
             shortest=512, longest=8192, heads=32, kv_heads=8, dim=128, block=16, window=0, sinks=0, lse=False),
        # Large trees over an 8-bit cache.
        dict(name="tree_large_8bit_bf16", op="tree", dtype="bf16", cache="e4m3", sequences=16, nodes_shortest=64, nodes_longest=64,
             shortest=1024, longest=8192, heads=32, kv_heads=8, dim=128, block=16, window=0, sinks=0, lse=False),
        # Ragged trees of more than 64 nodes under a window, heads in groups of seven, one sequence with no draft at all.
        dict(name="tree_window_odd_fp16", op="tree", dtype="fp16", cache="16 bit", sequences=5, nodes_shortest=0, nodes_longest=77,
             shortest=333, longest=6001, heads=14, kv_heads=2, dim=64, block=32, window=1000, sinks=4, lse=True),
        # The choice after one request's eight nodes.
        dict(name="accept_single_bf16", op="accept", dtype="bf16", sequences=1, nodes_shortest=8, nodes_longest=8, vocab=128256),
        # A batch of large trees.
        dict(name="accept_batch_bf16", op="accept", dtype="bf16", sequences=16, nodes_shortest=5, nodes_longest=64, vocab=128256),
        # What a batch of requests accepted, moved in every layer of a model.
        dict(name="keep_path_bf16", op="keep", cache="bf16", layers=32, sequences=16, nodes_shortest=16, nodes_longest=64,
             kept_percent=8, cached=1500, kv_heads=8, dim=128, block=16),
        # Half the rows of long 8-bit prefixes given up, odd sizes.
        dict(name="keep_half_8bit", op="keep", cache="e4m3", layers=4, sequences=7, nodes_shortest=2500, nodes_longest=4001,
             kept_percent=50, cached=0, kv_heads=8, dim=128, block=16),
        # Four beams of one request.
        dict(name="select_single_bf16", op="select", dtype="bf16", sequences=1, beams=4, number=8, vocab=128256),
        # Eight beams of a batch, logits in 32 bits, an odd vocabulary.
        dict(name="select_batch_fp32", op="select", dtype="fp32", sequences=32, beams=8, number=16, vocab=50257),
        # Four beams of one request take over their parents' last rows.
        dict(name="reorder_single_bf16", op="reorder", cache="bf16", layers=32, sequences=1, beams=4, shortest=1511, longest=1511,
             kv_heads=8, dim=128, block=16),
        # Eight beams of a batch with large blocks.
        dict(name="reorder_batch_8bit", op="reorder", cache="e4m3", layers=32, sequences=16, beams=8, shortest=500, longest=2046,
             kv_heads=8, dim=128, block=64),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "accept", "keep", "select", "reorder"])
    c = dict(op=op)
    if op in ("accept", "select"):
        c |= dict(dtype=rng.choice(["bf16", "fp16", "fp32"]), sequences=_spread(rng, 1, 48), vocab=_spread(rng, 33, 152000))
        most = max(1, 130_000_000 // (c["sequences"] * c["vocab"] * 2))
        if op == "accept":
            c["nodes_longest"] = _spread(rng, 1, min(256, most))
            return c | dict(nodes_shortest=rng.randint(0, c["nodes_longest"]))
        c["beams"] = _spread(rng, 1, min(32, most))
        return c | dict(number=rng.randint(1, min(64, 2 * c["beams"])))
    c |= dict(kv_heads=rng.choice([1, 2, 3, 8, 16]), dim=rng.choice([64, 80, 96, 112, 128]), block=rng.choice([16, 32, 64]))
    row = c["kv_heads"] * c["dim"]
    if op == "tree":
        c |= dict(dtype=rng.choice(["bf16", "fp16"]), cache=rng.choice(["e4m3", "16 bit"]), sequences=_spread(rng, 1, 48))
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 7, 8])
        c |= dict(window=_spread(rng, 64, 4096), sinks=rng.choice([0, 1, 4, rng.randint(5, 70)])) if rng.random() < 0.4 \
            else dict(window=0, sinks=0)
        c["lse"] = rng.random() < 0.5
        c["nodes_longest"] = _spread(rng, 1, 256)
        c["nodes_shortest"] = rng.randint(0, c["nodes_longest"])
        most = min(120_000_000 // (c["sequences"] * row), 250_000_000 // (c["sequences"] * c["heads"] * c["nodes_longest"]))
        c["longest"] = _spread(rng, 1, max(64, min(32768, most)))
        return c | dict(shortest=rng.randint(0, c["longest"]))
    c |= dict(cache=rng.choice(["e4m3", "bf16", "fp16"]), layers=_spread(rng, 1, 40), sequences=_spread(rng, 1, 24))
    most = 200_000_000 // (c["sequences"] * c["layers"] * row)
    if op == "keep":
        c["nodes_longest"] = _spread(rng, 1, max(1, min(4096, most)))
        return c | dict(nodes_shortest=rng.randint(0, c["nodes_longest"]), kept_percent=rng.randint(1, 100),
                        cached=rng.choice([0, rng.randint(1, 200)]))
    c["beams"] = _spread(rng, 1, min(32, max(1, most // 200)))
    c["longest"] = _spread(rng, 1, max(70, min(8192, (most - c["beams"] * c["block"]) // 2)))
    return c | dict(shortest=rng.randint(0, c["longest"]))


# ------------------------------------------------------------------ sizes
def _lengths(shortest, longest, n):
    return [longest if n == 1 else shortest + (longest - shortest) * i // (n - 1) for i in range(n)]


def _nodes(case):
    return _lengths(case["nodes_shortest"], case["nodes_longest"], case["sequences"])


def _cached(case):
    """Tokens cached ahead of the drafts, the longest of the batch beside its smallest tree."""
    return _lengths(case["shortest"], case["longest"], case["sequences"])[::-1]


def _kept(case):
    """Rows that stay of a sequence's n: the first, and others that all move."""
    return [max(1, min(n - 1, n * case["kept_percent"] // 100)) if n > 1 else n for n in _nodes(case)]


def _row_bytes(case):
    """K and V of one token in one layer."""
    return case["kv_heads"] * (2 * case["dim"] + 2 if case["cache"] == "e4m3" else 4 * case["dim"])


def work(case):
    if case["op"] == "tree":
        size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        w, s = case["window"], case["sinks"]
        keys = pairs = 0
        for n, base in zip(_nodes(case), _cached(case)):
            # (a tree of n nodes is about log n deep: its ancestors are few beside the cached tokens)
            seen = base if not w or w > base else w - 1 + min(s, base - w + 1)
            keys += seen + n if n else 0
            pairs += n * (seen + 1 + int(math.log2(n))) if n else 0
        rows = sum(_nodes(case)) * case["heads"]
        return {"bytes": keys * _row_bytes(case) + 2 * rows * case["dim"] * size + rows * 4 * case["lse"],
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    if case["op"] in ("accept", "select"):
        size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        rows = sum(_nodes(case)) if case["op"] == "accept" else case["sequences"] * case["beams"]
        values = rows * case["vocab"]
        return {"bytes": values * size + 16 * rows + 16 * case["sequences"], "flops": values * (1 if case["op"] == "accept" else 4)}
    if case["op"] == "keep":
        moved = sum(max(0, k - 1) for k in _kept(case))
        return {"bytes": 2 * moved * case["layers"] * _row_bytes(case) + 4 * sum(_kept(case)) + 8 * case["sequences"], "flops": 0}
    lens, b = _lengths(case["shortest"], case["longest"], case["sequences"]), case["beams"]
    rows = sum(n % case["block"] for n in lens) * (b - 1)  # of b beams one, on average, is its own parent
    tables = sum(n // case["block"] for n in lens) * b
    return {"bytes": 2 * rows * case["layers"] * _row_bytes(case) + 8 * tables + 8 * b * len(lens), "flops": 0}


# ----------------------------------------------------------------- inputs
def _tree(rng, n):
    """Parents of n nodes: every node but the first follows an earlier one, often a recent one."""
    return [-1] + [rng.randrange(i) if rng.random() < 0.5 else i - 1 - rng.randrange(min(i, 4)) for i in range(1, n)] if n else []


def _masks(parents, words):
    """Words of 64 bits (as signed numbers) of each node's ancestors and itself."""
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return [[((m >> 64 * w) + (1 << 63)) % (1 << 64) - (1 << 63) for w in range(words)] for m in seen]


def _forest(case, seed):
    rng = random.Random(seed)
    parents = [_tree(rng, n) for n in _nodes(case)]
    words = max(1, -(-case["nodes_longest"] // 64))
    mask = torch.tensor([m for p in parents for m in _masks(p, words)], dtype=torch.int64).view(-1, words)
    n = [len(p) for p in parents]
    cu = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32)
    return parents, mask.cuda(), cu.cuda()


def _rows(gen, shape, dtype, mul):
    """[..., heads, dim] as a projection leaves K or V: normal values, a few channels far larger than the rest."""
    x = torch.randn(shape, generator=gen, device="cuda") * mul
    x[..., ::shape[-1] // 5] *= 6
    return x.to(dtype)


def _quantise(x):
    """e4m3 codes of rows x [..., head_dim] (ordinary values), and the exponents (plus 127) of their scales."""
    mantissa, power = torch.frexp(x.abs().amax(-1, keepdim=True))  # 448 is 0.875 * 2^9
    e = (power - 9 + (mantissa > 0.875) + 127).clamp(1, 254)
    return (x * (254 - e << 23).view(torch.float32)).clamp(-448, 448).to(E4M3), e.squeeze(-1).to(torch.uint8)


def _tables(lens, block, gen, spare=3):
    """Block tables over a shuffled pool that has `spare` blocks more, and the pool's size."""
    have = [-(-n // block) for n in lens]
    order = torch.randperm(sum(have) + spare, generator=gen, dtype=torch.int32)
    table = torch.full((len(lens), max(1, max(have))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(have):
        table[b, :n] = order[at:at + n]
        at += n
    return table.cuda(), order.numel()


def _prepare_tree(case, gen, host, seed):
    kv, d, dtype, block = case["kv_heads"], case["dim"], DTYPES[case["dtype"]], case["block"]
    _, mask, cu = _forest(case, seed)
    lens = [a + b for a, b in zip(_cached(case), _nodes(case))]
    table, blocks = _tables(lens, block, host)
    k, v = (_rows(gen, (blocks, block, kv, d), torch.float32, m) for m in (0.5, 1.0))
    scales = None
    if case["cache"] == "e4m3":
        (k, ks), (v, vs) = _quantise(k), _quantise(v)
        scales = torch.stack([ks, vs], -1).transpose(1, 2).contiguous()
    else:
        k, v = k.to(dtype), v.to(dtype)
    total = sum(_nodes(case))
    q = (torch.randn(total, case["heads"], d, generator=gen, device="cuda") * 0.7).to(dtype)
    return dict(q=q, k_cache=k, v_cache=v, kv_scales=scales, block_tables=table, mask=mask, cu=cu, total=total,
                seq_lens=torch.tensor(lens, dtype=torch.int32).cuda(), longest=max(lens), window=case["window"] or None)


def _prepare_accept(case, gen, host, seed):
    parents, mask, cu = _forest(case, seed)
    total, vocab = sum(map(len, parents)), case["vocab"]
    logits = (torch.randn(total, vocab, generator=gen, device="cuda") * 2.5).to(DTYPES[case["dtype"]])
    # Drafts guess well: a node's token is the choice after its parent two times in three.
    first = [c for c, p in zip(cu.tolist(), parents) for _ in p]
    flat = [p for tree in parents for p in tree]
    parent = torch.tensor([at + max(p, 0) for at, p in zip(first, flat)], dtype=torch.long).cuda()
    guess = torch.randint(0, vocab, (total,), generator=gen, device="cuda")
    good = torch.rand(total, generator=gen, device="cuda") < 0.67
    choice = logits.float().argmax(1) if total else guess
    return dict(logits=logits, tokens=torch.where(good, choice[parent] if total else guess, guess), mask=mask, cu=cu, total=total,
                seq_lens=torch.randint(0, 4000, (len(parents),), generator=gen, device="cuda", dtype=torch.int32))


def _caches(case, gen, blocks):
    """K and V of all layers, and an 8-bit cache's scales, each one tensor [layers, ...]."""
    shape = (case["layers"], blocks, case["block"], case["kv_heads"], case["dim"])
    if case["cache"] != "e4m3":
        return (*(torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[case["cache"]]) for _ in range(2)), None)
    k, v = (torch.randint(0, 127, shape, generator=gen, device="cuda", dtype=torch.uint8).view(E4M3) for _ in range(2))
    scales = torch.randint(110, 130, (*shape[:2], shape[3], shape[2], 2), generator=gen, device="cuda", dtype=torch.uint8)
    return k, v, scales


def _prepare_keep(case, gen, host, seed):
    rng = random.Random(seed)
    nodes, kept, n = _nodes(case), _kept(case), case["sequences"]
    table, blocks = _tables([case["cached"] + m for m in nodes], case["block"], host)
    keep = torch.full((n, max(1, max(kept))), -1, dtype=torch.int32)
    for b, (m, c) in enumerate(zip(nodes, kept)):
        if c > 1:
            keep[b, 1:c] = torch.tensor(sorted(rng.sample(range(2, m), c - 1)), dtype=torch.int32)
        if c:
            keep[b, 0] = 0
    k, v, scales = _caches(case, gen, blocks)
    lens = torch.tensor([case["cached"] + c for c in kept], dtype=torch.int32)
    return dict(k=k, v=v, scales=scales, block_tables=table, keep=keep.cuda(), counts=torch.tensor(kept, dtype=torch.int32).cuda(),
                seq_lens=lens.cuda())


def _prepare_select(case, gen, host, seed):
    n, k = case["sequences"], case["beams"]
    logits = (torch.randn(n * k, case["vocab"], generator=gen, device="cuda") * 2.5).to(DTYPES[case["dtype"]])
    return dict(logits=logits, scores=-torch.rand(n, k, generator=gen, device="cuda") * 6 - 20)


def _prepare_reorder(case, gen, host, seed):
    n, k, block = case["sequences"], case["beams"], case["block"]
    lens = _lengths(case["shortest"], case["longest"], n)
    # Complete blocks are shared: each is one of two that some of the beams wrote. The last one is a beam's own.
    full = [x // block for x in lens]
    order = torch.randperm(sum(2 * f + k for f in full) + 3, generator=host, dtype=torch.int32)
    table, at = torch.full((n, k, max(full) + 1), -1, dtype=torch.int32), 0
    for b, f in enumerate(full):
        two = order[at:at + 2 * f].view(2, f)
        table[b, :, :f] = two.gather(0, torch.randint(0, 2, (k, f), generator=host))
        table[b, :, f] = order[at + 2 * f:at + 2 * f + k]
        at += 2 * f + k
    table, blocks = table.view(n * k, -1).cuda(), order.numel()
    kc, vc, scales = _caches(case, gen, blocks)
    return dict(k=kc, v=vc, scales=scales, block_tables=table, seq_lens=torch.tensor([x for x in lens for _ in range(k)], dtype=torch.int32).cuda(),
                parents=torch.randint(0, k, (n, k), generator=gen, device="cuda", dtype=torch.int32))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    s = {"tree": _prepare_tree, "accept": _prepare_accept, "keep": _prepare_keep, "select": _prepare_select,
         "reorder": _prepare_reorder}[case["op"]](case, gen, host, seed)
    s["case"] = case
    return s


# ------------------------------------------------------------ plain forms
def _places(s):
    """Sequence and index of each node of the packed rows."""
    t = torch.arange(s["total"], device="cuda")
    b = torch.bucketize(t, s["cu"][1:].long(), right=True)
    return b, t - s["cu"].long()[b]


def _bits(mask, n):
    """Whether each row's bits 0 .. n - 1 are set."""
    j = torch.arange(n, device="cuda")
    return (mask[:, j // 64] >> (j % 64) & 1).bool()


def _power(e):
    """2^(e - 127) in fp32, from its bits."""
    return (e.int() << 23).view(torch.float32)


def _tree_attention(s):
    case, lens = s["case"], s["seq_lens"].long()
    B, kv, group, d, block = case["sequences"], case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"], case["block"]
    most, S = max(1, case["nodes_longest"]), max(1, s["longest"])
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    base = lens - n
    at = torch.arange(S, device="cuda")
    held = at < lens[:, None]
    slot = torch.where(held, s["block_tables"][:, at // block].long() * block + at % block, 0)
    k, v = (s[name].view(torch.uint8).flatten(0, 1)[slot].view(E4M3).float() if s["kv_scales"] is not None
            else s[name].flatten(0, 1)[slot].float() for name in ("k_cache", "v_cache"))
    if s["kv_scales"] is not None:
        scale = _power(s["kv_scales"].transpose(1, 2).flatten(0, 1)[slot])
        k, v = k * scale[..., :1], v * scale[..., 1:]
    tb, ti = _places(s)
    q = torch.zeros(B, most, case["heads"], d, device="cuda")
    q[tb, ti] = s["q"].float()
    q = q.view(B, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(B, kv, group * most, d)
    bits = torch.zeros(B, most, most, dtype=torch.bool, device="cuda")
    bits[tb, ti] = _bits(s["mask"], most)
    draft = at - base[:, None]  # [B, S]
    seen = (draft < 0)[:, None].expand(-1, most, -1)
    if s["window"] is not None:
        p = base[:, None] + bits.sum(-1).clamp(min=1) - 1
        seen = seen & ((at > p[..., None] - s["window"]) | (at < case["sinks"]))
    drafted = bits.gather(2, draft.clamp(0, most - 1)[:, None].expand(-1, most, -1)) & (draft >= 0)[:, None]
    seen = (seen | drafted) & held[:, None]
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).mul_(1 / math.sqrt(d)).view(B, kv, group, most, S)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, kv, group * most, S), v.transpose(1, 2).contiguous()).view(B, kv, group, most, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, -1, d)[tb, ti].to(s["q"].dtype)
    if not case["lse"]:
        return o
    return o, (top + total.log()).view(B, -1, most).transpose(1, 2)[tb, ti].T.contiguous()


def _first_largest(x):
    """Index of each row's largest value, the first of equals."""
    return (x == x.amax(1, keepdim=True)).to(torch.uint8).argmax(1)


def _accept(s):
    B, most, total = s["case"]["sequences"], max(1, s["case"]["nodes_longest"]), s["total"]
    tb, ti = _places(s)
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    choice = torch.full((B, most), -1, device="cuda")
    tokens, bits = torch.full_like(choice, -2), torch.zeros(B, most, most, dtype=torch.bool, device="cuda")
    if total:
        choice[tb, ti] = _first_largest(s["logits"])
    tokens[tb, ti] = s["tokens"]
    bits[tb, ti] = _bits(s["mask"], most)
    eye = torch.eye(most, dtype=torch.bool, device="cuda")
    # child[b, i, j]: node j sees what i sees, and itself
    above = bits & ~eye
    child = (above[:, None] == bits[:, :, None]).all(-1) & torch.ones_like(eye).triu(1) & bits.any(-1)[:, :, None] & bits.any(-1)[:, None]
    taken = child & (tokens[:, None] == choice[:, :, None])          # the choice after i is j's token ..
    taken &= taken.int().cumsum(2) == 1                              # .. and that of none before it
    good = taken.any(1) | (torch.arange(most, device="cuda") == 0)
    path = (good[:, None] | ~bits).all(2) & bits.any(-1)             # all that a node sees are
    counts = path.sum(1)
    order = torch.where(path, torch.arange(most, device="cuda"), most).sort(1).values
    last = (counts - 1).clamp(min=0)[:, None]
    end = torch.where(n > 0, choice.gather(1, order.gather(1, last).clamp(max=most - 1))[:, 0], -1)
    s["seq_lens"] += counts.int()
    return torch.where(order < most, order, -1).int(), counts.int(), end, s["seq_lens"]


def _slot(s, b, position):
    block = s["case"]["block"]
    return s["block_tables"][b, position // block].long() * block + position % block


def _move(s, to, source):
    """Rows at the slots `source` of all layers to the slots `to`."""
    block = s["case"]["block"]
    for name in ("k", "v"):
        rows = s[name].view(torch.uint8) if s["scales"] is not None else s[name]
        rows = rows.flatten(1, 2)
        rows[:, to] = rows[:, source]
    if s["scales"] is not None:
        s["scales"][:, to // block, :, to % block] = s["scales"][:, source // block, :, source % block]


def _keep(s):
    start = (s["seq_lens"] - s["counts"]).long()
    i = torch.arange(s["keep"].shape[1], device="cuda")
    b, i = ((i < s["counts"][:, None]) & (s["keep"] > i)).nonzero(as_tuple=True)
    _move(s, _slot(s, b, start[b] + i), _slot(s, b, start[b] + s["keep"][b, i].long()))
    return s["k"], s["v"], s["scales"]


def _select(s):
    scores = s["scores"].double()
    n, k = scores.shape
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    x = x - (top + (x - top).exp().sum(1, keepdim=True).log())
    x = (scores.view(n * k, 1) + x).view(n, -1)
    best, at = x.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :s["case"]["number"]], at[:, :s["case"]["number"]]
    vocab = s["case"]["vocab"]
    return best.float(), (at // vocab).int(), at % vocab


def _reorder(s):
    n, k = s["parents"].shape
    block, parent = s["case"]["block"], s["parents"].long()
    length = s["seq_lens"].view(n, k)[:, 0].long()
    full = length // block
    b, beam, row = (torch.arange(block, device="cuda") < (length % block)[:, None, None]).expand(n, k, block).nonzero(as_tuple=True)
    at = full[b] * block + row
    _move(s, _slot(s, b * k + beam, at), _slot(s, b * k + parent[b, beam], at))
    table = s["block_tables"].view(n, k, -1)
    theirs = table.gather(1, parent[..., None].expand_as(table))
    s["block_tables"].copy_(torch.where(torch.arange(table.shape[2], device="cuda") < full[:, None, None], theirs, table).view(n * k, -1))
    return s["k"], s["v"], s["scales"], s["block_tables"]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"tree": _tree_attention, "accept": _accept, "keep": _keep, "select": _select, "reorder": _reorder}[op](s)
    from lightserve_amd.kernels.beam_search import beam_search_select, kv_cache_reorder
    from lightserve_amd.kernels.draft_tree import accept_drafts, kv_cache_keep, paged_tree_attention
    if op == "tree":
        return paged_tree_attention(s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["cu"], s["seq_lens"], s["mask"],
                                    max_nodes=s["case"]["nodes_longest"], return_lse=s["case"]["lse"], kv_scales=s["kv_scales"],
                                    window=s["window"], sinks=s["case"]["sinks"])
    if op == "accept":
        return *accept_drafts(s["logits"], s["tokens"], s["mask"], s["cu"], max_nodes=max(1, s["case"]["nodes_longest"]),
                              seq_lens=s["seq_lens"]), s["seq_lens"]
    if op == "select":
        return beam_search_select(s["logits"], s["scores"], s["case"]["number"])
    if op == "keep":
        kv_cache_keep(s["k"], s["v"], s["block_tables"], s["seq_lens"], s["keep"], s["counts"], kv_scales=s["scales"])
        return s["k"], s["v"], s["scales"]
    kv_cache_reorder(s["k"], s["v"], s["block_tables"], s["seq_lens"], s["parents"], kv_scales=s["scales"])
    return s["k"], s["v"], s["scales"], s["block_tables"]


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The outputs of tree and select in 64 bits. (accept gives whole numbers, keep and reorder move rows as they are.)"""
    if case["op"] not in ("tree", "select"):
        return None
    s = prepare(case, seed)
    if case["op"] == "select":
        n, k, vocab = case["sequences"], case["beams"], case["vocab"]
        out = torch.empty(n, case["number"], dtype=torch.double, device="cuda")
        for b in range(n):
            x = torch.log_softmax(s["logits"][b * k:(b + 1) * k].double(), 1) + s["scores"][b].double()[:, None]
            out[b] = torch.topk(x.view(-1), case["number"]).values
        return out, None, None
    kv, d, block, group = case["kv_heads"], case["dim"], case["block"], case["heads"] // case["kv_heads"]
    table, cu, lens, mask = (s[name].tolist() for name in ("block_tables", "cu", "seq_lens", "mask"))
    k, v = (s[name].double().flatten(0, 1) for name in ("k_cache", "v_cache"))
    if s["kv_scales"] is not None:
        scale = torch.exp2(s["kv_scales"].double() - 127).transpose(1, 2).flatten(0, 1)
        k, v = k * scale[..., :1], v * scale[..., 1:]
    out = torch.zeros(s["total"], case["heads"], d, device="cuda", dtype=torch.double)
    log = torch.full((s["total"], case["heads"]), -math.inf, device="cuda", dtype=torch.double)
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if not n:
            continue
        base = length - n
        hidden = torch.zeros(n, length, dtype=torch.bool)
        for i in range(n):
            m = sum((w % (1 << 64)) << 64 * j for j, w in enumerate(mask[cu[b] + i]))
            if case["window"]:
                low = base + bin(m).count("1") - case["window"]
                hidden[i, min(case["sinks"], max(0, low)):max(0, min(low, base))] = True
            hidden[i, base:] = torch.tensor([not m >> j & 1 for j in range(n)])
        hidden = hidden.cuda()
        at = torch.tensor([table[b][p // block] * block + p % block for p in range(length)], device="cuda")
        for h in range(case["heads"]):
            x = s["q"][cu[b]:cu[b + 1], h].double() @ k[at, h // group].T.contiguous() / math.sqrt(d)
            x[hidden] = -math.inf
            log[cu[b]:cu[b + 1], h] = x.logsumexp(1)
            out[cu[b]:cu[b + 1], h] = torch.softmax(x, 1).nan_to_num(0.0) @ v[at, h // group]
    return (out, log.T.contiguous()) if case["lse"] else out
