"""Decoding with several candidates per sequence, in float64 and one candidate at a time.

tree_reference     attention of draft trees over paged caches, with what an error bound needs
accept_reference   the path of each tree, its length and the token behind it
keep_reference     kv_cache_keep on copies of the caches
select_reference   beam_search_select
reorder_reference  kv_cache_reorder on copies of the caches and tables
"""
import math

import torch


def bits_of(row):
    """A mask's words (signed 64-bit) as one whole number."""
    return sum((int(w) % (1 << 64)) << 64 * i for i, w in enumerate(row.tolist()))


def _place(table, num_blocks, bs, b, pos):
    i = pos // bs
    if pos < 0 or i >= table.shape[1] or not 0 <= int(table[b, i]) < num_blocks:
        return None
    return int(table[b, i]), pos % bs


def tree_reference(q, k, v, table, cu, seq_lens, mask, window=None, sinks=0, sm_scale=None):
    """q [T, Hq, D], caches float64 [blocks, bs, Hkv, D] -> o, lse [T, Hq], sum w |v|, the largest sum |q k| |scale|, and sum |v|.
    Nobody sees what lies past the table."""
    T, hq, d = q.shape
    n_blocks, bs, hkv, _ = k.shape
    scale = 1 / math.sqrt(d) if sm_scale is None else sm_scale
    o, a, plain = (torch.zeros(T, hq, d, dtype=torch.double) for _ in range(3))
    lse, big = torch.full((T, hq), -math.inf, dtype=torch.double), torch.zeros(T, hq, dtype=torch.double)
    for b, length in enumerate(int(x) for x in seq_lens):
        t0, n = int(cu[b]), int(cu[b + 1] - cu[b])
        base, held = length - n, min(length, table.shape[1] * bs)
        rows = torch.zeros(max(length, 1), 2, hkv, d, dtype=torch.double)  # what no block holds reads as zeros
        for j in range(length):
            at = _place(table, n_blocks, bs, b, j)
            if at is not None:
                rows[j, 0], rows[j, 1] = k[at], v[at]
        for i in range(n):
            m = bits_of(mask[t0 + i]) & ((1 << n) - 1)
            pos = base + max(bin(m).count("1"), 1) - 1
            sees = [j for j in range(max(base, 0)) if window is None or j > pos - window or j < sinks]
            sees += [base + j for j in range(n) if m >> j & 1 and base + j >= 0]
            sees = [j for j in sees if j < held]
            if not sees:
                continue
            kk, vv = rows[sees, 0].repeat_interleave(hq // hkv, 1), rows[sees, 1].repeat_interleave(hq // hkv, 1)
            qq = q[t0 + i].double()
            x = (kk * qq).sum(-1) * scale
            lse[t0 + i] = x.logsumexp(0)
            w = torch.softmax(x, 0)[..., None]
            o[t0 + i], a[t0 + i] = (w * vv).sum(0), (w * vv.abs()).sum(0)
            plain[t0 + i] = vv.abs().sum(0)
            big[t0 + i] = ((kk * qq).abs().sum(-1) * abs(scale)).amax(0)
    return o, lse, a, big, plain


def first_largest(row):
    """torch's argmax in words: the first NaN, else the first of the largest."""
    best = 0
    for i, x in enumerate(row.tolist()):
        top = float(row[best])
        if (math.isnan(x) and not math.isnan(top)) or x > top:
            best = i
    return best


def accept_reference(logits, tokens, mask, cu, max_nodes):
    """path [B, max_nodes], counts [B], next tokens [B] (lists)."""
    paths, counts, following = [], [], []
    for b in range(len(cu) - 1):
        t0, nodes = int(cu[b]), int(cu[b + 1] - cu[b])
        n, known = min(nodes, max_nodes), (1 << nodes) - 1  # (bits past the nodes say nothing)
        path, nxt = [], -1
        if n > 0:
            path = [0]
            while True:
                cur = path[-1]
                nxt = first_largest(logits[t0 + cur].double())
                child = next((j for j in range(cur + 1, n) if int(tokens[t0 + j]) == nxt
                              and bits_of(mask[t0 + j]) & known == bits_of(mask[t0 + cur]) & known | 1 << j), None)
                if child is None:
                    break
                path.append(child)
        paths.append(path + [-1] * (max_nodes - len(path)))
        counts.append(len(path))
        following.append(nxt)
    return paths, counts, following


def keep_reference(caches, table, seq_lens, keep, counts, slot_first):
    """caches: tensors whose layers' first dims are (blocks, ..) with the slot at dim slot_first once a block is chosen. Copies with the rows moved."""
    out = [c.clone() for c in caches]
    bs = caches[0].shape[2]
    for b in range(len(seq_lens)):
        n = min(max(int(counts[b]), 0), keep.shape[1])
        start = int(seq_lens[b]) - n
        for i in range(n):
            if int(keep[b, i]) <= i:
                continue
            src, dst = (_place(table, caches[0].shape[1], bs, b, start + j) for j in (int(keep[b, i]), i))
            if src is None or dst is None:
                continue
            for o, c, at in zip(out, caches, slot_first):
                o[:, dst[0]].select(at, dst[1]).copy_(c[:, src[0]].select(at, src[1]))
    return out


def select_reference(logits, scores, num):
    """Lists of (score, beam, token) per sequence, best first, in float64."""
    n, k = scores.shape
    out = []
    for b in range(n):
        cands = []
        for j in range(k):
            x = logits[b * k + j].double()
            s = float(scores[b, j])
            if math.isnan(s) or s == -math.inf or torch.isnan(x).any() or x.max() == math.inf or x.max() == -math.inf:
                continue
            lse = float(x.logsumexp(0))
            cands += [(s + (float(e) - lse), j, v) for v, e in enumerate(x.tolist()) if e > -math.inf]
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        out.append(cands[:num] + [(-math.inf, 0, 0)] * max(0, num - len(cands)))
    return out


def reorder_reference(caches, table, seq_lens, parents, slot_first):
    """Copies of the caches and the table after kv_cache_reorder."""
    out, new = [c.clone() for c in caches], table.clone()
    bs, (n, k) = caches[0].shape[2], parents.shape
    for b in range(n):
        length = min(max(int(seq_lens[b * k]), 0), table.shape[1] * bs)
        full, rest = length // bs, length % bs
        for j in range(k):
            p = int(parents[b, j])
            p = p if 0 <= p < k else j
            new[b * k + j, :full] = table[b * k + p, :full]
            if p == j or rest == 0:
                continue
            src, dst = int(table[b * k + p, full]), int(table[b * k + j, full])
            if not (0 <= src < caches[0].shape[1] and 0 <= dst < caches[0].shape[1]):
                continue
            for o, c, at in zip(out, caches, slot_first):
                o[:, dst].narrow(at, 0, rest).copy_(c[:, src].narrow(at, 0, rest))
    return out, new
