"""Trees, batches and caches for the tests of decoding with several candidates per sequence."""
import random

import torch

from lightserve_amd.kernels.draft_tree import draft_tree
from tests.paged8_cases import offsets

E4M3 = torch.float8_e4m3fn


def random_parents(n, seed):
    rng = random.Random(seed)
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, n)] if n else []


def forest(nodes, seed, words=None):
    """Parents of each tree, masks of all nodes, offsets."""
    words = words or max(1, -(-max(nodes + [1]) // 64))
    parents = [random_parents(n, seed + b) for b, n in enumerate(nodes)]
    mask = torch.cat([draft_tree(p, words)[0] for p in parents]) if parents else torch.zeros(0, words, dtype=torch.int64)
    return parents, mask, offsets(nodes)


def layer_caches(kind, layers, pool, bs, heads, d, seed):
    """K, V and scales (or None) of all layers, on the CPU; 8-bit ones as uint8 codes."""
    g = torch.Generator().manual_seed(seed)
    shape = (layers, pool, bs, heads, d)
    if kind == E4M3:
        k, v = (torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) for _ in range(2))
        return k, v, torch.randint(0, 256, (layers, pool, heads, bs, 2), generator=g, dtype=torch.uint8)
    k, v = (torch.randn(shape, generator=g).to(kind) for _ in range(2))
    return k, v, None


def on_gpu(kind, k, v, scales):
    if kind == E4M3:
        return k.cuda().view(E4M3), v.cuda().view(E4M3), scales.cuda()
    return k.cuda(), v.cuda(), None


def raw(t):
    """Bits of a cache, on the CPU."""
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]
    return t.cpu().view(bits)
