"""Paged caches and batches for the tests of the 8-bit cache and of windowed attention."""
import torch


def offsets(lens):
    return torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32)


def tables(lens, bs, seed, spare=3, extra=2):
    """Block tables [batch, max_blocks] over a shuffled pool with `spare` blocks that no sequence holds; unused entries are
    -1, and there are `extra` of them behind the longest sequence's."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need + [0]) + extra), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def random_codes(shape, g):
    """e4m3 bits without NaN."""
    return torch.randint(0, 127, shape, generator=g, dtype=torch.uint8) | torch.randint(0, 2, shape, generator=g, dtype=torch.uint8) << 7


def cache8(blocks, bs, heads, d, seed):
    """Random codes with scales that make values of about one (uint8 codes K, V, exponents)."""
    g = torch.Generator().manual_seed(seed)
    k, v = (random_codes((blocks, bs, heads, d), g) for _ in range(2))
    return k, v, torch.randint(117, 121, (blocks, heads, bs, 2), generator=g, dtype=torch.uint8)
