"""Decoding with several candidates per sequence where a cache ends, on the CPU: the oracle, and checks of calls that reach past
what a cache or a launch has."""
import torch

from lightserve_amd.kernels.draft_tree import draft_tree
from oracle import candidates, paged8
from tests.paged8_cases import tables


def test_oracle_tree_past_the_table():
    """A chain that reaches past the table: each node whose row is there is the one-token step at its place."""
    n, had, end = 9, 58, 64
    table, pool = tables([had + n], 16, 1)
    table = table[:, :end // 16]
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(pool, 16, 2, 8, generator=g).double() for _ in range(2))
    q = torch.randn(n, 4, 8, generator=g)
    o, lse = candidates.tree_reference(q, k, v, table, [0, n], [had + n], draft_tree(range(-1, n - 1))[0])[:2]
    for i in range(n):
        length = min(had + i + 1, end)
        want = paged8.window_reference(q[i:i + 1], k, v, table, torch.tensor([0, 1], dtype=torch.int32), [length], None, 0)
        assert torch.allclose(o[i], want[0][0], atol=1e-12) and torch.allclose(lse[i], want[1][0], atol=1e-12), i
