"""Draft trees at the end of a cache: nodes whose rows the block table does not have, against the float64 oracle.

Bounds of the attention are those of test_draft_tree_gpu.py, whose derivation does not depend on where the keys end.
"""
import pytest
import torch

from lightserve_amd.kernels.draft_tree import paged_tree_attention
from oracle import candidates
from tests.candidate_cases import forest
from tests.paged8_cases import tables
from tests.test_draft_tree_gpu import KINDS, _assert_close, _cache, _i32

pytestmark = pytest.mark.gpu


def _past(kind, dtype, nodes, had, blocks, hq, hkv, d, bs, seed, window=None, sinks=0, what=""):
    """Trees behind `had` tokens over tables of `blocks` blocks, which lengths pass."""
    lens = [a + b for a, b in zip(nodes, had)]
    table, pool = tables(lens, bs, seed)
    table = table[:, :blocks]
    cache, vals = _cache(kind, dtype, pool, bs, hkv, d, seed + 1)
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(seed + 2)).to(dtype)
    _, tree, cu = forest(nodes, seed + 3)
    o, lse = paged_tree_attention(q.cuda(), *cache[:2], table.cuda(), cu.cuda(), _i32(lens).cuda(), tree.cuda(), return_lse=True,
                                  kv_scales=cache[2], window=window, sinks=sinks)
    torch.cuda.synchronize()
    _assert_close(o, lse.t(), candidates.tree_reference(q, *vals, table, cu, lens, tree, window, sinks), max(lens), what)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3), (6, 0), (300, 70), (90, 0), (300, 2)])
def test_tree_past_the_table(gpu, kind, dtype, hq, hkv, window, sinks):
    """Every number of rows past the table, tables that end inside a key tile, and lengths far behind them."""
    print(f"case past {kind} {dtype} {hq} {hkv} window={window} sinks={sinks}", flush=True)
    for blocks in (4, 3):
        end = 16 * blocks
        had = [end - 10, end - 9, end - 5, end - 1, end, end + 40, 3]
        _past(kind, dtype, [4] * len(had), had, blocks, hq, hkv, 64, 16, blocks, window, sinks, "few rows")
        _past(kind, dtype, [9] * len(had), had, blocks, hq, hkv, 64, 16, blocks, window, sinks, "more")
        _past(kind, dtype, [70] * len(had), had, blocks, hq, hkv, 64, 16, blocks, window, sinks, "many")


@pytest.mark.parametrize("kind,dtype", KINDS[::2])
@pytest.mark.parametrize("nodes", [[2, 2], [12, 7], [200, 100]])
def test_long_tree_past_the_table(gpu, kind, dtype, nodes):
    """Sequences that several workgroups share."""
    print(f"case past, long {kind} {dtype} {nodes}", flush=True)
    for window, sinks in ((None, 0), (2000, 5)):
        _past(kind, dtype, nodes, [3200, 3190], 200, 4, 2, 64, 16, 5, window, sinks, "long")
    _past(kind, dtype, nodes * 33, [390, 399] * 33, 25, 4, 2, 64, 16, 6, what="many sequences")


@pytest.mark.parametrize("nodes", [4, 9, 70])
def test_far_past_the_table(gpu, nodes):
    """A length of 2^31 - 1 is a length: the sequence's certain tokens that are held, and no draft."""
    print(f"case far past {nodes}", flush=True)
    table, pool = tables([60], 16, 1)
    cache, vals = _cache("16 bit", torch.bfloat16, pool, 16, 2, 64, 2)
    q = torch.randn(nodes, 8, 64, generator=torch.Generator().manual_seed(3)).bfloat16()
    _, tree, cu = forest([nodes], 4)
    for window, sinks in ((None, 0), (5, 2)):
        o, lse = paged_tree_attention(q.cuda(), *cache[:2], table.cuda()[:, :4], cu.cuda(), _i32([2 ** 31 - 1]).cuda(), tree.cuda(),
                                      return_lse=True, window=window, sinks=sinks)
        # (the oracle goes through a length's keys one by one)
        ref = candidates.tree_reference(q, *vals, table[:, :4], cu, [64 + 200 + nodes], tree, window, sinks)
        _assert_close(o, lse.t(), ref, 64, "far")
