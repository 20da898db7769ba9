"""Decoding with several candidates per sequence where a cache ends, on the CPU: the oracle, and checks of calls that reach past
what a cache or a launch has."""
from types import SimpleNamespace

import pytest
import torch

from lightserve_amd import _lib
from lightserve_amd.kernels.draft_tree import draft_tree
from lightserve_amd.model.candidates import LookupDrafts
from lightserve_amd.model.graph_decode import KVCacheDecoder, main
from lightserve_amd.model.minimal_llama import TOY_CONFIG
from oracle import candidates, paged8
from tests.paged8_cases import tables
from tests.test_candidates_cpu import WINDOW, _set


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


def _decoder(window, sinks=0):
    return KVCacheDecoder(SimpleNamespace(layers=[None]), TOY_CONFIG, 2, device="cpu", window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(4, 0), (4, 2)])
def test_oracle_tree_under_a_window(window, sinks):
    """Nodes less deep than the window are one-token steps; deeper ones see all of their ancestors, and are not."""
    n, had = 9, 30
    table, pool = tables([had + n], 16, 1)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(pool, 16, 2, 8, generator=g).double() for _ in range(2))
    q = torch.randn(n, 4, 8, generator=g)
    o = candidates.tree_reference(q, k, v, table, [0, n], [had + n], draft_tree(range(-1, n - 1))[0], window, sinks)[0]
    want = paged8.window_reference(q, k, v, table, torch.tensor([0, n], dtype=torch.int32), [had + n], window, sinks)[0]
    same = [torch.allclose(o[i], want[i], atol=1e-12) for i in range(n)]
    assert same == [i < window for i in range(n)]


def test_refuses_trees_deeper_than_the_window():
    for window in (1, 4):
        with pytest.raises(AssertionError, match="window"):
            LookupDrafts(_decoder(window), window, 2)
    LookupDrafts(_decoder(4), 3, 20)
    LookupDrafts(_decoder(None), 30)
    dec = _decoder(4, 2)
    step = (torch.zeros(2, 5, dtype=torch.long), torch.ones(10, 1, dtype=torch.int64), torch.zeros(2, 5, dtype=torch.int32))
    for deepest in (None, 4, 100):
        with pytest.raises(AssertionError, match="window"):
            dec.draft_step(*step, deepest=deepest)
    with pytest.raises(AttributeError):  # (past the checks: the decoder has no weights)
        dec.draft_step(*step, deepest=3)
    for words in (["--drafts", "4", "--window", "4"], ["--drafts", "9", "--window", "4", "--branches", "2"]):
        with pytest.raises(SystemExit):
            main(words)


def test_oracle_accept_reads_no_bits_past_the_nodes():
    logits = torch.eye(4)[[2, 1, 3, 0, 2]]
    mask, cu, tokens = draft_tree([-1, 0, 0, 2, 3])[0], torch.tensor([0, 5]), [0, 1, 2, 3, 0]
    want = candidates.accept_reference(logits, tokens, mask, cu, 5)
    assert want == ([[0, 2, 3, 4, -1]], [4], [2])
    for bits in (1 << 5, 1 << 62, -1 << 5):
        dirty = mask.clone()
        dirty[::2] |= bits
        assert candidates.accept_reference(logits, tokens, dirty, cu, 5) == want


def test_tree_check_counts_the_merging_launch(built_library):
    """The launch that merges partial results has 512 threads for each row tile and KV head, more than the first one where two or
    four waves take a tile: 2^23 of them are refused by the check, not by the launch."""
    def check(heads_kv, nodes, **kw):
        return _lib.tree_check(_set(_lib.TreeArgs, WINDOW, dict(
            tree_mask=4096, mask_stride=1, mask_words=1, batch=65535, tokens=65535 * nodes, max_seqlen_q=nodes, heads_kv=heads_kv, heads_q=heads_kv,
            max_seq_len=64, max_blocks_per_seq=4, workspace_bytes=1 << 60) | kw))
    assert check(127, 20)[0] == 0
    for heads_kv, nodes in ((129, 20), (129, 65), (400, 33)):
        rc, msg = check(heads_kv, nodes, mask_words=2, mask_stride=2)
        assert rc == -2 and "threads" in msg, (heads_kv, nodes, rc, msg)


def test_tree_check_counts_whatever_the_offsets(built_library):
    """Offsets are the device's to read: with some that let sequences share rows, every one of 65535 may have 256 nodes, and the numbers
    of their key tiles have to stay below 2^31."""
    def check(tokens, batch, **kw):
        return _lib.tree_check(_set(_lib.TreeArgs, WINDOW, dict(
            tree_mask=4096, mask_stride=4, mask_words=4, batch=batch, tokens=tokens, max_seqlen_q=256, heads_kv=8, heads_q=256, max_seq_len=16384,
            max_blocks_per_seq=1024, block_table_stride=1024, workspace_bytes=1 << 60) | kw))
    rc, msg = check(256, 65535)
    assert rc == -2 and "tiles" in msg
    assert check(256, 4096)[0] == 0 and check(256 * 4096, 4096)[0] == 0
    assert check(3, 65535)[0] == 0  # (three rows of q: no sequence has more)
