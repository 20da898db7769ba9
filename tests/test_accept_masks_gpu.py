"""Acceptance reads a mask's bits as far as the sequence has nodes, as the attention does. Whole numbers: equal."""
import pytest
import torch

from oracle import candidates
from tests.test_draft_tree_gpu import _accept, _drafts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nodes,words", [(n, w) for n in ([1, 8], [63, 0, 5], [64, 7], [100, 64, 65], [256, 130])
                                         for w in (1, 2, 4) if max(n) <= 64 * w])
def test_bits_past_the_nodes(gpu, nodes, words):
    print(f"case bits past {nodes} words={words}", flush=True)
    logits, tokens, mask, cu = _drafts(nodes, 300, torch.bfloat16, 3, right=0.95)
    g = torch.Generator().manual_seed(4)
    dirty = torch.randint(-2 ** 63, 2 ** 63 - 1, (mask.shape[0], words), generator=g)
    for b, n in enumerate(nodes):
        for w in range(words):
            rows, bits = slice(int(cu[b]), int(cu[b]) + n), min(max(n - 64 * w, 0), 64)
            known = torch.tensor(-1 if bits == 64 else (1 << bits) - 1)
            own = mask[rows, w] if w < mask.shape[1] else torch.zeros(n, dtype=torch.int64)
            dirty[rows, w] = dirty[rows, w] & ~known | own
    most = max(nodes)
    clean = candidates.accept_reference(logits, tokens, mask, cu, most)
    assert max(clean[1]) > 2 and clean == candidates.accept_reference(logits, tokens, dirty, cu, most)
    _accept(logits, tokens, dirty, cu, "bits past the nodes")
    _accept(logits, tokens, dirty, cu, "fewer nodes taken", max_nodes=max(1, most - 3))
