"""Decoding with several candidates per sequence, on the CPU: the masks of draft trees, the oracle against formulas written
apart from it, the checks of the Python calls and those of the C entry points."""
import ctypes
import math

import pytest
import torch

from lightserve_amd import _lib
from lightserve_amd.kernels.beam_search import beam_search_select, kv_cache_reorder
from lightserve_amd.kernels.draft_tree import accept_drafts, draft_tree, kv_cache_keep, paged_tree_attention
from oracle import candidates, paged8
from tests.candidate_cases import forest, random_parents
from tests.paged8_cases import offsets, tables


# -------------------------------------------------------------- draft_tree
@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 256])
def test_draft_tree(n):
    """Bit j of node i: j is on the way from i to node 0."""
    parents = random_parents(n, n)
    mask, depth = draft_tree(parents)
    assert mask.dtype == torch.int64 and mask.shape == (n, max(1, -(-n // 64))) and depth.dtype == torch.int32
    for i in range(n):
        way, j = set(), i
        while j >= 0:
            way.add(j)
            j = parents[j]
        assert {j for j in range(64 * mask.shape[1]) if int(mask[i, j // 64]) >> (j % 64) & 1} == way
        assert int(depth[i]) == len(way) - 1
    if n <= 64:
        wide, _ = draft_tree(parents, words=3)
        assert torch.equal(wide[:, :1], mask) and not wide[:, 1:].any()


def test_draft_tree_refusals():
    for parents in ([0], [-1, 1], [-1, -1], [-1, 0, 5], [-2], range(-1, 256)):
        with pytest.raises(AssertionError):
            draft_tree(parents)
    with pytest.raises(AssertionError):
        draft_tree(range(-1, 64), words=1)
    with pytest.raises(AssertionError):
        draft_tree([-1], words=5)


# ------------------------------------------------------------------ oracle
def test_oracle_tree_of_a_chain_is_a_chunk():
    n, had = [3, 7, 0], [20, 0, 9]
    lens = [a + b for a, b in zip(n, had)]
    table, pool = tables(lens, 16, 1)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(pool, 16, 2, 8, generator=g).double() for _ in range(2))
    q = torch.randn(sum(n), 4, 8, generator=g)
    mask = torch.cat([draft_tree(range(-1, m - 1))[0] for m in n])
    for window, sinks in ((None, 0), (9, 2)):  # (a window no shorter than a chain)
        a = candidates.tree_reference(q, k, v, table, offsets(n), lens, mask, window, sinks)
        b = paged8.window_reference(q, k, v, table, offsets(n), lens, window, sinks)
        assert torch.allclose(a[0], b[0], atol=1e-12) and torch.allclose(a[1], b[1], atol=1e-12)


def test_oracle_tree_masks():
    """Against attention with an explicit mask."""
    nodes, had = [9], [21]
    table, pool = tables([30], 16, 1)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(pool, 16, 1, 8, generator=g).double() for _ in range(2))
    q = torch.randn(9, 2, 8, generator=g)
    parents, mask, cu = forest(nodes, 5)
    rows = [(int(table[0, j // 16]), j % 16) for j in range(30)]
    kk, vv = (torch.stack([c[r] for r in rows])[:, 0] for c in (k, v))
    seen = torch.zeros(9, 30, dtype=torch.bool)
    seen[:, :21] = True
    for i in range(9):
        j = i
        while j >= 0:
            seen[i, 21 + j] = True
            j = parents[0][j]
    for h in range(2):
        x = (q[:, h].double() @ kk.T / math.sqrt(8)).masked_fill(~seen, -math.inf)
        o = candidates.tree_reference(q, k, v, table, cu, [30], mask)[0]
        assert torch.allclose(o[:, h], torch.softmax(x, 1) @ vv, atol=1e-12)


def test_oracle_accept():
    logits = torch.full((5, 4), 0.0)
    for i, c in enumerate((2, 1, 3, 0, 2)):
        logits[i, c] = 1.0
    mask = draft_tree([-1, 0, 0, 2, 3])[0]
    cu = torch.tensor([0, 5, 5])
    assert candidates.accept_reference(logits, [0, 1, 2, 3, 0], mask, cu, 5) == ([[0, 2, 3, 4, -1], [-1] * 5], [4, 0], [2, -1])
    assert candidates.accept_reference(logits, [0, 2, 2, 3, 0], mask, cu, 5) == ([[0, 1, -1, -1, -1], [-1] * 5], [2, 0], [1, -1])
    assert candidates.first_largest(torch.tensor([1.0, math.nan, 5.0, math.nan])) == 1


def test_oracle_select():
    g = torch.Generator().manual_seed(1)
    x, scores = torch.randn(6, 50, generator=g), torch.randn(2, 3, generator=g)
    all_of = (torch.log_softmax(x.double(), 1).view(2, 3, 50) + scores.double()[..., None]).view(2, -1)
    want = all_of.topk(7)
    for b, row in enumerate(candidates.select_reference(x, scores, 7)):
        assert [c[1] * 50 + c[2] for c in row] == want.indices[b].tolist()
        assert torch.allclose(torch.tensor([c[0] for c in row], dtype=torch.double), want.values[b])


def test_oracle_moves():
    c = torch.arange(1 * 3 * 4 * 1 * 1).view(1, 3, 4, 1, 1)
    table = torch.tensor([[2, 0]])
    out, = candidates.keep_reference([c], table, [4], torch.tensor([[0, 2, 5]]), [3], (1,))
    flat = out.flatten().tolist()  # rows 1 + (0, 2, 5) -> rows 1, 2, 3: positions of block 2
    assert flat[8:12] == [8, 9, 11, 2] and flat[:8] == list(range(8))
    (out,), new = candidates.reorder_reference([c], torch.tensor([[0, 1], [0, 2]]), [6, 6], torch.tensor([[1, 0]]), (1,))
    assert out.flatten().tolist() == [0, 1, 2, 3, 8, 9, 6, 7, 4, 5, 10, 11] and new.tolist() == [[0, 1], [0, 2]]


# --------------------------------------------------------------- refusals
def _tree_call(**kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16),
             v_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), block_tables=torch.zeros(1, 4, dtype=torch.int32),
             cu_seqlens_q=torch.tensor([0, 3], dtype=torch.int32), seq_lens_k=torch.tensor([3], dtype=torch.int32),
             tree_mask=torch.ones(3, 1, dtype=torch.int64)) | kw
    return paged_tree_attention(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(), "GPU"), (dict(tree_mask=torch.ones(3, 1, dtype=torch.int32)), "tree_mask"),
    (dict(tree_mask=torch.ones(2, 1, dtype=torch.int64)), "tree_mask"), (dict(tree_mask=torch.ones(3, 5, dtype=torch.int64)), "tree_mask"),
    (dict(tree_mask=torch.ones(3, dtype=torch.int64)), "tree_mask"), (dict(max_nodes=257), "nodes"), (dict(max_nodes=65), "bit"),
    (dict(max_nodes=-1), "nodes"), (dict(q=torch.zeros(3, 4, 64)), "bf16"), (dict(q=torch.zeros(3, 64)), "packed"),
    (dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), "multiple"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.float16)), "dtype"),
    (dict(k_cache=torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16)), "k_cache"),
    (dict(cu_seqlens_q=torch.tensor([0, 3], dtype=torch.int64)), "cu_seqlens_q"),
    (dict(cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32)), "cu_seqlens_q")])
def test_tree_attention_refusals(kw, word):
    with pytest.raises(AssertionError, match=word):
        _tree_call(**kw)


@pytest.mark.parametrize("kw,word", [
    (dict(), "GPU"), (dict(logits=torch.zeros(3, 8, dtype=torch.double)), "logits"), (dict(logits=torch.zeros(24)), "logits"),
    (dict(logits=torch.zeros(3, 0)), "vocabulary"), (dict(tokens=torch.zeros(3, dtype=torch.int32)), "tokens"),
    (dict(tokens=torch.zeros(2, dtype=torch.int64)), "tokens"), (dict(tree_mask=torch.ones(3, 9, dtype=torch.int64)), "tree_mask"),
    (dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), "cu_seqlens"), (dict(cu_seqlens=torch.tensor([0, 3])), "cu_seqlens"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32)), "seq_lens"), (dict(seq_lens=torch.zeros(1, dtype=torch.int64)), "seq_lens")])
def test_accept_refusals(kw, word):
    a = dict(logits=torch.zeros(3, 8), tokens=torch.zeros(3, dtype=torch.int64), tree_mask=torch.ones(3, 1, dtype=torch.int64),
             cu_seqlens=torch.tensor([0, 3], dtype=torch.int32)) | kw
    with pytest.raises(AssertionError, match=word):
        accept_drafts(**a)


def _cache(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=torch.float32).to(dtype)


E4M3 = torch.float8_e4m3fn
ROWS = [
    (dict(), "GPU"), (dict(k_cache=_cache(4, 16, 2, 64, dtype=torch.float16)), "share"), (dict(k_cache=_cache(4, 16, 2, 32)), "both"),
    (dict(k_cache=_cache(16, 2, 64), v_cache=_cache(16, 2, 64)), "both"),
    (dict(k_cache=_cache(4, 16, 2, 64, dtype=torch.double), v_cache=_cache(4, 16, 2, 64, dtype=torch.double)), "share"),
    (dict(k_cache=_cache(4, 16, 2, 64, dtype=E4M3), v_cache=_cache(4, 16, 2, 64, dtype=E4M3)), "kv_scales"),
    (dict(kv_scales=torch.zeros(4, 2, 16, 2, dtype=torch.uint8)), "kv_scales"),
    (dict(k_cache=_cache(4, 16, 2, 64, dtype=E4M3), v_cache=_cache(4, 16, 2, 64, dtype=E4M3),
          kv_scales=torch.zeros(4, 16, 2, 2, dtype=torch.uint8)), "kv_scales"),
    (dict(v_cache=_cache(4, 16, 64, 2).transpose(2, 3)), "head-dim"), (dict(k_cache=_cache(1, 16, 2, 64).expand(4, -1, -1, -1)), "memory"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "seq_lens"), (dict(block_tables=torch.zeros(2, 4)), "block_tables"),
    (dict(block_tables=torch.zeros(3, 4, dtype=torch.int32)), "block_tables")]


@pytest.mark.parametrize("kw,word", ROWS + [
    (dict(counts=torch.zeros(3, dtype=torch.int32)), "counts"), (dict(keep=torch.zeros(2, 3)), "keep"), (dict(keep=torch.zeros(2, dtype=torch.int32)), "keep")])
def test_keep_refusals(kw, word):
    a = dict(k_cache=_cache(4, 16, 2, 64), v_cache=_cache(4, 16, 2, 64), block_tables=torch.zeros(2, 4, dtype=torch.int32),
             seq_lens=torch.zeros(2, dtype=torch.int32), keep=torch.zeros(2, 3, dtype=torch.int32), counts=torch.zeros(2, dtype=torch.int32)) | kw
    with pytest.raises(AssertionError, match=word):
        kv_cache_keep(**a)


@pytest.mark.parametrize("kw,word", ROWS + [
    (dict(parents=torch.zeros(1, 2)), "parents"), (dict(parents=torch.zeros(1, 65, dtype=torch.int32)), "beams"),
    (dict(block_tables=torch.zeros(4, 2, dtype=torch.int32).t()), "block_tables"),
    (dict(block_tables=torch.zeros(1, 4, dtype=torch.int32).expand(2, -1)), "block_tables")])
def test_reorder_refusals(kw, word):
    a = dict(k_cache=_cache(4, 16, 2, 64), v_cache=_cache(4, 16, 2, 64), block_tables=torch.zeros(2, 4, dtype=torch.int32),
             seq_lens=torch.zeros(2, dtype=torch.int32), parents=torch.zeros(1, 2, dtype=torch.int32)) | kw
    with pytest.raises(AssertionError, match=word):
        kv_cache_reorder(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(), "GPU"), (dict(num=0), "candidates"), (dict(num=65), "candidates"), (dict(scores=torch.zeros(2, 2, dtype=torch.double)), "scores"),
    (dict(scores=torch.zeros(4)), "scores"), (dict(scores=torch.zeros(2, 3)), "row"), (dict(logits=torch.zeros(4, 0)), "vocabulary"),
    (dict(logits=torch.zeros(4, 5, dtype=torch.int32)), "logits"), (dict(logits=torch.zeros(65, 5), scores=torch.zeros(1, 65)), "beams")])
def test_select_refusals(kw, word):
    with pytest.raises(AssertionError, match=word):
        beam_search_select(**(dict(logits=torch.zeros(4, 9), scores=torch.zeros(2, 2)) | kw))


# ------------------------------------------------------------- C entries
def test_struct_sizes(built_library):
    """The mirrors have the C structs' sizes, and the packed forms theirs."""
    import os
    import shutil
    import subprocess
    import tempfile
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    names = {"lsfa_tree_args": _lib.TreeArgs, "lsfa_accept_args": _lib.AcceptArgs, "lsfa_beam_args": _lib.BeamArgs,
             "lsfa_kv_rows_args": _lib.KvRowsArgs}
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    with tempfile.TemporaryDirectory() as tmp:
        src = os.path.join(tmp, "s.c")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include "lightserve_fa.h"\nint main(void){'
                    + "".join(f'printf("%zu\\n", sizeof({n}));' for n in names) + "return 0;}")
        subprocess.run([cc, "-I", include, src, "-o", os.path.join(tmp, "s")], check=True)
        sizes = [int(x) for x in subprocess.run([os.path.join(tmp, "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(c) for c in names.values()] == [_lib._PACK[c].size for c in names.values()]


def _set(cls, base, kw):
    a = cls()
    for name, value in (base | kw).items():
        field = getattr(a, name)
        setattr(a, name, type(field)(*value) if isinstance(value, tuple) else value)
    return a


WINDOW = dict(q=4096, k_cache=4096, v_cache=4096, o=4096, cu_seqlens_q=4096, seq_lens=4096, block_tables=4096, workspace=4096,
              workspace_bytes=1 << 40, q_stride=(512, 64), k_stride=(4096, 256, 64), v_stride=(4096, 256, 64), o_stride=(512, 64),
              block_table_stride=8, dtype=_lib.DTYPE_BF16, batch=2, tokens=9, heads_q=8, heads_kv=4, head_dim=64, block_size=16,
              num_blocks=20, max_blocks_per_seq=8, max_seqlen_q=6, max_seq_len=100, causal=1, sm_scale=0.1)


def test_tree_check(built_library):
    def check(tree=(), **kw):
        return _lib.tree_check(_set(_lib.TreeArgs, WINDOW, dict(tree_mask=4096, mask_stride=1, mask_words=1) | dict(tree) | kw))
    assert check()[0] == 0
    assert check(causal=0, window=5)[0] == 0  # (causal is not read)
    for tree, kw, code, word in [
            (dict(tree_mask=0), {}, -1, "tree_mask"), (dict(tree_mask=4100), {}, -1, "aligned"), (dict(mask_words=0), {}, -1, "mask_words"),
            (dict(mask_words=5, mask_stride=5), {}, -1, "mask_words"), (dict(mask_stride=0), {}, -1, "mask_stride"),
            ({}, dict(max_seqlen_q=65), -1, "bit"), ({}, dict(max_seqlen_q=257), -2, "drafts"), ({}, dict(cu_seqlens_q=0), -1, "cu_seqlens_q"),
            ({}, dict(dtype=_lib.DTYPE_FP32), -2, "bf16"), ({}, dict(head_dim=136), -2, ""), ({}, dict(block_size=8), -2, ""),
            ({}, dict(batch=2, workspace_bytes=8, max_seq_len=100000, max_blocks_per_seq=10000, block_table_stride=10000), -1, "workspace")]:
        rc, msg = check(tree, **kw)
        assert rc == code and word in msg, (tree, kw, rc, msg)
    assert _lib.load().lsfa_tree_check(None) == -1
    assert check(dict(tree_mask=0), tokens=0)[0] == 0  # nothing to do


def test_accept_check(built_library):
    base = dict(logits=4096, tokens=4096, tree_mask=4096, cu_seqlens=4096, path=4096, counts=4096, next_tokens=4096, workspace=4096,
                workspace_bytes=1 << 40, logits_stride=1000, mask_stride=1, dtype=_lib.DTYPE_BF16, rows=9, cols=1000, batch=2, mask_words=1,
                max_nodes=6)
    assert _lib.accept_check(_set(_lib.AcceptArgs, base, {}))[0] == 0
    for kw, code, word in [
            (dict(dtype=7), -1, "dtype"), (dict(cols=0), -1, "empty"), (dict(logits=0), -1, "logits"), (dict(logits_stride=999), -1, "logits_stride"),
            (dict(logits=4097), -1, "aligned"), (dict(rows=-1), -1, "negative"), (dict(batch=-1), -1, "negative"), (dict(path=0), -1, "path"),
            (dict(tokens=0), -1, "tokens"), (dict(max_nodes=300, mask_words=4, mask_stride=4), -2, "drafts"), (dict(max_nodes=65), -1, "mask_words"),
            (dict(mask_words=5, mask_stride=5), -1, "mask_words"), (dict(mask_stride=0), -1, "mask_stride"), (dict(batch=70000), -2, "sequences"),
            (dict(cols=1 << 21, logits_stride=1 << 21), -2, "columns"), (dict(rows=1 << 21), -2, "rows"), (dict(workspace=0), -1, "workspace"),
            (dict(workspace_bytes=100), -1, "workspace_bytes"), (dict(workspace=4100), -1, "aligned")]:
        rc, msg = _lib.accept_check(_set(_lib.AcceptArgs, base, kw))
        assert rc == code and word in msg, (kw, rc, msg)
    _lib.accept(_set(_lib.AcceptArgs, base, dict(batch=0, cu_seqlens=0)), 0)  # empty: no-op
    assert _lib.accept_check(_set(_lib.AcceptArgs, base, dict(rows=0, logits=0, tokens=0, tree_mask=0, workspace=0)))[0] == 0


def test_beam_check(built_library):
    base = dict(logits=4096, scores=4096, out_scores=4096, out_beams=4096, out_tokens=4096, workspace=4096, workspace_bytes=1 << 40,
                logits_stride=1000, dtype=_lib.DTYPE_FP16, batch=2, beams=4, cols=1000, num=8)
    assert _lib.beam_check(_set(_lib.BeamArgs, base, {}))[0] == 0
    for kw, code, word in [
            (dict(beams=0), -2, "beams"), (dict(beams=65), -2, "beams"), (dict(num=0), -2, "candidates"), (dict(num=65), -2, "candidates"),
            (dict(batch=-1), -1, "negative"), (dict(cols=0), -1, "empty"), (dict(scores=0), -1, "scores"), (dict(out_tokens=0), -1, "outputs"),
            (dict(dtype=5), -1, "dtype"), (dict(batch=70000), -2, "sequences"), (dict(workspace_bytes=10), -1, "workspace_bytes"),
            (dict(beams=64, cols=1 << 20, logits_stride=1 << 20), -2, "chunks")]:
        rc, msg = _lib.beam_check(_set(_lib.BeamArgs, base, kw))
        assert rc == code and word in msg, (kw, rc, msg)
    _lib.beam(_set(_lib.BeamArgs, base, dict(batch=0, logits=0)), 0)


def test_kv_rows_check(built_library):
    base = dict(k_cache=4096, v_cache=4096, block_tables=4096, seq_lens=4096, index=4096, counts=4096, k_stride=(65536, 4096, 256, 64),
                v_stride=(65536, 4096, 256, 64), block_table_stride=8, index_stride=4, elem_bytes=2, layers=2, batch=3, heads_kv=4, head_dim=64,
                block_size=16, num_blocks=16, max_blocks_per_seq=8, width=4)
    both = [
        (dict(elem_bytes=3), -1, "elem_bytes"), (dict(head_dim=60), -2, "head_dim"), (dict(head_dim=2048), -2, "head_dim"),
        (dict(block_size=24), -2, "block_size"), (dict(k_stride=(65536, 4096, 256, 60)), -2, "strides"), (dict(v_stride=(65536, -4096, 256, 64)), -2, "strides"),
        (dict(k_cache=4104), -2, "aligned"), (dict(kv_scales=4097), -2, "kv_scales"), (dict(block_table_stride=7), -1, "block_table_stride"),
        (dict(index_stride=3), -1, "index_stride"), (dict(batch=70000), -2, "sequences"), (dict(layers=-1), -1, "negative"),
        (dict(max_blocks_per_seq=1 << 27, block_table_stride=1 << 27), -2, "tokens"), (dict(index=0), -1, "index"), (dict(k_cache=0), -1, "k_cache")]
    for check, more in ((_lib.kv_keep_check, [(dict(counts=0), -1, "counts")]),
                        (_lib.kv_reorder_check, [(dict(width=65, index_stride=65), -2, "beams"), (dict(layers=5000), -2, "rows")])):
        assert check(_set(_lib.KvRowsArgs, base, {}))[0] == 0
        for kw, code, word in both + more:
            rc, msg = check(_set(_lib.KvRowsArgs, base, kw))
            assert rc == code and word in msg, (kw, rc, msg)
    assert _lib.kv_reorder_check(_set(_lib.KvRowsArgs, base, dict(counts=0)))[0] == 0
    for call in (_lib.kv_keep, _lib.kv_reorder):
        for kw in (dict(layers=0), dict(batch=0), dict(width=0)):
            call(_set(_lib.KvRowsArgs, base, kw), 0)
