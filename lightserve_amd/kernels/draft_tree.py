"""Trees of drafted tokens over a paged KV cache on MI355X: one step that verifies several drafts per sequence.

The reference decodes one token per sequence and step (model/cuda_graph_decode.py:114, :145). With drafts (from a smaller model,
or from the text so far) a step takes a tree of them per sequence: node 0 is the last certain token, every other node a
draft that continues an earlier node. All nodes' K and V rows are cached behind the sequence's tokens (as kv_cache_append
or apply_rope_ store a chunk's), at the rotary positions of their depth, and then:

    tree_mask, depth = draft_tree(parents)            # once for a tree's shape (host)

    o = paged_tree_attention(q, k_cache, v_cache, block_tables, cu_seqlens_q, seq_lens_k, tree_mask, *, max_nodes=None,
                             sm_scale=None, return_lse=False, kv_scales=None, window=None, sinks=0)
    path, counts, next_tokens = accept_drafts(logits, tokens, tree_mask, cu_seqlens, *, max_nodes=None, seq_lens=None)
    kv_cache_keep(k_cache, v_cache, block_tables, seq_lens, path, counts, *, kv_scales=None)

tree_mask is int64 [total_q, words]: bit j of a row (word j // 64, bit j % 64) says that the node sees node j of its sequence;
bits past the sequence's nodes say nothing.
paged_tree_attention takes the arguments of paged_prefill (paged_attention.py): seq_lens_k counts each sequence's cached
keys with its n nodes, which are the last n. A node sees all keys before those, under a window the ones that a query
at position seq_len - n + (nodes it sees) - 1 sees, and the nodes of its mask, whatever the window: a tree less deep than the window is
what its tokens are one by one, while in a deeper one nodes see ancestors that a single token's window would leave out. Any mask does; a node that
sees nothing gets o = 0 and lse = -inf. A length may pass the block table, as where a tree is longer than what is left of a cache: the
nodes stand where the length says, and nobody sees the rows that the table does not have, so that a node's o is right as long as its
own row and its ancestors' are cached. Sequences may have 0 to 256 nodes each; max_nodes bounds them (read from cu_seqlens_q
when None, a device sync, so pass it under graph capture); o's rows behind the last sequence, and of nodes past max_nodes, are
not written. 8- and 16-bit caches, bf16 and fp16, head dims that are multiples of
16 (8 over 16-bit caches) up to 128, power-of-two block sizes of at least 16.

accept_drafts takes the logits [total, vocab] (fp32, fp16 or bf16) and the tokens int64 [total] of all nodes. The path of a sequence begins at its
node 0 and goes on, from node i, to the lowest node j > i that sees what i sees and itself and whose token is i's greedy
choice (greedy_next_token's: NaN above all, ties to the lower index). It returns path int32 [batch, max_nodes] (-1
behind the path), counts int32 [batch] and next_tokens int64 [batch], the choice after the path's last node. A sequence without
nodes has count 0 and next token -1. A node whose mask is 0 follows no other: so drafts whose rows the cache does not hold, whose logits mean
nothing, are kept off the paths. seq_lens, when given, grows by counts in the same launch.

kv_cache_keep moves rows inside the cache: row start + keep[b, i] becomes row start + i for i < counts[b], start = seq_lens[b] -
counts[b] (seq_lens counts what is cached once the rows are kept, as accept_drafts leaves it; counts are held to 0 .. keep's width). Entries with keep[b, i] <= i stay where they
are, and so do rows that the block table or the cache does not have. keep may have any width and need not be a path: with
it a sequence drops rows from its middle, too. Caches are [num_blocks, block_size, heads_kv, head_dim] in any of fp32, bf16,
fp16 or 8 bits with kv_scales (quantized_kv_cache.py), or the same for all layers as one tensor [layers, ...]: one launch. Sequences must not share
blocks that hold rows from start on.
"""
import torch

from .. import _lib
from .paged_attention import windowed_attention
from .quantized_kv_cache import check_device
from .tiled_matmul import stream_workspace

MAX_NODES = 256  # LSFA_TREE_MAX_NODES
_I32, _I64 = torch.int32, torch.int64
_ELEMENTS = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2, torch.float8_e4m3fn: 1}


def draft_tree(parents, words=None):
    """The mask int64 [n, words] and depths int32 [n] of a tree, on the CPU. parents[i] < i is the node that node i continues, -1 for
    node 0; words (default: as many as n needs) is the width of a batch's masks."""
    parents = [int(p) for p in parents]
    assert len(parents) <= MAX_NODES, f"at most {MAX_NODES} nodes"
    need = max(1, (len(parents) + 63) // 64)
    words = need if words is None else words
    assert need <= words <= MAX_NODES // 64, "words must hold a bit for each node"
    seen, depth = [], []
    for i, p in enumerate(parents):
        assert (p == -1 and i == 0) or 0 <= p < i, "node 0 has no parent (-1), the others one before them"
        seen.append((seen[p] if i else 0) | 1 << i)
        depth.append(depth[p] + 1 if i else 0)
    signed = [[((m >> 64 * w) + (1 << 63)) % (1 << 64) - (1 << 63) for w in range(words)] for m in seen]
    return torch.tensor(signed, dtype=_I64).view(-1, words), torch.tensor(depth, dtype=_I32)


def _check_mask(tree_mask, total):
    assert tree_mask.dtype == _I64 and tree_mask.dim() == 2 and tree_mask.shape[0] == total and \
        1 <= tree_mask.shape[1] <= MAX_NODES // 64, f"tree_mask must be int64 [total, words] of 1 to {MAX_NODES // 64} words"
    return tree_mask if tree_mask.stride(1) == 1 and tree_mask.stride(0) >= tree_mask.shape[1] else _lib.packed(tree_mask)


def _longest(cu):
    return int((cu[1:] - cu[:-1]).max().item()) if cu.numel() > 1 else 0


def _check_nodes(max_nodes, tree_mask):
    assert 0 <= max_nodes <= MAX_NODES, f"0 to {MAX_NODES} nodes a sequence"
    assert max_nodes <= 64 * tree_mask.shape[1], "tree_mask must hold a bit for each of max_nodes nodes"


def paged_tree_attention(q, k_cache, v_cache, block_tables, cu_seqlens_q, seq_lens_k, tree_mask, *, max_nodes=None,
                         sm_scale=None, return_lse=False, kv_scales=None, window=None, sinks=0):
    assert q.dim() == 3, "q must be packed [total_q, heads_q, head_dim]"
    tree_mask = _check_mask(tree_mask, q.shape[0])
    if max_nodes is None:
        max_nodes = _longest(cu_seqlens_q)
    _check_nodes(max_nodes, tree_mask)
    keys = block_tables.shape[-1] * k_cache.shape[1] if k_cache.dim() == 4 else 0
    got = windowed_attention(q, k_cache, v_cache, block_tables, cu_seqlens_q, seq_lens_k, max_nodes, keys, True, sm_scale, return_lse,
                             kv_scales, window, sinks, tree_mask)
    return (got[0], got[1].t()) if return_lse else got


def launch_with_workspace(device, args, size, call):
    """One launch on the device's current stream that keeps arrival counters and partial results in the stream's workspace."""
    nbytes = size(args)
    with _lib.device_guard(device):
        stream = _lib.current_stream(device)
        if nbytes == 0:
            call(args, stream)
            return
        ws, launching = stream_workspace(device, stream, nbytes)
        args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
        with launching:
            call(args, stream)


def accept_drafts(logits, tokens, tree_mask, cu_seqlens, *, max_nodes=None, seq_lens=None):
    assert logits.dim() == 2 and logits.dtype in _lib.TORCH_TO_LSFA, "logits must be [total, vocab] in fp32, fp16 or bf16"
    total, vocab = logits.shape
    assert tokens.dtype == _I64 and tokens.shape == (total,), "tokens must be int64 [total]"
    tree_mask = _check_mask(tree_mask, total)
    assert cu_seqlens.dtype == _I32 and cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1, "cu_seqlens must be int32 [batch + 1]"
    batch = cu_seqlens.numel() - 1
    if seq_lens is not None:
        assert seq_lens.dtype == _I32 and seq_lens.shape == (batch,) and (batch == 0 or seq_lens.is_contiguous()), \
            "seq_lens must be contiguous int32 [batch]"
    assert total == 0 or vocab > 0, "the vocabulary must not be empty"
    on = logits.get_device()
    if not (on >= 0 and on == tokens.get_device() == tree_mask.get_device() == cu_seqlens.get_device()
            and (seq_lens is None or seq_lens.get_device() == on)):
        check_device((("logits", logits), ("tokens", tokens), ("tree_mask", tree_mask), ("cu_seqlens", cu_seqlens),
                      *((("seq_lens", seq_lens),) if seq_lens is not None else ())))
    if max_nodes is None:
        max_nodes = _longest(cu_seqlens)
    _check_nodes(max_nodes, tree_mask)
    if total and (logits.stride(1) != 1 or logits.stride(0) < vocab):
        logits = _lib.packed(logits)
    device = logits.device
    path, counts, following = cu_seqlens.new_empty((batch, max_nodes)), cu_seqlens.new_empty(batch), tokens.new_empty(batch)
    if batch > 0:
        tokens, cu = tokens.contiguous(), cu_seqlens.contiguous()
        args = _lib.pack(
            _lib.AcceptArgs, logits.data_ptr(), tokens.data_ptr(), tree_mask.data_ptr(), cu.data_ptr(),
            seq_lens.data_ptr() if seq_lens is not None else 0, path.data_ptr(), counts.data_ptr(), following.data_ptr(), 0, 0,
            max(logits.stride(0), vocab), max(tree_mask.stride(0), tree_mask.shape[1]), _lib.TORCH_TO_LSFA[logits.dtype], total, vocab,
            batch, tree_mask.shape[1], max_nodes)
        launch_with_workspace(device, args, _lib.accept_workspace_size, _lib.accept)
    return path, counts, following


def cache_rows(call, k_cache, v_cache, kv_scales, block_tables, seq_lens, index, counts):
    """Checks of the calls that move rows inside caches of one or all layers, and the launch."""
    shape, strides = k_cache.shape, (k_cache.stride(), v_cache.stride())
    layers = len(shape) == 5
    assert len(shape) in (4, 5) and v_cache.shape == shape, \
        "k_cache and v_cache must both be [num_blocks, block_size, heads_kv, head_dim], or [layers, ...] of them"
    assert k_cache.dtype in _ELEMENTS and v_cache.dtype == k_cache.dtype, "k_cache and v_cache must share one of fp32, bf16, fp16 and e4m3"
    L, (n, bs, h, d) = shape[0] if layers else 1, shape[-4:]
    assert strides[0][-1] == 1 and strides[1][-1] == 1, "the caches' head-dim stride must be 1"
    for s in strides:
        assert min(s) > 0 or all(x > 0 or m == 1 for x, m in zip(s, shape)), "rows of the caches must not share memory"
    assert (kv_scales is None) == (k_cache.dtype != torch.float8_e4m3fn), "an 8-bit cache, and no other, has kv_scales"
    scale_layer = 0
    if kv_scales is not None:
        assert kv_scales.dtype == torch.uint8 and kv_scales.shape == (*shape[:-4], n, h, bs, 2) and \
            kv_scales.stride()[-4:] == (h * bs * 2, bs * 2, 2, 1) and (not layers or L == 1 or kv_scales.stride(0) >= n * h * bs * 2), \
            "kv_scales must be uint8 [num_blocks, heads_kv, block_size, 2], or [layers, ...], contiguous in each layer"
        scale_layer = kv_scales.stride(0) if layers else 0
    assert block_tables.dtype == _I32 and block_tables.dim() == 2, "block_tables must be int32 [rows, max_blocks]"
    on = k_cache.get_device()
    if not (on >= 0 and on == v_cache.get_device() == block_tables.get_device() == seq_lens.get_device() == index.get_device()
            and (counts is None or counts.get_device() == on) and (kv_scales is None or kv_scales.get_device() == on)):
        check_device((("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables), ("seq_lens", seq_lens),
                      ("the rows' index", index), *((("counts", counts),) if counts is not None else ()),
                      *((("kv_scales", kv_scales),) if kv_scales is not None else ())))
    batch, width = index.shape
    if batch == 0 or width == 0 or k_cache.numel() == 0:
        return
    if index.stride(1) != 1 or index.stride(0) < width:
        index = _lib.packed(index)
    ks, vs = (s if layers else (0, *s) for s in strides)
    args = _lib.pack(
        _lib.KvRowsArgs, k_cache.data_ptr(), v_cache.data_ptr(), kv_scales.data_ptr() if kv_scales is not None else 0,
        block_tables.data_ptr(), seq_lens.data_ptr(), index.data_ptr(), counts.data_ptr() if counts is not None else 0, *ks[:4], *vs[:4],
        scale_layer, max(block_tables.stride(0), block_tables.shape[1]), max(index.stride(0), width), _ELEMENTS[k_cache.dtype], L, batch,
        h, d, bs, n, block_tables.shape[1], width, 0)
    device = k_cache.device
    with _lib.device_guard(device):
        call(args, _lib.current_stream(device))


def kv_cache_keep(k_cache, v_cache, block_tables, seq_lens, keep, counts, *, kv_scales=None):
    assert keep.dtype == _I32 and keep.dim() == 2, "keep must be int32 [batch, width]"
    batch = keep.shape[0]
    assert block_tables.dim() == 2 and block_tables.shape[0] == batch, "block_tables must be int32 [batch, max_blocks]"
    assert seq_lens.dtype == _I32 and counts.dtype == _I32 and seq_lens.shape == counts.shape == (batch,), \
        "seq_lens and counts must be int32 [batch]"
    cache_rows(_lib.kv_keep, k_cache, v_cache, kv_scales, _lib.table_rows(block_tables), seq_lens.contiguous(), keep, counts.contiguous())
