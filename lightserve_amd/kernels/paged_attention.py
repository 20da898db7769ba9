"""Paged-KV decode attention on MI355X: one new query token per sequence
against a KV cache addressed through block tables.

The reference has no such kernel. Its engine keeps the block tables
(engine/block_manager.py:56-60: entry i of a request's table holds tokens
[i*block_size, (i+1)*block_size)) and documents decode attention as the
missing piece (engine/README.md, "No decode-shaped attention kernel": Nq = 1
against a paged Nkv; engine/request.py is_prefill). A cache block holds
block_size x n_kv_heads x head_dim elements per layer for K and for V
(engine/config.py:5-7), so the caches here are
[num_blocks, block_size, heads_kv, head_dim].

    paged_attention_decode(q, k_cache, v_cache, block_tables, seq_lens, *,
                           max_seq_len=None, sm_scale=None, return_lse=False)

q is [batch, heads_q, head_dim]; block_tables int32 [batch, max_blocks];
seq_lens int32 [batch] counts each sequence's cached tokens (the new token's
K/V already written). Query head h reads KV head h // (heads_q // heads_kv).
Returns o like q (and lse fp32 [batch, heads_q], natural log, when asked).
max_seq_len bounds seq_lens and sets how sequences are split across
workgroups; when it is None it is read from seq_lens (a device sync, so pass
it under graph capture).

    paged_prefill(q, k_cache, v_cache, block_tables, cu_seqlens_q, seq_lens_k, *,
                  max_seqlen_q=None, causal=True, sm_scale=None, return_lse=False)

Chunked prefill against the same cache: the engine's scheduled-tokens > 1
path, which its scheduler documents as missing (engine/request.py:86-93,
engine/scheduler.py:34-44). q is packed [total_q, heads_q, head_dim] with
sequence b owning rows cu_seqlens_q[b] .. cu_seqlens_q[b+1]-1 (a chunk of
new tokens); seq_lens_k int32 [batch] counts the sequence's cached keys
with the chunk's own K/V already written. Causal masking is bottom-right
aligned: chunk query i of n sits at position seq_lens_k[b] - n + i. Returns
o like q (and lse fp32 [heads_q, total_q] when asked); block_size must be a
power of two of at least 16. One launch of the forward kernel with its K/V
tiles gathered through the block tables.

Both calls take three more keyword arguments:

    kv_scales=None   the caches are 8-bit ones (quantized_kv_cache.py) with these scales
    window=None      sliding window: a query at position p sees keys j > p - window ...
    sinks=0          ... and the sequence's first `sinks` keys (attention sinks)

A window is causal and counts the query's own token. Blocks that hold only keys
which no query of the call sees are not read, so their table entries may be
anything (an engine can give those blocks back). These calls need a
power-of-two block_size of at least 16 (any heads_q / heads_kv) and, over 8-bit
caches, a head_dim that is a multiple of 16. A query that sees no key gets o = 0
and lse = -inf. Infinities and NaN in the cache reach only the queries that see
their keys. fp16 queries need rows of an 8-bit cache that fp16 holds (those
appended in fp16 always are; the values are fp16 in the products, except that
a decode step or a chunk of up to 32 rows a KV head multiplies K's scales in fp32).
"""
import math

import torch

from .. import _lib
from .flash_attention import SPLIT_MAX_TILES, SPLIT_MIN_KEYS
from .quantized_kv_cache import check_device, check_quantized
from .tiled_matmul import stream_workspace


def windowed_attention(q, k_cache, v_cache, block_tables, cu_seqlens_q, seq_lens, max_seqlen_q, max_seq_len, causal, sm_scale,
                       return_lse, kv_scales, window, sinks, tree_mask=None):
    """Attention over an 8-bit cache or under a window (lsfa_window), or of draft trees (lsfa_tree, with a checked
    tree_mask); the lse is [tokens, heads_q]."""
    rows, dtype = q.shape, q.dtype
    assert len(rows) == 3, "q must be [tokens, heads_q, head_dim]"
    assert dtype == torch.bfloat16 or dtype == torch.float16, "windowed paged attention supports bf16 and fp16"
    if kv_scales is not None:
        shape = check_quantized(k_cache, v_cache, kv_scales)
    else:
        shape = k_cache.shape
        assert len(shape) == 4 and v_cache.shape == shape, \
            "k_cache and v_cache must both be [num_blocks, block_size, heads_kv, head_dim]"
        assert dtype == k_cache.dtype == v_cache.dtype, "q, k_cache and v_cache must share a dtype (or give kv_scales)"
        assert k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the caches' head-dim stride must be 1"
    T, Hq, D = rows
    num_blocks, block_size, Hkv, _ = shape
    assert D == shape[3], "head_dim of q and of the caches differ"
    assert Hq % Hkv == 0, "heads_q must be a multiple of heads_kv"
    assert block_tables.dim() == 2 and block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32, \
        "block_tables [batch, max_blocks] and the sequence lengths must be int32"
    B, max_blocks = block_tables.shape
    assert seq_lens.shape == (B,), "the sequence lengths must be [batch]"
    if cu_seqlens_q is None:
        assert T == B, "block_tables must be [batch, max_blocks]"
    else:
        assert cu_seqlens_q.dtype == torch.int32 and cu_seqlens_q.shape == (B + 1,), "cu_seqlens_q must be int32 [batch + 1]"
    on = q.get_device()
    if not (on >= 0 and on == k_cache.get_device() == v_cache.get_device() == block_tables.get_device()
            == seq_lens.get_device() and (cu_seqlens_q is None or cu_seqlens_q.get_device() == on)
            and (kv_scales is None or kv_scales.get_device() == on) and (tree_mask is None or tree_mask.get_device() == on)):
        check_device((("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables),
                      ("seq_lens", seq_lens), *((("cu_seqlens_q", cu_seqlens_q),) if cu_seqlens_q is not None else ()),
                      *((("kv_scales", kv_scales),) if kv_scales is not None else ()),
                      *((("tree_mask", tree_mask),) if tree_mask is not None else ())))
    if window is None:
        assert sinks == 0, "sinks need a window"
    else:
        assert window >= 1 and sinks >= 0, "window must be at least 1 and sinks not negative"
        assert causal, "a window is causal"
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    qs = q.stride()
    if qs[2] != 1 or qs[0] % 8 != 0 or qs[1] % 8 != 0 or q.data_ptr() % 16 != 0:
        q = _lib.packed(q)
        qs = q.stride()
    bt = _lib.table_rows(block_tables)
    sl = seq_lens.contiguous()
    cu = cu_seqlens_q.contiguous() if cu_seqlens_q is not None else None
    device = q.device
    o = torch.empty(rows, device=device, dtype=dtype)
    lse, ls = None, (0, 0)
    if return_lse:
        lse = torch.empty((T, Hq) if cu is None else (Hq, T), device=device, dtype=torch.float32)
        if cu is not None:
            lse = lse.t()
        ls = lse.stride()
    if T > 0:
        keys = min(int(max_seq_len), max_blocks * block_size)
        ks, vs = k_cache.stride(), v_cache.stride()
        fields = (
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(),
            lse.data_ptr() if return_lse else 0, kv_scales.data_ptr() if kv_scales is not None else 0,
            cu.data_ptr() if cu is not None else 0, sl.data_ptr(), bt.data_ptr(), 0, 0,  # the workspace follows
            qs[0], qs[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], Hq * D, D, ls[0], ls[1], bt.stride(0),
            _lib.TORCH_TO_LSFA[dtype], B, T, Hq, Hkv, D, block_size, num_blocks, max_blocks, int(max_seqlen_q), keys,
            bool(causal),
            # a window or sinks past the longest sequence say no more than its length (a tree's length may pass the table's keys)
            0 if window is None else min(int(window), keys + 1 if tree_mask is None else 1 << 30), min(int(sinks), keys), scale, 0)
        if tree_mask is None:
            args = _lib.pack(_lib.WindowArgs, *fields)
            size, launch = _lib.window_workspace_size, _lib.window
        else:
            args = _lib.pack(_lib.TreeArgs, *fields, tree_mask.data_ptr(), max(tree_mask.stride(0), tree_mask.shape[1]),
                             tree_mask.shape[1], 0)
            size, launch = _lib.tree_workspace_size, _lib.tree
        nbytes = size(args)
        with _lib.device_guard(device):
            stream = _lib.current_stream(device)
            if nbytes > 0:  # arrival counters, kept at zero from call to call, and partial results
                ws, launching = stream_workspace(device, stream, nbytes)
                args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
                with launching:
                    launch(args, stream)
            else:
                launch(args, stream)
    return (o, lse) if return_lse else o


def _check(q, k_cache, v_cache, block_tables, seq_lens):
    assert q.dim() == 3, "q must be [batch, heads_q, head_dim]"
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape, \
        "k_cache and v_cache must both be [num_blocks, block_size, heads_kv, head_dim]"
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables),
                    ("seq_lens", seq_lens)):
        assert t.is_cuda, f"{name} must be a GPU tensor"
    assert q.dtype == k_cache.dtype == v_cache.dtype, "q, k_cache and v_cache must share a dtype"
    assert q.dtype in (torch.float16, torch.bfloat16), "paged decode supports bf16 and fp16"
    assert block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32, \
        "block_tables and seq_lens must be int32"
    assert block_tables.dim() == 2 and block_tables.shape[0] == q.shape[0], "block_tables must be [batch, max_blocks]"
    assert seq_lens.shape == (q.shape[0],), "seq_lens must be [batch]"
    assert q.shape[2] == k_cache.shape[3], "head_dim of q and of the caches differ"
    assert q.shape[1] % k_cache.shape[2] == 0, "heads_q must be a multiple of heads_kv"


def paged_attention_decode(q, k_cache, v_cache, block_tables, seq_lens, *, max_seq_len=None, sm_scale=None,
                           return_lse=False, kv_scales=None, window=None, sinks=0):
    if kv_scales is not None or window is not None or sinks != 0:
        if max_seq_len is None:
            max_seq_len = int(seq_lens.max().item()) if seq_lens.numel() > 0 else 0
        return windowed_attention(q, k_cache, v_cache, block_tables, None, seq_lens, 1, max_seq_len, True, sm_scale, return_lse,
                         kv_scales, window, sinks)
    _check(q, k_cache, v_cache, block_tables, seq_lens)
    B, Hq, D = q.shape
    num_blocks, block_size, Hkv, _ = k_cache.shape
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    if max_seq_len is None:
        max_seq_len = int(seq_lens.max().item()) if B > 0 else 0
    q_ = q if (q.stride(-1) == 1 and all(s % 8 == 0 for s in q.stride()[:2]) and q.data_ptr() % 16 == 0) \
        else _lib.packed(q)
    bt = _lib.table_rows(block_tables)
    sl = seq_lens.contiguous()
    o = torch.empty(B, Hq, D, device=q.device, dtype=q.dtype)
    lse = torch.empty(B, Hq, device=q.device, dtype=torch.float32) if return_lse else None
    args = _lib.pack(
        _lib.DecodeArgs, q_.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(),
        lse.data_ptr() if return_lse else 0, bt.data_ptr(), sl.data_ptr(), 0, 0,  # the workspace follows
        *q_.stride(), *k_cache.stride(), *v_cache.stride(), *o.stride(), *(lse.stride() if return_lse else (0, 0)),
        bt.stride(0), _lib.TORCH_TO_LSFA[q.dtype], B, Hq, Hkv, D, block_size, num_blocks, bt.shape[1],
        int(max_seq_len), scale)
    nbytes = _lib.decode_workspace_size(args)
    ws = None
    if nbytes > 0:
        ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)  # 512-byte aligned blocks
        args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    with _lib.device_guard(q.device):
        _lib.decode(args, _lib.current_stream(q.device))
    return (o, lse) if return_lse else o


def paged_prefill(q, k_cache, v_cache, block_tables, cu_seqlens_q, seq_lens_k, *, max_seqlen_q=None, causal=True,
                  sm_scale=None, return_lse=False, kv_scales=None, window=None, sinks=0):
    if kv_scales is not None or window is not None or sinks != 0:
        if max_seqlen_q is None:
            max_seqlen_q = int((cu_seqlens_q[1:] - cu_seqlens_q[:-1]).max().item()) if cu_seqlens_q.numel() > 1 else 0
        most = block_tables.shape[-1] * k_cache.shape[1]
        got = windowed_attention(q, k_cache, v_cache, block_tables, cu_seqlens_q, seq_lens_k, max_seqlen_q, most, causal, sm_scale,
                        return_lse, kv_scales, window, sinks)
        return (got[0], got[1].t()) if return_lse else got
    assert q.dim() == 3, "q must be packed [total_q, heads_q, head_dim]"
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape, \
        "k_cache and v_cache must be [num_blocks, block_size, heads_kv, head_dim] of one shape"
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables),
                    ("cu_seqlens_q", cu_seqlens_q), ("seq_lens_k", seq_lens_k)):
        assert t.is_cuda, f"{name} must be a GPU tensor"
    assert q.dtype == k_cache.dtype == v_cache.dtype, "q, k_cache and v_cache must share a dtype"
    assert q.dtype in (torch.float16, torch.bfloat16), "paged prefill supports bf16 and fp16"
    assert block_tables.dtype == torch.int32 and cu_seqlens_q.dtype == torch.int32 and \
        seq_lens_k.dtype == torch.int32, "block_tables, cu_seqlens_q and seq_lens_k must be int32"
    assert block_tables.dim() == 2, "block_tables must be [batch, max_blocks]"
    B = block_tables.shape[0]
    assert cu_seqlens_q.shape == (B + 1,) and seq_lens_k.shape == (B,), \
        "cu_seqlens_q must be [batch + 1] and seq_lens_k [batch]"
    assert q.shape[2] == k_cache.shape[3], "head_dim of q and of the caches differ"
    assert q.shape[1] % k_cache.shape[2] == 0, "heads_q must be a multiple of heads_kv"
    T, Hq, D = q.shape
    num_blocks, block_size, Hkv, _ = k_cache.shape
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    if max_seqlen_q is None:
        max_seqlen_q = int((cu_seqlens_q[1:] - cu_seqlens_q[:-1]).max().item()) if B > 0 else 0
    q_ = q if (q.stride(-1) == 1 and all(s % 8 == 0 for s in q.stride()[:2]) and q.data_ptr() % 16 == 0) \
        else _lib.packed(q)
    assert k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the caches' head-dim stride must be 1"
    bt = _lib.table_rows(block_tables)
    cu, sl = cu_seqlens_q.contiguous(), seq_lens_k.contiguous()  # kept alive until the launch
    o = torch.empty(T, Hq, D, device=q.device, dtype=q.dtype)
    lse = torch.empty(Hq, T, device=q.device, dtype=torch.float32) if return_lse else None
    args = _lib.pack(
        _lib.PrefillPagedArgs, q_.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(),
        lse.data_ptr() if return_lse else 0, cu.data_ptr(), sl.data_ptr(), bt.data_ptr(),
        *q_.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3], *o.stride()[:2],
        *(lse.stride() if return_lse else (0, 0)), bt.stride(0), _lib.TORCH_TO_LSFA[q.dtype], B, Hq, Hkv, D,
        block_size, num_blocks, bt.shape[1], int(max_seqlen_q), bool(causal), scale, 0)
    if T > 0:
        # few query tiles for the GPU: their keys are shared out over several workgroups
        nbytes = 0
        if bt.shape[1] * block_size >= SPLIT_MIN_KEYS and B * Hq * ((args.max_seqlen_q + 127) // 128) <= SPLIT_MAX_TILES:
            nbytes = _lib.prefill_paged_workspace_size(args)
        with _lib.device_guard(q.device):
            if nbytes > 0:
                ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)  # 512-byte aligned blocks
                _lib.prefill_paged_split(args, ws.data_ptr(), nbytes, _lib.current_stream(q.device))
            else:
                _lib.prefill_paged(args, _lib.current_stream(q.device))
    return (o, lse) if return_lse else o
