"""An 8-bit paged KV cache on MI355X: K and V quantised as they are written, and read back.

The reference's engine sizes its cache for the model's own type
(engine/config.py:5-7: a block holds block_size x n_kv_heads x head_dim
elements per layer for K and for V). This cache holds one byte for each of them
and two bytes for each token and KV head:

    quantized_kv_cache(num_blocks, block_size, heads_kv, head_dim, device="cuda")
        -> k_cache, v_cache (float8_e4m3fn [num_blocks, block_size, heads_kv, head_dim]),
           kv_scales (uint8 [num_blocks, heads_kv, block_size, 2])

    kv_cache_append(k, v, k_cache, v_cache, kv_scales, block_tables, seq_lens, cu_seqlens=None)
    kv_cache_read(k_cache, v_cache, kv_scales, block_tables, cu_seqlens, *, total=None, dtype=bf16) -> k, v

paged_attention_decode and paged_prefill (paged_attention.py) read it with
kv_scales=. A row (the head_dim values of one token and KV head) stands for
code * 2^(e - 127), e = kv_scales[block, head, slot, 0] for K and [..., 1] for
V: the least power of two that brings the row's largest finite magnitude within
448, e4m3's largest value. Codes are rounded to nearest even; an infinity or NaN
becomes NaN. Where 256 * 2^(e - 127) does not fit the rows' own type (fp16 rows
above 57344, bf16 and fp32 rows above 448 * 2^119), magnitudes are held to 240 *
2^(e - 127), so that a row always reads back finite in the type it came in. A
power of two costs no precision here: e4m3's relative step does not depend on
it, and codes are exact in it.

kv_cache_append takes new rows k, v [tokens, heads_kv, head_dim] (bf16, fp16 or
fp32) with the arguments of the attention call that follows: sequence b's rows
are cu_seqlens[b] .. cu_seqlens[b+1]-1 (None: one row each, a decode step) and
its last row goes to position seq_lens[b] - 1 of block_tables int32 [batch,
max_blocks]. Rows behind the last sequence, before position 0 and in blocks
outside the cache are not stored; nothing else in the caches changes. Two
sequences of one call must not write to the same slot. kv_cache_read returns
rows 0 .. cu_seqlens[b+1] - cu_seqlens[b] - 1 of each sequence, packed as
flash_attention_varlen_forward takes them; total is the rows of the result (read
from cu_seqlens when None, a device sync, so pass it under graph capture), and
rows behind the last sequence or in no block are zeros.
"""
import torch

from .. import _lib


def quantized_kv_cache(num_blocks, block_size, heads_kv, head_dim, device="cuda"):
    """Caches of zeros."""
    k_cache, v_cache = (torch.zeros(num_blocks, block_size, heads_kv, head_dim, dtype=torch.uint8, device=device)
                        .view(torch.float8_e4m3fn) for _ in range(2))
    return k_cache, v_cache, torch.ones(num_blocks, heads_kv, block_size, 2, dtype=torch.uint8, device=device)


def check_quantized(k_cache, v_cache, kv_scales):
    """What a cache must be, for the calls here and for the attention over it."""
    assert k_cache.dtype == v_cache.dtype == torch.float8_e4m3fn, "an 8-bit cache holds float8_e4m3fn"
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape, \
        "k_cache and v_cache must both be [num_blocks, block_size, heads_kv, head_dim]"
    n, bs, h, _ = k_cache.shape
    assert kv_scales.dtype == torch.uint8 and kv_scales.shape == (n, h, bs, 2) and kv_scales.is_contiguous(), \
        "kv_scales must be contiguous uint8 [num_blocks, heads_kv, block_size, 2]"
    assert k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the caches' head-dim stride must be 1"


def _check(k_cache, v_cache, kv_scales, block_tables, others):
    check_quantized(k_cache, v_cache, kv_scales)
    assert block_tables.dtype == torch.int32 and block_tables.dim() == 2, "block_tables must be int32 [batch, max_blocks]"
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("kv_scales", kv_scales), ("block_tables", block_tables),
                    *others):
        assert t.is_cuda and t.device == k_cache.device, f"{name} must be a GPU tensor on the cache's device"


def _args(k, v, k_cache, v_cache, kv_scales, block_tables, seq_lens, cu_seqlens):
    num_blocks, block_size, heads, dim = k_cache.shape
    return _lib.pack(
        _lib.KvCacheArgs, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), kv_scales.data_ptr(),
        block_tables.data_ptr(), seq_lens.data_ptr() if seq_lens is not None else 0,
        cu_seqlens.data_ptr() if cu_seqlens is not None else 0, *k.stride()[:2], *v.stride()[:2],
        *k_cache.stride()[:3], *v_cache.stride()[:3], block_tables.stride(0), _lib.TORCH_TO_LSFA[k.dtype],
        block_tables.shape[0], k.shape[0], heads, dim, block_size, num_blocks, block_tables.shape[1])


def _addressable(t):
    per16 = 16 // t.element_size()
    return t.stride(2) == 1 and t.stride(0) % per16 == 0 and t.stride(1) % per16 == 0 and t.data_ptr() % 16 == 0


def kv_cache_append(k, v, k_cache, v_cache, kv_scales, block_tables, seq_lens, cu_seqlens=None):
    assert k.dim() == 3 and v.shape == k.shape and v.dtype == k.dtype, "k and v must both be [tokens, heads_kv, head_dim]"
    assert k.dtype in _lib.TORCH_TO_LSFA, f"unsupported dtype {k.dtype}"
    offsets = () if cu_seqlens is None else (("cu_seqlens", cu_seqlens),)
    _check(k_cache, v_cache, kv_scales, block_tables, (("k", k), ("v", v), ("seq_lens", seq_lens), *offsets))
    assert k.shape[1:] == k_cache.shape[2:], "heads_kv / head_dim of k and of the caches differ"
    batch = block_tables.shape[0]
    assert seq_lens.dtype == torch.int32 and seq_lens.shape == (batch,), "seq_lens must be int32 [batch]"
    if cu_seqlens is None:
        assert k.shape[0] == batch, "without cu_seqlens k and v hold one row per sequence"
    else:
        assert cu_seqlens.dtype == torch.int32 and cu_seqlens.shape == (batch + 1,), "cu_seqlens must be int32 [batch + 1]"
        cu_seqlens = cu_seqlens.contiguous()
    if k.shape[0] == 0:
        return
    k, v = (t if _addressable(t) else t.contiguous() for t in (k, v))
    bt = block_tables if block_tables.stride(1) == 1 else block_tables.contiguous()
    sl = seq_lens.contiguous()
    args = _args(k, v, k_cache, v_cache, kv_scales, bt, sl, cu_seqlens)
    with _lib.device_guard(k.device):
        _lib.kv_append(args, _lib.current_stream(k.device))


def kv_cache_read(k_cache, v_cache, kv_scales, block_tables, cu_seqlens, *, total=None, dtype=torch.bfloat16):
    _check(k_cache, v_cache, kv_scales, block_tables, (("cu_seqlens", cu_seqlens),))
    assert dtype in _lib.TORCH_TO_LSFA, f"unsupported dtype {dtype}"
    batch = block_tables.shape[0]
    assert cu_seqlens.dtype == torch.int32 and cu_seqlens.shape == (batch + 1,), "cu_seqlens must be int32 [batch + 1]"
    if total is None:
        total = int(cu_seqlens[-1].item())
    assert total >= 0, "total must not be negative"
    k, v = (torch.empty(total, *k_cache.shape[2:], dtype=dtype, device=k_cache.device) for _ in range(2))
    if k.numel() == 0:
        return k, v
    bt = block_tables if block_tables.stride(1) == 1 else block_tables.contiguous()
    cu = cu_seqlens.contiguous()
    args = _args(k, v, k_cache, v_cache, kv_scales, bt, None, cu)
    with _lib.device_guard(k.device):
        _lib.kv_read(args, _lib.current_stream(k.device))
    return k, v
