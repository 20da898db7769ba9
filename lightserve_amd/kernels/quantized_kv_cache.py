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
sequences of one call must not write to the same slot, and it takes fewer than
2^28 rows (tokens * heads_kv; 2^29 up to head_dim 64). kv_cache_read returns
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


_E4M3, _U8, _I32 = torch.float8_e4m3fn, torch.uint8, torch.int32


def check_quantized(k_cache, v_cache, kv_scales):
    """What a cache must be, for the calls here and for the attention over it; its shape."""
    shape = k_cache.shape
    assert k_cache.dtype == _E4M3 and v_cache.dtype == _E4M3, "an 8-bit cache holds float8_e4m3fn"
    assert len(shape) == 4 and v_cache.shape == shape, \
        "k_cache and v_cache must both be [num_blocks, block_size, heads_kv, head_dim]"
    n, bs, h, _ = shape
    assert kv_scales.dtype == _U8 and kv_scales.shape == (n, h, bs, 2) and kv_scales.is_contiguous(), \
        "kv_scales must be contiguous uint8 [num_blocks, heads_kv, block_size, 2]"
    assert k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "the caches' head-dim stride must be 1"
    return shape


def check_device(named):
    """All of these ((name, tensor), ...) on one GPU."""
    for name, t in named:
        assert t.is_cuda and t.device == named[0][1].device, f"{name} must be a GPU tensor on {named[0][0]}'s device"


def _launch(call, k, v, k_cache, v_cache, kv_scales, shape, block_tables, seq_lens, cu_seqlens):
    """The launch of one of the two calls on checked arguments; k and v are contiguous in head_dim."""
    bt = _lib.table_rows(block_tables)
    kc, vc = k_cache.stride(), v_cache.stride()
    ks, vs = k.stride(), v.stride()
    rows, max_blocks = bt.shape
    args = _lib.pack(
        _lib.KvCacheArgs, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), kv_scales.data_ptr(),
        bt.data_ptr(), seq_lens.data_ptr() if seq_lens is not None else 0,
        cu_seqlens.data_ptr() if cu_seqlens is not None else 0, ks[0], ks[1], vs[0], vs[1], kc[0], kc[1], kc[2], vc[0],
        vc[1], vc[2], bt.stride(0), _lib.TORCH_TO_LSFA[k.dtype], rows, k.shape[0], shape[2], shape[3], shape[1], shape[0],
        max_blocks)
    device = k.device
    with _lib.device_guard(device):
        call(args, _lib.current_stream(device))


def _addressable(t):
    s0, s1, s2 = t.stride()
    per16 = 16 // t.element_size()
    return s2 == 1 and s0 % per16 == 0 and s1 % per16 == 0 and t.data_ptr() % 16 == 0


def kv_cache_append(k, v, k_cache, v_cache, kv_scales, block_tables, seq_lens, cu_seqlens=None):
    rows = k.shape
    assert len(rows) == 3 and v.shape == rows and v.dtype == k.dtype, "k and v must both be [tokens, heads_kv, head_dim]"
    assert k.dtype in _lib.TORCH_TO_LSFA, f"unsupported dtype {k.dtype}"
    shape = check_quantized(k_cache, v_cache, kv_scales)
    assert block_tables.dtype == _I32 and block_tables.dim() == 2, "block_tables must be int32 [batch, max_blocks]"
    on = k_cache.get_device()
    if not (on >= 0 and on == v_cache.get_device() == kv_scales.get_device() == block_tables.get_device()
            == k.get_device() == v.get_device() == seq_lens.get_device()
            and (cu_seqlens is None or cu_seqlens.get_device() == on)):
        check_device((("k_cache", k_cache), ("v_cache", v_cache), ("kv_scales", kv_scales), ("block_tables", block_tables),
                      ("k", k), ("v", v), ("seq_lens", seq_lens),
                      *((("cu_seqlens", cu_seqlens),) if cu_seqlens is not None else ())))
    assert rows[1:] == shape[2:], "heads_kv / head_dim of k and of the caches differ"
    batch = block_tables.shape[0]
    assert seq_lens.dtype == _I32 and seq_lens.shape == (batch,), "seq_lens must be int32 [batch]"
    if cu_seqlens is None:
        assert rows[0] == batch, "without cu_seqlens k and v hold one row per sequence"
    else:
        assert cu_seqlens.dtype == _I32 and cu_seqlens.shape == (batch + 1,), "cu_seqlens must be int32 [batch + 1]"
        cu_seqlens = cu_seqlens.contiguous()
    if rows[0] == 0:
        return
    if not _addressable(k):
        k = _lib.packed(k)
    if not _addressable(v):
        v = _lib.packed(v)
    _launch(_lib.kv_append, k, v, k_cache, v_cache, kv_scales, shape, block_tables, seq_lens.contiguous(), cu_seqlens)


def kv_cache_read(k_cache, v_cache, kv_scales, block_tables, cu_seqlens, *, total=None, dtype=torch.bfloat16):
    shape = check_quantized(k_cache, v_cache, kv_scales)
    assert block_tables.dtype == _I32 and block_tables.dim() == 2, "block_tables must be int32 [batch, max_blocks]"
    on = k_cache.get_device()
    if not (on >= 0 and on == v_cache.get_device() == kv_scales.get_device() == block_tables.get_device()
            == cu_seqlens.get_device()):
        check_device((("k_cache", k_cache), ("v_cache", v_cache), ("kv_scales", kv_scales), ("block_tables", block_tables),
                      ("cu_seqlens", cu_seqlens)))
    assert dtype in _lib.TORCH_TO_LSFA, f"unsupported dtype {dtype}"
    batch = block_tables.shape[0]
    assert cu_seqlens.dtype == _I32 and cu_seqlens.shape == (batch + 1,), "cu_seqlens must be int32 [batch + 1]"
    if total is None:
        total = int(cu_seqlens[-1].item())
    assert total >= 0, "total must not be negative"
    k = torch.empty((total, shape[2], shape[3]), dtype=dtype, device=k_cache.device)
    v = torch.empty_like(k)
    if total > 0:
        _launch(_lib.kv_read, k, v, k_cache, v_cache, kv_scales, shape, block_tables, None, cu_seqlens.contiguous())
    return k, v
