"""What the calls on 8-bit caches and under a window refuse, without a GPU: the C ABI's own checks, then the Python entry points'."""
import ctypes

import pytest
import torch

from lightserve_amd import _lib
from lightserve_amd.kernels.paged_attention import paged_attention_decode, paged_prefill
from lightserve_amd.kernels.quantized_kv_cache import kv_cache_append, kv_cache_read, quantized_kv_cache

P = 1 << 20  # stands for a device address: the checks read nothing there


def _kv(**kw):
    a = _lib.KvCacheArgs(k=P, v=P, k_cache=P, v_cache=P, kv_scales=P, block_tables=P, seq_lens=P, cu_seqlens=P,
                         k_stride=(1024, 128), v_stride=(1024, 128), k_cache_stride=(16384, 1024, 128),
                         v_cache_stride=(16384, 1024, 128), block_table_stride=10, dtype=_lib.DTYPE_BF16, batch=3, tokens=20,
                         heads_kv=8, head_dim=128, block_size=16, num_blocks=30, max_blocks_per_seq=10)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def _win(**kw):
    # (one query each: the launch that shares key tiles out and so needs a workspace)
    a = _lib.WindowArgs(q=P, k_cache=P, v_cache=P, o=P, lse=P, kv_scales=P, cu_seqlens_q=P, seq_lens=P, block_tables=P,
                        workspace=P, workspace_bytes=1 << 40, q_stride=(4096, 128), k_stride=(16384, 1024, 128),
                        v_stride=(16384, 1024, 128), o_stride=(4096, 128), lse_stride=(32, 1), block_table_stride=10,
                        dtype=_lib.DTYPE_BF16, batch=3, tokens=20, heads_q=32, heads_kv=8, head_dim=128, block_size=16,
                        num_blocks=30, max_blocks_per_seq=10, max_seqlen_q=1, max_seq_len=160, causal=1, window=50, sinks=4,
                        sm_scale=0.1)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


BOTH = [(dict(head_dim=72), -2, "multiple of 16"), (dict(head_dim=144), -2, "multiple of 16"), (dict(head_dim=0), -2, "multiple"),
        (dict(block_size=8), -2, "power of two"), (dict(block_size=48), -2, "power of two"), (dict(num_blocks=-1), -1, "negative"),
        (dict(batch=-1), -1, "negative"), (dict(tokens=-1), -1, "negative"), (dict(heads_kv=0), -1, "no heads"),
        (dict(dtype=7), -1, "dtype"), (dict(block_table_stride=9), -1, "block_table_stride"), (dict(k_cache=None), -1, "non-NULL"),
        (dict(v_cache=P + 8), -2, "aligned"), (dict(kv_scales=P + 4), -2, "aligned"), (dict(block_tables=None), -1, "non-NULL"),
        (dict(max_blocks_per_seq=1 << 27, block_table_stride=1 << 27), -2, "2^30")]


@pytest.mark.parametrize("change,status,word", BOTH + [
    (dict(k_cache_stride=(16384, 1032, 128)), -2, "16 bytes"), (dict(v_cache_stride=(16384, 1 << 23, 128)), -2, "slot strides"),
    (dict(k=None), -1, "non-NULL"), (dict(v=P + 2), -2, "aligned"), (dict(k_stride=(1028, 128)), -2, "16 bytes"),
    (dict(tokens=1 << 30), -2, "rows"), (dict(kv_scales=None), -1, "non-NULL")])
def test_cache_refusals(built_library, change, status, word):
    for check in (_lib.kv_append_check, _lib.kv_read_check):
        assert check(_kv())[0] == 0
        rc, msg = check(_kv(**change))
        assert rc == status and word in msg, (rc, msg)


def test_cache_refusals_of_one_call(built_library):
    rc, msg = _lib.kv_append_check(_kv(cu_seqlens=None))
    assert rc == -1 and "20 rows for 3 sequences" in msg
    assert _lib.kv_append_check(_kv(cu_seqlens=None, tokens=3))[0] == 0
    assert _lib.kv_append_check(_kv(seq_lens=None))[0] == -1 and _lib.kv_read_check(_kv(seq_lens=None))[0] == 0
    assert _lib.kv_read_check(_kv(cu_seqlens=None))[0] == -1
    for check in (_lib.kv_append_check, _lib.kv_read_check):
        assert check(_kv(tokens=0, k=None, v=None))[0] == 0
        assert check(_kv(num_blocks=0, k_cache=None, v_cache=None, kv_scales=None))[0] == 0
        assert check(_kv(dtype=_lib.DTYPE_FP32, k_stride=(1028, 132), v_stride=(1028, 132)))[0] == 0  # 16 bytes of fp32
    assert _lib.load().lsfa_kv_append_check(None) == -1 and _lib.load().lsfa_kv_read_check(None) == -1
    assert _lib.load().lsfa_kv_append(None, None) == -1 and _lib.load().lsfa_kv_read(None, None) == -1


@pytest.mark.parametrize("change,status,word", BOTH + [
    (dict(k_stride=(16384, 1032, 128)), -2, "16 bytes"), (dict(v_stride=(16384, 1 << 23, 128)), -2, "slot strides"),
    (dict(dtype=_lib.DTYPE_FP32), -2, "bf16 and fp16"), (dict(heads_q=33), -1, "multiple of heads_kv"),
    (dict(window=-1), -1, "window"), (dict(sinks=-1), -1, "sinks"), (dict(window=0), -1, "sinks need a window"),
    (dict(causal=0), -1, "causal"), (dict(sm_scale=float("inf")), -1, "finite"), (dict(sm_scale=float("nan")), -1, "finite"),
    (dict(q=None), -1, "non-NULL"), (dict(o=None), -1, "non-NULL"), (dict(seq_lens=None), -1, "non-NULL"),
    (dict(cu_seqlens_q=None), -1, "one query"), (dict(q_stride=(4100, 128)), -2, "multiples of 8"), (dict(o=P + 8), -2, "aligned"),
    (dict(max_seq_len=-1), -1, "negative"), (dict(max_seqlen_q=-1), -1, "negative"), (dict(batch=70000), -2, "65535"),
    (dict(max_seqlen_q=1 << 26), -2, "2^30"), (dict(workspace=None), -1, "workspace"), (dict(workspace=P + 16), -1, "aligned"),
    (dict(workspace_bytes=16), -1, "below")])
def test_window_refusals(built_library, change, status, word):
    assert _lib.window_check(_win()) == (0, "")
    rc, msg = _lib.window_check(_win(**change))
    assert rc == status and word in msg, (rc, msg)


def test_window_sizes(built_library):
    """Head dims that 16-bit caches allow; nothing to do; workspaces of sizes that are refused elsewhere."""
    assert _lib.window_check(_win(kv_scales=None, head_dim=72))[0] == 0
    assert _lib.window_check(_win(kv_scales=None, head_dim=60))[0] == -2
    for nothing in (dict(batch=0), dict(tokens=0), dict(max_seqlen_q=0)):
        assert _lib.window_check(_win(workspace=None, q=None, **nothing))[0] == 0
        assert _lib.window_workspace_size(_win(**nothing)) == 0
    assert _lib.window_workspace_size(_win()) > 0
    assert _lib.load().lsfa_window_check(None) == -1 and _lib.load().lsfa_window(None, None) == -1
    n = ctypes.c_uint64(5)
    assert _lib.load().lsfa_window_workspace_size(None, ctypes.byref(n)) == -1
    assert _lib.load().lsfa_window_workspace_size(ctypes.byref(_win()), None) == -1
    for bad in (dict(heads_kv=0), dict(block_size=0), dict(head_dim=0), dict(max_seqlen_q=-3)):
        with pytest.raises(RuntimeError):
            _lib.window_workspace_size(_win(**bad))


def test_window_sizes_past_32_bits(built_library):
    """Key tiles of all sequences, tokens and windows that positions of 32 bits would not hold."""
    huge = dict(max_blocks_per_seq=1 << 26, block_table_stride=1 << 26, max_seq_len=1 << 30, window=0, sinks=0)
    assert _lib.window_check(_win(**huge, batch=31, tokens=31, workspace_bytes=1 << 40)) == (0, "")
    for change in (dict(batch=33, tokens=33), dict(batch=65535, tokens=65535)):
        rc, msg = _lib.window_check(_win(**huge, **change))
        assert rc == -2 and "tiles" in msg, (rc, msg)
    rc, msg = _lib.window_check(_win(tokens=(1 << 30) + 1, heads_q=1, heads_kv=1))
    assert rc == -2 and "tokens" in msg, (rc, msg)
    assert _lib.window_check(_win(**{**huge, "window": 4096}, batch=65535, tokens=65535)) == (0, "")
    assert _lib.window_check(_win(window=2 ** 31 - 1, workspace_bytes=1 << 40)) == (0, "")
    rc, msg = _lib.window_check(_win(block_size=1 << 27, max_blocks_per_seq=1))
    assert rc == -2 and "block" in msg, (rc, msg)


def test_struct_sizes_match_the_header(built_library, tmp_path):
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    include = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "include")
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "lightserve_fa.h"\n'
                   'int main(void){printf("%zu %zu %zu %zu %zu\\n", sizeof(lsfa_kv_cache_args), offsetof(lsfa_kv_cache_args, dtype),'
                   ' sizeof(lsfa_window_args), offsetof(lsfa_window_args, dtype), offsetof(lsfa_window_args, sm_scale)); return 0;}\n')
    subprocess.run([cc, "-I", include, str(src), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.KvCacheArgs), _lib.KvCacheArgs.dtype.offset, ctypes.sizeof(_lib.WindowArgs),
                   _lib.WindowArgs.dtype.offset, _lib.WindowArgs.sm_scale.offset]


def _tensors():
    kc, vc, sc = quantized_kv_cache(4, 16, 2, 64, device="cpu")
    return kc, vc, sc, torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.arange(3, dtype=torch.int32)


def test_an_empty_cache():
    kc, vc, sc, *_ = _tensors()
    assert kc.dtype == vc.dtype == torch.float8_e4m3fn and kc.shape == vc.shape == (4, 16, 2, 64)
    assert sc.dtype == torch.uint8 and sc.shape == (4, 2, 16, 2) and (kc.view(torch.uint8) == 0).all()
    assert kc.data_ptr() != vc.data_ptr()


def test_python_refusals_of_the_cache():
    kc, vc, sc, bt, sl, cu = _tensors()
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for args, word in (((rows, rows, kc, vc, sc, bt, sl), "GPU tensor"),
                       ((rows, rows[:1], kc, vc, sc, bt, sl), "tokens, heads_kv"),
                       ((rows, rows.float(), kc, vc, sc, bt, sl), "tokens, heads_kv"),
                       ((rows.long(), rows.long(), kc, vc, sc, bt, sl), "unsupported dtype"),
                       ((rows, rows, kc.view(torch.uint8), vc, sc, bt, sl), "float8_e4m3fn"),
                       ((rows, rows, kc, vc[:2], sc, bt, sl), "must both be"),
                       ((rows, rows, kc, vc, sc.transpose(1, 2).contiguous(), bt, sl), "kv_scales"),
                       ((rows, rows, kc, vc, sc.int(), bt, sl), "kv_scales"),
                       ((rows, rows, kc, vc, sc, bt.long(), sl), "block_tables")):
        with pytest.raises(AssertionError, match=word):
            kv_cache_append(*args)
    with pytest.raises(AssertionError, match="GPU tensor"):
        kv_cache_read(kc, vc, sc, bt, cu)
    with pytest.raises(AssertionError, match="kv_scales"):
        kv_cache_read(kc, vc, sc[:3], bt, cu)


def test_python_refusals_of_the_attention():
    kc, vc, sc, bt, sl, cu = _tensors()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    half = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)

    def decode(q=q, k=kc, v=vc, bt=bt, sl=sl, **kw):
        return paged_attention_decode(q, k, v, bt, sl, max_seq_len=16, **({"kv_scales": sc} | kw))

    def chunk(q=q, k=kc, v=vc, bt=bt, cu=cu, sl=sl, **kw):
        return paged_prefill(q, k, v, bt, cu, sl, max_seqlen_q=1, **({"kv_scales": sc} | kw))

    for call in (decode, chunk):
        for kw, word in ((dict(), "GPU tensor"), (dict(q=q.float()), "bf16 and fp16"), (dict(q=q[0]), "must be"),
                         (dict(k=half, v=half), "float8_e4m3fn"), (dict(k=half, v=half, kv_scales=None, window=3), "GPU tensor"),
                         (dict(k=half.half(), v=half.half(), kv_scales=None, window=3), "share a dtype"),
                         (dict(kv_scales=sc[:2]), "kv_scales"), (dict(q=q[:, :3]), "multiple of heads_kv"),
                         (dict(q=q[:, :, :32]), "head_dim"), (dict(bt=bt.long()), "int32"), (dict(sl=sl[:1]), "batch")):
            with pytest.raises(AssertionError, match=word):
                call(**kw)
    with pytest.raises(AssertionError, match="cu_seqlens_q"):
        chunk(cu=cu[:2])
    with pytest.raises(AssertionError, match="batch"):
        decode(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16))


@pytest.mark.parametrize("kw,word", [(dict(sinks=1), "sinks need"), (dict(window=0), "at least 1"), (dict(window=-3), "at least 1"),
                                     (dict(window=4, sinks=-1), "not negative")])
def test_window_arguments(monkeypatch, kw, word):
    """Checked after the tensors, so these stand on the GPU here in name."""
    kc, vc, sc, bt, sl, cu = _tensors()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    with pytest.raises(AssertionError, match=word):
        paged_attention_decode(q, kc, vc, bt, sl, max_seq_len=16, kv_scales=sc, **kw)
    with pytest.raises(AssertionError, match=word):
        paged_prefill(q, kc, vc, bt, cu, sl, max_seqlen_q=1, kv_scales=sc, **kw)
    with pytest.raises(AssertionError, match="causal"):
        paged_prefill(q, kc, vc, bt, cu, sl, max_seqlen_q=1, kv_scales=sc, causal=False, window=3)


@pytest.fixture
def checked(built_library, monkeypatch):
    """The calls on CPU tensors, each launch replaced by the library's own check of its arguments; the pointers of q (k for the
    append) that it got."""
    import contextlib
    at = []

    def check(name, first):
        def launch(args, stream):
            rc, message = getattr(_lib, name + "_check")(args)
            assert rc == 0, message
            at.append(getattr(args, first))
        return launch

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_lib, "device_guard", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "current_stream", lambda device: 11)
    for name, first in (("window", "q"), ("kv_append", "k"), ("decode", "q"), ("prefill_paged", "q")):
        monkeypatch.setattr(_lib, name, check(name, first))
    yield at
    from lightserve_amd.kernels import tiled_matmul
    tiled_matmul.release_workspaces()


def _all_calls(q, k, bt):
    """The append and the attentions, over 8-bit caches and older ones; a row each."""
    kc, vc, sc, _, sl, cu = _tensors()
    half = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    sl, cu = sl[:q.shape[0]], cu[:q.shape[0] + 1]
    return (lambda: kv_cache_append(k, k, kc, vc, sc, bt, sl), lambda: kv_cache_append(k, k, kc, vc, sc, bt, sl, cu),
            lambda: paged_attention_decode(q, kc, vc, bt, sl, max_seq_len=16, kv_scales=sc),
            lambda: paged_prefill(q, kc, vc, bt, cu, sl, max_seqlen_q=1, kv_scales=sc),
            lambda: paged_attention_decode(q, half, half, bt, sl, max_seq_len=16),
            lambda: paged_prefill(q, half, half, bt, cu, sl, max_seqlen_q=1))


def test_packed_rows_at_odd_addresses_are_copied(checked):
    """Tensors that are contiguous but begin between two 16-byte pieces, and single rows whose strides say nothing."""
    def shifted(*shape):
        n = torch.Size(shape).numel()
        t = torch.zeros(n + 8, dtype=torch.bfloat16)[1:n + 1].view(shape)
        assert t.is_contiguous() and t.data_ptr() % 16 != 0
        return t

    single = [torch.zeros(h * 64 + 3, dtype=torch.bfloat16).as_strided((1, h, 64), (h * 64 + 3, 64, 1)) for h in (4, 2)]
    assert all(t.is_contiguous() and t.stride(0) % 8 != 0 for t in single)
    bt = torch.zeros(2, 2, dtype=torch.int32)
    for q, k, table in ((shifted(2, 4, 64), shifted(2, 2, 64), bt), (*single, bt[:1])):
        for call in _all_calls(q, k, table):
            call()
    assert len(checked) == 12 and all(p % 16 == 0 for p in checked)


def test_tables_whose_rows_overlap_are_copied(checked):
    """A table that all sequences share (a row expanded), and one sequence's that was a column."""
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for call in _all_calls(q, k, torch.zeros(2, dtype=torch.int32).expand(2, 2)):
        call()
    for call in _all_calls(q[:1], k[:1], torch.zeros(2, 1, dtype=torch.int32).t()):
        call()
    assert len(checked) == 12


@pytest.mark.parametrize("d", [64, 60])
def test_the_dense_kernels_layout_of_odd_addresses(d):
    from lightserve_amd.kernels.flash_attention import as_kernel_layout
    t = torch.arange(2 * 3 * 5 * d + 1, dtype=torch.float32).to(torch.bfloat16)[1:].view(2, 3, 5, d)
    got = as_kernel_layout(t, 64)
    assert _lib.fast_layout_ok(got) and torch.equal(got[..., :d], t) and (got[..., d:] == 0).all()


@pytest.mark.parametrize("d,lanes", [(128, 16), (80, 16), (64, 8), (16, 8)])
def test_more_rows_than_a_launch_has_threads_for(built_library, d, lanes):
    """A launch has fewer than 2^32 threads: `lanes` a row for the append, half as many for a large read."""
    for check, rows in ((_lib.kv_append_check, (1 << 32) // lanes), (_lib.kv_read_check, (1 << 33) // lanes)):
        most = min(rows - 64, 2 ** 31 - 1)
        assert check(_kv(heads_kv=1, head_dim=d, tokens=most)) == (0, "")
        rc, msg = check(_kv(heads_kv=1, head_dim=d, tokens=min(rows, 2 ** 31 - 1)))
        assert rc == -2 and "rows" in msg, (rc, msg)


def test_more_rows_of_queries_than_a_launch_has_threads_for(built_library):
    """Two threads a (token, query head) row."""
    big = dict(kv_scales=None, window=0, sinks=0, heads_q=8, heads_kv=1, head_dim=8, batch=8, q_stride=(64, 8), o_stride=(64, 8),
               max_seqlen_q=1 << 27)
    assert _lib.window_check(_win(**big, tokens=(1 << 28) - 4096)) == (0, "")
    for call in (_lib.window_check, lambda a: _lib.window_workspace_size(a)):
        try:
            rc, msg = call(_win(**big, tokens=1 << 28))
        except RuntimeError as e:
            rc, msg = -2, str(e)
        assert rc == -2 and "threads" in msg, (rc, msg)
