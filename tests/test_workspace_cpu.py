"""The skinny GEMM's workspaces under graph capture, with the captures played
on the host: which buffer a call gets and what was filled for it."""
import pytest
import torch

from lightserve_amd import _lib
from lightserve_amd.kernels import tiled_matmul as tm

STREAM, CPU = 7, torch.device("cpu")


@pytest.fixture
def capture(monkeypatch):
    """capture(id): the stream captures from now on (0: it does not)."""
    now = [0]
    monkeypatch.setattr(_lib, "capture_id", lambda stream: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] != 0)
    tm.release_workspaces()
    yield lambda n: now.__setitem__(0, n)
    tm.release_workspaces()


def _use(nbytes=1 << 20):
    """One product: the counters it finds, and what it leaves beside them."""
    ws = tm._workspace(CPU, STREAM, nbytes)
    assert ws.numel() >= nbytes
    return ws


def _clean(ws):
    return bool((ws[:_lib.GEMV_COUNTER_BYTES] == 0).all())


@pytest.mark.parametrize("eager_first", [True, False])
def test_a_capture_shares_with_nothing(capture, eager_first):
    if eager_first:
        assert _use() is _use()
    capture(1)
    first = _use()
    assert first is _use() and _clean(first)
    first[:_lib.GEMV_COUNTER_BYTES] = 5  # nothing that a capture records has run
    capture(2)
    second = _use()
    assert second is not first and second is _use() and _clean(second)
    second[:_lib.GEMV_COUNTER_BYTES] = 5
    capture(0)
    eager = _use()
    assert eager is not first and eager is not second and eager is _use() and _clean(eager)


def test_growth_inside_a_capture_is_filled(capture):
    capture(3)
    small = _use()
    big = _use(small.numel() + 1)
    assert big is not small and _clean(big) and big is _use()


def test_the_cache_keeps_one_workspace_per_capture_stream(capture):
    import weakref
    seen = []
    for n in range(1, 6):
        capture(n)
        seen.append(weakref.ref(_use()))
    assert [r() is not None for r in seen] == [False] * 4 + [True]


@pytest.fixture
def played(built_library, capture, monkeypatch):
    """Calls on CPU tensors up to their launches: played(launch) puts launch(args, stream) in the library's place."""
    import contextlib

    def put(launch, stream=lambda device: STREAM):
        monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
        monkeypatch.setattr(_lib, "device_guard", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(_lib, "current_stream", stream)
        for name in ("window", "gemv"):
            monkeypatch.setattr(_lib, name, launch)
    return put


def _products_and_attention():
    """A skinny product, and calls of windowed attention whose partial results a second launch merges (key splits of a chunk,
    long runs of a decode step)."""
    from lightserve_amd.kernels.paged_attention import paged_attention_decode, paged_prefill
    x, w = torch.zeros(1, 256, dtype=torch.bfloat16), torch.zeros(256, 256, dtype=torch.bfloat16)
    cache = torch.zeros(1, 16, 8, 64, dtype=torch.bfloat16)
    table, q = torch.zeros(2, 2048, dtype=torch.int32), torch.zeros(64, 16, 64, dtype=torch.bfloat16)
    lens, cu = torch.tensor([30000, 30000], dtype=torch.int32), torch.tensor([0, 32, 64], dtype=torch.int32)
    return [lambda: tm.skinny_matmul(x, w),
            lambda: paged_prefill(q, cache, cache, table, cu, lens, max_seqlen_q=32, window=30000),
            lambda: paged_attention_decode(q[:2], cache, cache, table, lens, max_seq_len=30000, window=30000)]


def test_threads_on_one_stream_keep_a_calls_launches_together(played):
    """What one call's first launch leaves in the stream's workspace is its second launch's: no other call that uses the
    workspace is launched in between."""
    import threading
    import time
    log = []

    def launch(args, stream):
        assert args.workspace
        log.append(("first launch", threading.get_ident()))
        time.sleep(0.002)
        log.append(("second launch", threading.get_ident()))

    played(launch)
    threads = [threading.Thread(target=call) for call in _products_and_attention() * 4]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(log) == 2 * len(threads)
    assert all(a[1] == b[1] and a[0] != b[0] for a, b in zip(log[::2], log[1::2])), "another call's launch in between"


def test_threads_on_streams_of_their_own_do_not_wait(played):
    """Two calls on two streams can be in the middle of their launches at the same time."""
    import threading
    meet, met = threading.Barrier(2), []

    def launch(args, stream):
        meet.wait(timeout=20)
        met.append(args.workspace)

    played(launch, stream=lambda device: threading.get_ident())
    threads = [threading.Thread(target=call) for call in _products_and_attention()[1:]]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(met)) == 2


def test_a_workspace_that_the_cache_has_no_room_for(capture):
    """More streams with a captured graph than the cache keeps: an eager call on another stream still gets a workspace and its
    lock, which it can take twice (a finalizer or signal handler may make a call of its own)."""
    for n in range(tm.MAX_CACHED_STREAMS):
        capture(n + 1)
        tm._workspace(CPU, 100 + n, 1 << 20)
    capture(0)
    first, launching = tm.stream_workspace(CPU, STREAM, 1 << 20)
    again, other = tm.stream_workspace(CPU, STREAM, 1 << 20)
    assert _clean(first) and _clean(again) and (first is again) == (launching is other)
    with launching, launching:
        pass
