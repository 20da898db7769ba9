"""The oracle of the 8-bit paged cache and of windowed attention, pinned on the CPU."""
import math

import pytest
import torch

from oracle import paged8
from oracle.attention import attention_reference, paged_prefill_reference


def test_magnitudes_are_e4m3s():
    bits = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(paged8.e4m3_magnitudes(), bits.view(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_codes_are_torchs_cast_of_the_scaled_rows(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(400, 64, generator=g) * torch.exp2(torch.randint(-18, 14, (400, 1), generator=g).float())).to(dtype)
    codes, e = paged8.quantise_rows(x)
    scaled = x.double() / torch.pow(2.0, e.double() - 127)[:, None]
    assert scaled.abs().amax(-1).max() <= 448
    assert ((scaled.abs().amax(-1) > 224) | (e == 1)).all()  # half the scale would not hold the row
    assert torch.equal(codes, scaled.to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("dtype,top", [(torch.float16, 135), (torch.bfloat16, 247), (torch.float32, 247)])
def test_edges_of_a_row(dtype, top):
    big = torch.finfo(dtype).max
    x = torch.tensor([[0.0, -0.0, 0.0], [big, -big, big / 2], [448.0, 1.0, -447.0], [449 if dtype == torch.float32 else 450, 0, 0],
                      [math.inf, 2.0, 1.0], [math.nan, -math.inf, 0.0], [336.0, 1.0, 0.0]]).to(dtype)
    codes, e = paged8.quantise_rows(x)
    v = paged8.values(codes, e)
    assert e[0] == 1 and (v[0] == 0).all() and codes[0, 1] == 128
    assert e[1] == top and torch.isfinite(v[1].to(dtype)).all() and v[1, 0] == 240 * 2.0 ** (top - 127) == -v[1, 1]
    assert e[2] == 127 and v[2, 0] == 448 and v[2, 2] == -448
    assert e[3] == 128 if dtype != torch.bfloat16 else 127
    assert math.isnan(v[4, 0]) and v[4, 1] == 2 and math.isnan(v[5, 0]) and math.isnan(v[5, 1]) and v[5, 2] == 0
    assert v[6, 0] == 320  # halfway between 320 and 352: the even code


def test_append_and_read_by_hand():
    kc, vc = (torch.full((3, 4, 1, 2), 9, dtype=torch.uint8) for _ in range(2))
    sc = torch.full((3, 1, 4, 2), 100, dtype=torch.uint8)
    table = torch.tensor([[2, 0], [1, -1]], dtype=torch.int32)
    k = torch.tensor([[[448.0, 1.0]], [[2.0, 3.0]], [[5.0, 6.0]], [[7.0, 8.0]]])
    cu = torch.tensor([0, 2, 4], dtype=torch.int32)
    # sequence 0's rows at 3 and 4 (blocks 2 and 0), sequence 1's at 3 and 4 (block 1, then none)
    k2, v2, s2 = paged8.append_reference(k, -k, kc, vc, sc, table, torch.tensor([5, 5]), cu)
    kv, vv = paged8.cache_values(k2, v2, s2)
    assert kv[2, 3, 0].tolist() == [448, 1] and vv[2, 3, 0].tolist() == [-448, -1]
    assert kv[0, 0, 0].tolist() == [2, 3] and kv[1, 3, 0].tolist() == [5, 6]
    same = torch.ones(3, 4, dtype=torch.bool)
    same[2, 3] = same[0, 0] = same[1, 3] = False
    assert (k2[same] == 9).all() and (v2[same] == 9).all() and (s2.transpose(1, 2)[same] == 100).all()
    rk, rv = paged8.read_reference(k2, v2, s2, table, torch.tensor([0, 5, 10]), 12)
    assert rk[3, 0].tolist() == [448, 1] and rk[4, 0].tolist() == [2, 3] and rk[8, 0].tolist() == [5, 6]
    assert (rk[9:] == 0).all() and (rv[9:] == 0).all()


def _case(lens_k, lens_q, hq, hkv, d, bs, seed):
    g = torch.Generator().manual_seed(seed)
    nblk = [-(-n // bs) for n in lens_k]
    perm = torch.randperm(sum(nblk) + 1, generator=g)
    table = torch.full((len(lens_k), max(nblk)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(nblk):
        table[b, :n] = perm[at:at + n].to(torch.int32)
        at += n
    kc, vc = (torch.randn(sum(nblk) + 1, bs, hkv, d, generator=g, dtype=torch.float64) for _ in range(2))
    cu = torch.tensor([0] + [sum(lens_q[:i + 1]) for i in range(len(lens_q))], dtype=torch.int32)
    return torch.randn(sum(lens_q), hq, d, generator=g, dtype=torch.float64), kc, vc, table, cu, torch.tensor(lens_k)


@pytest.mark.parametrize("causal", [True, False])
def test_without_a_window_it_is_the_chunked_prefill(causal):
    case = _case([20, 7, 33], [5, 7, 1], 4, 2, 16, 8, 1)
    o, lse, a, big = paged8.window_reference(*case, causal=causal)
    want, want_lse = paged_prefill_reference(*case, causal)
    torch.testing.assert_close(o, want, atol=1e-12, rtol=0)
    torch.testing.assert_close(lse, want_lse.T, atol=1e-12, rtol=0)
    assert (a >= o.abs() - 1e-12).all() and (big > 0).all()


def test_window_and_sinks_by_loops():
    q, kc, vc, table, cu, sl = _case([40, 9], [6, 9], 2, 1, 8, 8, 2)
    o, lse, *_ = paged8.window_reference(q, kc, vc, table, cu, sl, window=5, sinks=2)
    for b, (nk, n) in enumerate(((40, 6), (9, 9))):
        k, v = (paged8.rows_of(c, table, b, nk) for c in (kc, vc))
        for i in range(n):
            p = nk - n + i
            keys = [j for j in range(nk) if j <= p and (p - j < 5 or j < 2)]
            for h in range(2):
                want, want_lse = attention_reference(q[int(cu[b]) + i, h][None, None], k[keys, 0][None], v[keys, 0][None], False)
                torch.testing.assert_close(o[int(cu[b]) + i, h], want[0, 0], atol=1e-12, rtol=0)
                assert abs(lse[int(cu[b]) + i, h] - want_lse[0, 0]) < 1e-12


def test_a_planted_window_offset_shows():
    q, kc, vc, table, cu, sl = _case([40], [6], 2, 1, 8, 8, 5)
    a = paged8.window_reference(q, kc, vc, table, cu, sl, window=5, sinks=2)[0]
    assert (a - paged8.window_reference(q, kc, vc, table, cu, sl, window=6, sinks=2)[0]).abs().max() > 1e-3
    assert (a - paged8.window_reference(q, kc, vc, table, cu, sl, window=5, sinks=1)[0]).abs().max() > 1e-3


def test_rows_that_see_nothing():
    q, kc, vc, table, cu, sl = _case([4, 8], [6, 3], 2, 1, 8, 8, 3)  # two queries before position 0
    o, lse, *_ = paged8.window_reference(q, kc, vc, table, cu, sl, window=3)
    assert (o[:2] == 0).all() and (lse[:2] == -math.inf).all() and torch.isfinite(lse[2:]).all()
