"""The log-sums of beam search's selection, where the rounding of 32-bit differences of logits would show.

Peaks everywhere among equal logits: each difference of those from a peak is rounded alike, by up to 2^-22 where it lies between four and
eight, and so a log-sum that took the rounded ones would be off by nearly as much. The exponentials are exp2's of the hardware,
within one step of themselves: a sum of them is off by at most 2^-23 of itself and its logarithm by as much, and a score in
32 bits by 2^-24 |score| more. Beams that are 1.5e-7 apart are told apart where one's sum has a single term and is exact.
"""
import math

import pytest
import torch

from lightserve_amd.kernels.beam_search import beam_search_select

pytestmark = pytest.mark.gpu
VOCAB, APART = 50257, 250  # (fewer than the logits of one wave, whose own largest is subtracted)
# (peaks, the others): differences that 32 bits round down and up, by most of 2^-22
NEAR = math.floor(0.1 * 2 ** 21) / 2 ** 21
ROWS = {torch.float32: [(4.25, NEAR + s * 0.48 * 2 ** -21) for s in (1, -1)] + [(5.0, NEAR + s * 0.47 * 2 ** -21) for s in (1, -1)],
        torch.bfloat16: [(4.25, s * 2.0 ** -22 * 0.984375) for s in (1, -1)],
        torch.float16: [(4.25, s * 3 * 2.0 ** -24) for s in (1, -1)]}


def _row(dtype, peak, others):
    x = torch.full((VOCAB,), others, dtype=torch.double).to(dtype)
    x[::APART] = peak
    n = len(range(0, VOCAB, APART))
    peak, others = x[0].double().item(), x[1].double().item()
    assert 1.7e-7 < abs((x[1].float() - x[0].float()).double().item() - (others - peak)) < 2.0 ** -22
    return x, -math.log(n + (VOCAB - n) * math.exp(others - peak))  # a peak's log probability


@pytest.mark.parametrize("dtype", list(ROWS))
def test_log_sums(gpu, dtype):
    """Scores near zero, whose own rounding is none: what is left is the log-sum's error."""
    print(f"case log sums {dtype}", flush=True)
    for peak, others in ROWS[dtype]:
        x, p = _row(dtype, peak, others)
        s = torch.tensor([[-p]])  # rounded to 32 bits
        for rows in (1, 7, 256):  # (chunks of all sizes)
            got = beam_search_select(x.cuda().repeat(rows, 1), s.cuda().repeat(rows, 1), 1)
            want = s.double().item() + p
            assert abs(want) < 2.0 ** -21 and not got[2].any()
            off = (got[0].double().cpu() - want).abs().max().item()
            print(f"[sum] {peak} {others} rows={rows}: off by {off:.2e}", flush=True)
            assert off <= 2.0 ** -23 + 2.0 ** -24 * abs(want)


@pytest.mark.parametrize("dtype", list(ROWS))
@pytest.mark.parametrize("gap", [1.5e-7, -1.5e-7])
def test_beams_near_each_other(gpu, dtype, gap):
    """Beam 1 offers one candidate, its score itself, this far above beam 0's best."""
    print(f"case near beams {dtype} {gap}", flush=True)
    for peak, others in ROWS[dtype]:
        x, p = _row(dtype, peak, others)
        alone = torch.full((VOCAB,), -math.inf, dtype=dtype)
        alone[7] = 1.0
        first = -round(p * 1024) / 1024
        s = torch.tensor([[first, first + p + gap]])
        assert 1.45e-7 < (s[0, 1].double().item() - (first + p)) * math.copysign(1, gap) < 1.55e-7
        got = beam_search_select(torch.stack([x, alone]).cuda(), s.cuda(), 1)
        assert (got[1].item(), got[2].item()) == ((1, 7) if gap > 0 else (0, 0)), (peak, others)
