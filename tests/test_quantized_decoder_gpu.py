"""KVCacheDecoder over an 8-bit cache and under a window: prompts and decode steps against a float64 forward.

The forward takes K and V as the decoder's cache holds them: its own rows, off by a bf16 activation's error, would fall on the
other side of a code's rounding here and there, and one e4m3 step is more than all the errors that are looked for. The cache's
rows are compared with the forward's on their own: half a step of the code (2^-4 of the value, 2^-10 of the scale, which is at
most amax / 224, below the smallest normal one), and what bf16 activations are off by, at most 5% of the row's amax.
The bound of the logits is the reference's own: its bf16 forward's mean distance from float64 on the same tokens (without a
window), twice that for two independent roundings of every activation. The forward with a window or a sink more or less, or
with rows that were not quantised, must lie further away than that, so that the comparison tells them apart.
"""
from dataclasses import replace

import pytest
import torch

from lightserve_amd.model.graph_decode import KVCacheDecoder, capture, main
from lightserve_amd.model.minimal_llama import TOY_CONFIG, init_weights
from oracle import paged8
from oracle.model import reference_llama_forward, windowed_llama_forward

pytestmark = pytest.mark.gpu


def _model(n_kv_heads=2):
    """A toy model whose attention matters: q, k and v four times the usual."""
    config = replace(TOY_CONFIG, n_kv_heads=n_kv_heads)
    weights = init_weights(config, device="cuda", seed=0)
    for layer in weights.layers:
        for name in ("q_proj", "k_proj", "v_proj"):
            getattr(layer, name).mul_(4)
    return config, weights


@pytest.mark.parametrize("kv_e4m3,window,sinks", [(True, None, 0), (True, 16, 2), (False, 16, 2), (True, 1, 0)])
@pytest.mark.parametrize("n_kv_heads", [2, None])
def test_prompt_and_steps(gpu, n_kv_heads, kv_e4m3, window, sinks):
    print(f"case decoder kv={n_kv_heads} e4m3={kv_e4m3} window={window} sinks={sinks}", flush=True)
    config, weights = _model(n_kv_heads)
    dec = KVCacheDecoder(weights, config, batch_size=2, block_size=16, kv_e4m3=kv_e4m3, window=window, sinks=sinks)
    ids = torch.randint(0, config.vocab_size, (2, 41), generator=torch.Generator().manual_seed(3)).cuda()
    got = [dec.prefill(ids[:, :30], 13)]
    for t in range(30, 41):
        dec.tokens.copy_(ids[:, t])
        got.append(dec.step())
        dec.seq_lens.add_(1)
    got = torch.stack(got, 1).double().cpu()

    held, rows = [], []
    table = dec.block_tables.cpu()
    for kc, vc, sc in zip(dec.k_cache, dec.v_cache, dec.kv_scales):
        both = (kc.double().cpu(), vc.double().cpu()) if sc is None else \
            paged8.cache_values(*(t.cpu().view(torch.uint8) for t in (kc, vc, sc)))
        held.append(tuple(torch.stack([paged8.rows_of(c, table, b, 41) for b in range(2)]) for c in both))

    def forward(w=window, s=sinks, h=held, rows=None):
        return windowed_llama_forward(weights, config, ids, w, s, h, rows)[:, 29:]

    def distance(a, b):
        return (a - b).abs().mean().item()

    right = forward(rows=rows)
    for layer, own in zip(held, rows):
        for a, b in zip(layer, own):
            amax = b.abs().amax(-1, keepdim=True)
            assert ((a - b).abs() <= (2.0 ** -4 * b.abs() + 2.0 ** -10 * amax / 224 if kv_e4m3 else 0) + 0.05 * amax).all()
    bound = 2 * distance(reference_llama_forward(weights, config, ids).double().cpu(), windowed_llama_forward(weights, config, ids))
    others = [forward(h=rows)] if kv_e4m3 else []
    if window is not None:
        others += [forward(w=window + 1), forward(s=sinks + 1), forward(w=None, s=0)]
    print(f"[decoder] {distance(got, right):.2e} of {bound:.2e}, others {[f'{distance(got, o):.2e}' for o in others]}", flush=True)
    assert distance(got, right) <= bound < min(distance(got, o) for o in others)


def test_replayed_steps_equal_eager_ones(gpu):
    print("case decoder graph replay, 8 bits and a window", flush=True)
    config, weights = _model()
    eager, graphed = (KVCacheDecoder(weights, config, batch_size=3, block_size=16, kv_e4m3=True, window=5, sinks=1)
                      for _ in range(2))
    graph, out = capture(graphed.step)
    graphed.seq_lens.zero_()
    graphed.tokens.fill_(1)
    for t in range(12):
        ref = eager.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref), f"step {t}"
        eager.advance(ref)
        graphed.advance(out)
    for a, b in zip(eager.k_cache + eager.v_cache + eager.kv_scales, graphed.k_cache + graphed.v_cache + graphed.kv_scales):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_the_command(gpu, capsys):
    print("case decode command, 8 bits and a window", flush=True)
    r = main(["--mode", "kvcache", "--n-layers", "1", "--num-steps", "3", "--warmup-steps", "1", "--max-seq-len", "64", "--gqa",
              "--kv-e4m3", "--window", "32", "--sinks", "4"])
    assert r["kvcache"]["graph"]["median_ms"] > 0
    r = main(["--prefill", "100", "--chunk", "64", "--n-layers", "1", "--num-steps", "2", "--warmup-steps", "1", "--gqa", "--kv-e4m3"])
    assert r["median_ms"] > 0
