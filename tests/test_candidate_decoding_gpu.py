"""Decode loops with draft trees and beams over KVCacheDecoder.

Logits are held to float64 forwards of each candidate's own tokens, with the bound of test_quantized_decoder_gpu.py: the
reference's bf16 forward's mean distance from float64 on the same tokens, twice for two independent roundings of every
activation. The forwards take K and V as the cache holds them, as there. What a loop keeps is exact given its logits: tokens,
text and cache rows.
"""
from dataclasses import replace

import pytest
import torch

from lightserve_amd.kernels.draft_tree import draft_tree
from lightserve_amd.model.candidates import BeamSearch, LookupDrafts
from lightserve_amd.model.graph_decode import KVCacheDecoder, capture, main
from lightserve_amd.model.minimal_llama import TOY_CONFIG, init_weights
from oracle import candidates, paged8
from oracle.model import reference_llama_forward, windowed_llama_forward

pytestmark = pytest.mark.gpu


def _model():
    """A toy model whose attention matters: q, k and v four times the usual."""
    config = replace(TOY_CONFIG, n_kv_heads=2)
    weights = init_weights(config, device="cuda", seed=0)
    for layer in weights.layers:
        for name in ("q_proj", "k_proj", "v_proj"):
            getattr(layer, name).mul_(4)
    return config, weights


def _held(dec, b, total):
    """What the cache stands for of sequence b's first rows: (k, v) of each layer."""
    table, out = dec.block_tables.cpu(), []
    for kc, vc, sc in zip(dec.k_cache, dec.v_cache, dec.kv_scales):
        both = (kc.double().cpu(), vc.double().cpu()) if sc is None else \
            paged8.cache_values(*(t.cpu().view(torch.uint8) for t in (kc, vc, sc)))
        out.append(tuple(paged8.rows_of(c, table, b, total) for c in both))
    return out


def _path(parents, i):
    nodes = []
    while i >= 0:
        nodes.insert(0, i)
        i = parents[i]
    return nodes


@pytest.mark.parametrize("kv_e4m3,window,sinks", [(False, None, 0), (True, None, 0), (True, 16, 2)])
def test_draft_steps(gpu, kv_e4m3, window, sinks):
    """Steps over random trees whose tokens are partly the model's own choice: logits of every node, then path and cache."""
    print(f"case draft steps e4m3={kv_e4m3} window={window}", flush=True)
    config, weights = _model()
    dec = KVCacheDecoder(weights, config, 2, kv_e4m3=kv_e4m3, window=window, sinks=sinks)
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, config.vocab_size, (2, 25), generator=g)
    dec.prefill(prompt.cuda(), 13)
    text = [row.tolist() + [t] for row, t in zip(prompt, dec.tokens.tolist())]
    parents = [-1, 0, 1, 0, 3, 3, 2, 4]
    mask, depth = draft_tree(parents)
    mask, depth = mask.repeat(2, 1).cuda(), depth.repeat(2, 1).cuda()
    kept = []
    for step in range(3):
        tokens = torch.randint(0, config.vocab_size, (2, len(parents)), generator=g)
        tokens[:, 0] = torch.tensor([t[-1] for t in text])
        # node 3 is the choice after node 0, node 5 the one after node 3 in the first sequence
        for node, parent in ((3, 0), (5, 3)):
            choice = dec.draft_step(tokens.cuda(), mask, depth).view(2, len(parents), -1)[:, parent].argmax(-1).cpu()
            tokens[:, node] = choice if node == 3 else torch.stack([choice[0], (choice[1] + 1) % config.vocab_size])
        logits = dec.draft_step(tokens.cuda(), mask, depth)
        base = dec.seq_lens.tolist()
        got, want, ref, other = [], [], [], []
        rows = [_held(dec, b, base[b] + len(parents)) for b in range(2)]
        for b in range(2):
            for i in range(len(parents)):
                path = _path(parents, i)
                at = list(range(base[b])) + [base[b] + j for j in path]
                ids = torch.tensor([text[b][:-1] + [tokens[b, j].item() for j in path]])
                held = [tuple(c[at].unsqueeze(0) for c in layer) for layer in rows[b]]
                got.append(logits[b * len(parents) + i].double().cpu())
                want.append(windowed_llama_forward(weights, config, ids, window, sinks, held)[0, -1])
                ref.append((reference_llama_forward(weights, config, ids.cuda()).double().cpu()[0, -1],
                            windowed_llama_forward(weights, config, ids)[0, -1]))
                if i in (2, 4, 5, 6, 7):  # the same node with its parent's row unseen
                    less = ids[:, :-2].new_tensor([ids[0, :-2].tolist() + [ids[0, -1].item()]])
                    cut = [tuple(torch.cat([c[:, :-2], c[:, -1:]], 1) for c in layer) for layer in held]
                    other.append((got[-1], windowed_llama_forward(weights, config, less, window, sinks, cut)[0, -1]))
        bound = 2 * torch.stack([(a - c).abs().mean() for a, c in ref]).mean()
        off = torch.stack([(a - c).abs().mean() for a, c in zip(got, want)]).mean()
        wrong = torch.stack([(a - c).abs().mean() for a, c in other]).mean()
        print(f"[drafts] {off:.2e} of {bound:.2e}, without the parent {wrong:.2e}", flush=True)
        assert off <= bound < wrong
        path, counts, following = dec.accept(logits, tokens.cuda(), mask)
        cu = torch.tensor([0, len(parents), 2 * len(parents)], dtype=torch.int32)
        paths, many, after = candidates.accept_reference(logits.cpu(), tokens.view(-1), mask.cpu(), cu, len(parents))
        assert path.tolist() == paths and counts.tolist() == many and following.tolist() == after == dec.tokens.tolist()
        assert many[0] >= 3 and many[1] >= 2 and paths[0][:3] == [0, 3, 5]
        assert dec.seq_lens.tolist() == [a + c for a, c in zip(base, many)]
        for b in range(2):
            now = _held(dec, b, base[b] + many[b])
            at = list(range(base[b])) + [base[b] + j for j in paths[b][:many[b]]]
            assert all(torch.equal(x, y[at]) for layer, had in zip(now, rows[b]) for x, y in zip(layer, had))
            text[b] += [tokens[b, j].item() for j in paths[b][1:many[b]]] + [after[b]]
        kept.append(many)
    print(kept, flush=True)


@pytest.mark.parametrize("kv_e4m3", [False, True])
@pytest.mark.parametrize("branches", [1, 3])
def test_lookup_drafts(gpu, kv_e4m3, branches):
    """Replayed steps keep what eager ones do, and every token they keep is the choice of the logits before it."""
    print(f"case lookup e4m3={kv_e4m3} branches={branches}", flush=True)
    config, weights = _model()
    eager, graphed = (LookupDrafts(KVCacheDecoder(weights, config, 3, kv_e4m3=kv_e4m3), 3, branches) for _ in range(2))
    graph, _ = capture(graphed.step)
    prompt = torch.randint(0, config.vocab_size, (3, 6), generator=torch.Generator().manual_seed(5)).repeat(1, 4).cuda()
    for loop in (eager, graphed):
        loop.start(prompt, 16)
    first = eager.propose().cpu()
    # the prompt repeats itself: with the period's next token as the current one, its continuation is drafted
    current = eager.dec.tokens.clone()
    eager.text[:, 24] = prompt[:, 0]
    eager.dec.tokens.copy_(prompt[:, 0])
    drafted = eager.propose().cpu()
    assert torch.equal(drafted, torch.cat([prompt[:, :1], *([prompt[:, 1:4]] * branches)], 1).cpu()) and first.shape == drafted.shape
    eager.dec.tokens.copy_(current)
    eager.text[:, 24] = current
    for step in range(4):
        was = eager.dec.seq_lens.tolist()
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in ((eager.text, graphed.text), (eager.dec.seq_lens, graphed.dec.seq_lens), (eager.dec.tokens, graphed.dec.tokens),
                     (eager.places, graphed.places), (eager.before, graphed.before)):
            assert torch.equal(a[..., :-1] if a.dim() == 2 and a.shape[1] == 65 else a, b[..., :-1] if b.dim() == 2 and b.shape[1] == 65 else b)
        now = eager.dec.seq_lens.tolist()
        assert all(n > w for n, w in zip(now, was))
        assert [eager.text[b, n].item() for b, n in enumerate(now)] == eager.dec.tokens.tolist()
    # every kept token's logits in float64 are within the models' rounding of that position's largest
    lens = eager.dec.seq_lens.tolist()
    for b in range(3):
        ids = eager.text[b:b + 1, :lens[b]]
        held = [tuple(c.unsqueeze(0) for c in layer) for layer in _held(eager.dec, b, lens[b])]
        exact = windowed_llama_forward(weights, config, ids, None, 0, held)[0]
        plain = windowed_llama_forward(weights, config, ids)[0]
        bound = 2 * (reference_llama_forward(weights, config, ids).double().cpu()[0] - plain).abs().amax(-1)
        for p in range(24, lens[b]):
            short = exact[p - 1].max() - exact[p - 1, eager.text[b, p]]
            assert short <= 2 * bound[p - 1], (b, p, short, bound[p - 1])


@pytest.mark.parametrize("kv_e4m3", [False, True])
def test_beam_search(gpu, kv_e4m3):
    """Replayed steps keep what eager ones do; the texts are those that the choices name, and scores the sums of their tokens'
    log probabilities in float64 forwards, within the forwards' own rounding."""
    print(f"case beams e4m3={kv_e4m3}", flush=True)
    config, weights = _model()
    sequences, beams, P, steps = 2, 3, 14, 22
    eager, graphed = (BeamSearch(KVCacheDecoder(weights, config, sequences * beams, kv_e4m3=kv_e4m3), beams) for _ in range(2))
    graph, _ = capture(graphed.step)
    prompt = torch.randint(0, config.vocab_size, (sequences, P), generator=torch.Generator().manual_seed(5)).cuda()
    own = eager.dec.block_tables.clone()
    for loop in (eager, graphed):
        loop.start(prompt, 16)
    assert torch.equal(own, graphed.dec.own_tables) and (eager.scores[:, 1:] <= eager.scores[:, :-1]).all()
    for step in range(steps):
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in ((eager.text, graphed.text), (eager.scores, graphed.scores), (eager.dec.tokens, graphed.dec.tokens),
                     (eager.dec.block_tables, graphed.dec.block_tables), (eager.dec.seq_lens, graphed.dec.seq_lens)):
            assert torch.equal(a, b), step
    assert not torch.equal(eager.dec.block_tables, own), "complete blocks are shared"
    n = P + steps
    assert eager.dec.seq_lens.tolist() == [n] * (sequences * beams)
    for b in range(sequences):
        assert len({tuple(t) for t in eager.text[b, :, :n + 1].tolist()}) == beams
        for k in range(beams):
            row = b * beams + k
            ids = eager.text[b, k, :n].view(1, -1)
            assert torch.equal(ids[0, :P], prompt[b]) and eager.text[b, k, n] == eager.dec.tokens[row]
            held = [tuple(c.unsqueeze(0) for c in layer) for layer in _held(eager.dec, row, n)]

            def total(logits):
                p = logits.double().log_softmax(-1)[0, P - 1:]
                return p.gather(1, eager.text[b, k, P:n + 1].cpu().view(-1, 1)).sum().item()
            plain = windowed_llama_forward(weights, config, ids)
            # a token's log probability is off by at most twice its logits' largest error
            bound = 4 * (reference_llama_forward(weights, config, ids).double().cpu() - plain)[0, P - 1:].abs().amax(-1).sum().item()
            off = abs(total(windowed_llama_forward(weights, config, ids, None, 0, held)) - eager.scores[b, k].item())
            print(f"[beams] {b} {k}: {off:.3f} of {bound:.3f}", flush=True)
            assert off <= bound


def test_one_beam_is_greedy(gpu):
    print("case one beam", flush=True)
    config, weights = _model()
    prompt = torch.randint(0, config.vocab_size, (2, 9), generator=torch.Generator().manual_seed(8)).cuda()
    dec, loop = KVCacheDecoder(weights, config, 2), BeamSearch(KVCacheDecoder(weights, config, 2), 1)
    dec.prefill(prompt, 16)
    loop.start(prompt, 16)
    for _ in range(20):
        assert torch.equal(dec.tokens, loop.dec.tokens)
        dec.advance(dec.step())
        loop.step()
    for a, b in zip(dec.caches[:2], loop.dec.caches[:2]):
        assert torch.equal(a, b)


def test_reset_after_a_search(gpu):
    print("case reset", flush=True)
    config, weights = _model()
    loop = BeamSearch(KVCacheDecoder(weights, config, 4), 4)
    texts = []
    for _ in range(2):
        for _ in range(40):
            loop.step()
        texts.append((loop.text.clone(), loop.scores.clone()))
        loop.reset()
    assert torch.equal(texts[0][0], texts[1][0]) and torch.equal(texts[0][1], texts[1][1])


def test_full_cache(gpu):
    """Steps past the cache's end store nothing outside it and do not fail."""
    print("case full", flush=True)
    config, weights = _model()
    for make in (lambda d: LookupDrafts(d, 4, 2), lambda d: BeamSearch(d, 2)):
        for kv_e4m3 in (False, True):
            loop = make(KVCacheDecoder(weights, config, 2, kv_e4m3=kv_e4m3))
            loop.start(torch.ones(2 if isinstance(loop, LookupDrafts) else 1, 58, dtype=torch.long, device="cuda"), 32)
            for _ in range(12):
                loop.step()
            torch.cuda.synchronize()
            assert (loop.dec.seq_lens > 64).all()


def test_refusals(gpu):
    config, weights = _model()
    dec = KVCacheDecoder(weights, config, 3)
    for make in (lambda: LookupDrafts(dec, 0), lambda: LookupDrafts(dec, 128, 2), lambda: BeamSearch(dec, 2), lambda: BeamSearch(dec, 0)):
        with pytest.raises(AssertionError):
            make()
    with pytest.raises(AssertionError):
        dec.draft_step(torch.zeros(2, 4, dtype=torch.long, device="cuda"), None, torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    for words in (["--drafts", "2", "--beams", "2"], ["--drafts", "-1"], ["--drafts", "100", "--branches", "3"], ["--beams", "65"]):
        with pytest.raises(SystemExit):
            main(words)


@pytest.mark.parametrize("words", [["--drafts", "3", "--branches", "2"], ["--beams", "4", "--batch-size", "2", "--kv-e4m3"]])
def test_the_command(gpu, words):
    print("case command", words, flush=True)
    r = main([*words, "--n-layers", "1", "--num-steps", "3", "--warmup-steps", "1", "--gqa"])
    assert r["graph"]["median_ms"] > 0 and r["tokens_per_step"] >= 1
