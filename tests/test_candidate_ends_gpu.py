"""Decode loops with draft trees up to the last row of a cache.

As in test_candidate_decoding_gpu.py logits are held to float64 forwards of each candidate's own tokens over K and V as the cache
holds them, by twice the reference's bf16 forward's mean distance from float64 on the same tokens; paths, tokens and rows are
exact given the logits.
"""
from dataclasses import replace

import pytest
import torch

from lightserve_amd.kernels.draft_tree import draft_tree
from lightserve_amd.model.candidates import BeamSearch, LookupDrafts
from lightserve_amd.model.graph_decode import KVCacheDecoder, capture
from oracle import candidates
from oracle.model import reference_llama_forward, windowed_llama_forward
from tests.candidate_cases import raw
from tests.test_candidate_decoding_gpu import _held, _model, _path

pytestmark = pytest.mark.gpu


def _fenced(dec):
    """The decoder's caches put between blocks that no table names; those blocks, and what they hold."""
    fences, caches = [], []
    for c in dec.caches:
        if c is None:
            caches.append(None)
            continue
        wide = torch.empty(c.shape[0], c.shape[1] + 2, *c.shape[2:], dtype=torch.uint8, device="cuda").view(c.dtype) if c.element_size() == 1 \
            else torch.empty(c.shape[0], c.shape[1] + 2, *c.shape[2:], dtype=c.dtype, device="cuda")
        wide.view(torch.uint8).fill_(0x3b)
        wide[:, 1:-1].view(torch.uint8).copy_(c.view(torch.uint8))
        caches.append(wide[:, 1:-1])
        fences += [wide[:, :1], wide[:, -1:]]
    dec.caches = tuple(caches)
    dec.k_cache, dec.v_cache, dec.kv_scales = ([None] * dec.caches[0].shape[0] if c is None else list(c.unbind(0)) for c in caches)
    return fences, [raw(f.contiguous()).clone() for f in fences]


@pytest.mark.parametrize("kv_e4m3,window,sinks", [(False, None, 0), (True, None, 0), (False, 16, 2)])
@pytest.mark.parametrize("room", [(8, 5, 2), (7, 6, 1), (3, 4, 12)])
def test_draft_steps_at_the_end(gpu, kv_e4m3, window, sinks, room):
    """Trees of 8 nodes where sequences have this many rows left: nodes whose rows are cached are what they are anywhere, and no
    others are accepted, right as their tokens may be."""
    print(f"case drafts at the end e4m3={kv_e4m3} window={window} room={room}", flush=True)
    config, weights = _model()
    dec = KVCacheDecoder(weights, config, 3, kv_e4m3=kv_e4m3, window=window, sinks=sinks)
    fences, had = _fenced(dec)
    end, g = config.max_seq_len, torch.Generator().manual_seed(3)
    prompt = torch.randint(0, config.vocab_size, (3, end), generator=g)
    base = [end - r for r in room]
    dec.prefill(prompt[:, :max(base)].cuda(), 13)
    dec.seq_lens.copy_(torch.tensor(base))
    dec.tokens.copy_(torch.tensor([prompt[b, n] for b, n in enumerate(base)]))
    parents = [-1, 0, 1, 0, 3, 3, 2, 4]
    n = len(parents)
    mask, depth = draft_tree(parents)
    mask, depth = mask.repeat(3, 1).cuda(), depth.repeat(3, 1).cuda()
    tokens = torch.randint(0, config.vocab_size, (3, n), generator=g)
    tokens[:, 0] = dec.tokens.cpu()
    for node, parent in ((3, 0), (5, 3)):  # the choices after node 0, and after node 3
        tokens[:, node] = dec.draft_step(tokens.cuda(), mask, depth).view(3, n, -1)[:, parent].argmax(-1).cpu()
    logits = dec.draft_step(tokens.cuda(), mask, depth)
    held = [_held(dec, b, min(base[b] + n, end)) for b in range(3)]
    for b in range(3):
        off, bound = [], []
        for i in range(min(n, room[b])):
            path = _path(parents, i)
            at = list(range(base[b])) + [base[b] + j for j in path]
            ids = torch.tensor([prompt[b, :base[b]].tolist() + [tokens[b, j].item() for j in path]])
            rows = [tuple(c[at].unsqueeze(0) for c in layer) for layer in held[b]]
            want = windowed_llama_forward(weights, config, ids, window, sinks, rows)[0, -1]
            off.append((logits[b * n + i].double().cpu() - want).abs().mean())
            bound.append((reference_llama_forward(weights, config, ids.cuda()).double().cpu()[0, -1]
                          - windowed_llama_forward(weights, config, ids)[0, -1]).abs().mean())
        off, bound = torch.stack(off).mean(), 2 * torch.stack(bound).mean()
        print(f"[end] room {room[b]}: {off:.2e} of {bound:.2e}", flush=True)
        assert off <= bound, f"{room[b]} rows left"
    path, counts, following = dec.accept(logits, tokens.cuda(), mask)
    kept = torch.cat([mask.cpu()[b * n:(b + 1) * n] * (torch.arange(n) < room[b])[:, None] for b in range(3)])
    cu = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32)
    paths, many, after = candidates.accept_reference(logits.cpu(), tokens.view(-1), kept, cu, n)
    assert path.tolist() == paths and counts.tolist() == many and following.tolist() == after == dec.tokens.tolist()
    assert [p[:m] for p, m in zip(paths, many)] == [[0, 3, 5][:1 + (r > 3) + (r > 5)] for r in room]
    assert dec.seq_lens.tolist() == [a + c for a, c in zip(base, many)] and max(dec.seq_lens.tolist()) <= end
    for b in range(3):
        now, at = _held(dec, b, base[b] + many[b]), list(range(base[b])) + [base[b] + j for j in paths[b][:many[b]]]
        assert all(torch.equal(x, y[at]) for layer, was in zip(now, held[b]) for x, y in zip(layer, was))
    assert all(torch.equal(raw(f.contiguous()), w) for f, w in zip(fences, had)), "blocks of no table were written"


@pytest.mark.parametrize("kv_e4m3", [False, True])
@pytest.mark.parametrize("drafts,branches", [(3, 3), (8, 1), (20, 12)])
@pytest.mark.parametrize("end,block_size", [(64, 16), (59, 32)])
def test_lookup_drafts_to_the_end(gpu, kv_e4m3, drafts, branches, end, block_size):
    """Every token up to the cache's end is the choice of the logits before it, eagerly and in replays, for sequences that get there
    one after another; steps past the end write nothing outside the cache."""
    print(f"case lookup to the end e4m3={kv_e4m3} drafts={drafts} branches={branches} end={end}", flush=True)
    config, weights = _model()
    config = replace(config, max_seq_len=end)
    eager, graphed = (LookupDrafts(KVCacheDecoder(weights, config, 3, block_size, kv_e4m3=kv_e4m3), drafts, branches) for _ in range(2))
    fences, had = _fenced(eager.dec)
    graph, _ = capture(graphed.step)
    P = 49
    prompt = torch.randint(0, config.vocab_size, (3, 7), generator=torch.Generator().manual_seed(5)).repeat(1, 7).cuda()
    for loop in (eager, graphed):
        loop.start(prompt, 16)
        for b, shorter in enumerate((0, 2, 5)):  # (a shorter prompt: its next token as the current one)
            loop.dec.seq_lens[b] -= shorter
            loop.dec.tokens[b] = loop.text[b, P - shorter]
    steps = 0
    while eager.dec.seq_lens.min() < end + 2:
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        steps += 1
        was = eager.dec.seq_lens.clamp(max=end).tolist()
        assert was == graphed.dec.seq_lens.clamp(max=end).tolist() and steps < 40
        for b in range(3):
            m = min(was[b], end - 1)
            assert torch.equal(eager.text[b, :m + 1], graphed.text[b, :m + 1])
    for b in range(3):
        ids = eager.text[b:b + 1, :end]
        held = [tuple(c.unsqueeze(0) for c in layer) for layer in _held(eager.dec, b, end)]
        exact = windowed_llama_forward(weights, config, ids, None, 0, held)[0]
        plain = windowed_llama_forward(weights, config, ids)[0]
        bound = 2 * (reference_llama_forward(weights, config, ids).double().cpu()[0] - plain).abs().amax(-1)
        for p in range(P + 1, end):
            short = exact[p - 1].max() - exact[p - 1, eager.text[b, p]]
            assert short <= 2 * bound[p - 1], (b, p, short, bound[p - 1])
    assert all(torch.equal(raw(f.contiguous()), w) for f, w in zip(fences, had)), "blocks of no table were written"


@pytest.mark.parametrize("drafts,branches,window,sinks", [(3, 2, 4, 0), (3, 5, 4, 2), (7, 1, 8, 1)])
def test_lookup_drafts_under_a_short_window(gpu, drafts, branches, window, sinks):
    """As many drafts as a window allows: the tokens are the windowed choices."""
    print(f"case lookup window={window} drafts={drafts}", flush=True)
    config, weights = _model()
    loop = LookupDrafts(KVCacheDecoder(weights, config, 2, window=window, sinks=sinks), drafts, branches)
    prompt = torch.randint(0, config.vocab_size, (2, 6), generator=torch.Generator().manual_seed(5)).repeat(1, 4).cuda()
    loop.start(prompt, 16)
    for _ in range(12):
        loop.step()
    lens = loop.dec.seq_lens.tolist()
    for b in range(2):
        ids = loop.text[b:b + 1, :lens[b]]
        held = [tuple(c.unsqueeze(0) for c in layer) for layer in _held(loop.dec, b, lens[b])]
        exact = windowed_llama_forward(weights, config, ids, window, sinks, held)[0]
        plain = windowed_llama_forward(weights, config, ids)[0]
        bound = 2 * (reference_llama_forward(weights, config, ids).double().cpu()[0] - plain).abs().amax(-1)
        for p in range(24, lens[b]):
            short = exact[p - 1].max() - exact[p - 1, loop.text[b, p]]
            assert short <= 2 * bound[p - 1], (b, p, short, bound[p - 1])


@pytest.mark.parametrize("kv_e4m3", [False, True])
def test_beam_search_to_the_end(gpu, kv_e4m3):
    """Beams that fill the cache to its last row have the sums of their tokens' log probabilities as scores (bounds as in
    test_candidate_decoding_gpu.py), and steps past it write nothing outside the cache."""
    print(f"case beams to the end e4m3={kv_e4m3}", flush=True)
    config, weights = _model()
    sequences, beams, P, end = 2, 3, 45, config.max_seq_len
    loop = BeamSearch(KVCacheDecoder(weights, config, sequences * beams, kv_e4m3=kv_e4m3), beams)
    fences, had = _fenced(loop.dec)
    prompt = torch.randint(0, config.vocab_size, (sequences, P), generator=torch.Generator().manual_seed(6)).cuda()
    loop.start(prompt, 16)
    for _ in range(end - P):
        loop.step()
    assert loop.dec.seq_lens.tolist() == [end] * (sequences * beams)
    for b in range(sequences):
        for k in range(beams):
            ids = loop.text[b, k, :end].view(1, -1)
            held = [tuple(c.unsqueeze(0) for c in layer) for layer in _held(loop.dec, b * beams + k, end)]
            plain = windowed_llama_forward(weights, config, ids)
            bound = 4 * (reference_llama_forward(weights, config, ids).double().cpu() - plain)[0, P - 1:].abs().amax(-1).sum().item()
            p = windowed_llama_forward(weights, config, ids, None, 0, held).double().log_softmax(-1)[0, P - 1:]
            off = abs(p.gather(1, loop.text[b, k, P:end + 1].cpu().view(-1, 1)).sum().item() - loop.scores[b, k].item())
            print(f"[beams] {b} {k}: {off:.3f} of {bound:.3f}", flush=True)
            assert off <= bound
    for _ in range(4):
        loop.step()
    torch.cuda.synchronize()
    assert all(torch.equal(raw(f.contiguous()), w) for f, w in zip(fences, had)), "blocks of no table were written"
