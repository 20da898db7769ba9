"""Decode loops with several candidates per sequence, over a KVCacheDecoder (graph_decode.py).

The reference's loop keeps one token per sequence and step, the argmax of its logits (model/cuda_graph_decode.py:114, :145).

    LookupDrafts(dec, drafts, branches=1)   the same tokens in fewer steps: each step verifies `branches` drafted
                                            continuations of `drafts` tokens and keeps what the argmax agrees with
    BeamSearch(dec, beams)                  the `beams` most probable continuations of each sequence; dec's batch is
                                            sequences * beams

step() issues only device work of static shape and returns nothing, so it can be captured and replayed; reset() goes back to
the seed token, and start(prompt) to the end of a prompt [sequences, P].
"""
import torch

from ..kernels.beam_search import beam_search_select, kv_cache_reorder
from ..kernels.draft_tree import draft_tree


BUCKETS = 1 << 16  # of LookupDrafts' index: pairs of tokens that fall together give drafts that are not accepted


class LookupDrafts:
    """Greedy decoding with drafts from the text itself: the continuations of the `branches` latest earlier places where its
    last two tokens stand. Where there are fewer, any other draft costs its rows of the step and nothing else. Under a window
    drafts must be fewer than its tokens (KVCacheDecoder.draft_step).

    text int64 [B, max_seq_len + 1]: each sequence's tokens, the current one last, at seq_lens (the last column is scratch, and
    so is what follows once the cache is full)."""

    def __init__(self, dec, drafts, branches=1):
        assert drafts >= 1 and branches >= 1, "at least one draft"
        window = dec.attention["window"]
        assert window is None or drafts < window, f"drafts must be fewer than the window's tokens ({drafts} of {window})"
        self.dec, self.drafts, self.branches = dec, drafts, branches
        self.n = 1 + drafts * branches
        # node 0, then one chain after another, each from node 0 on
        mask, depth = draft_tree([-1] + [0 if j == 0 else w * drafts + j for w in range(branches) for j in range(drafts)])
        device = dec.tokens.device
        self.mask = mask.repeat(dec.B, 1).to(device)
        self.depth = depth.repeat(dec.B, 1).to(device)
        self.text = torch.zeros(dec.B, dec.cfg.max_seq_len + 1, dtype=torch.long, device=device)
        # the place where a pair of tokens stood last (its second token, once that is followed), and before each place the one before
        self.places = torch.zeros(dec.B, BUCKETS, dtype=torch.long, device=device)
        self.before = torch.zeros_like(self.text)
        self.reset()

    def reset(self):
        self.dec.reset()
        self.text.zero_()
        self.text[:, 0] = self.dec.tokens
        self.places.zero_()
        self.before.zero_()

    def start(self, prompt, chunk_size=512):
        self.reset()
        logits = self.dec.prefill(prompt, chunk_size)
        P = prompt.shape[1]
        self.text[:, :P] = prompt
        self.text[:, P] = self.dec.tokens
        places = torch.arange(P, device=prompt.device).repeat(self.dec.B, 1)
        key, order = self._bucket(places).sort(dim=1, stable=True)
        earlier = torch.where(key[:, 1:] == key[:, :-1], order[:, :-1], 0)
        self.before.scatter_(1, order[:, 1:], earlier)
        self.places.scatter_reduce_(1, self._bucket(places), places, "amax")
        return logits

    def _bucket(self, places):
        pair = self.text.gather(1, (places - 1).clamp(min=0)) * 31337 + self.text.gather(1, places)
        return pair % BUCKETS

    def _last(self):
        """Where the current tokens stand [B, 1]."""
        return self.dec.seq_lens.long().clamp(max=self.text.shape[1] - 1).view(-1, 1)

    def propose(self):
        """The nodes' tokens [B, n]."""
        text, last = self.text, self._last()
        found = [self.places.gather(1, self._bucket(last))]
        for _ in range(self.branches - 1):
            found.append(self.before.gather(1, found[-1]))
        found = torch.cat(found, 1).minimum((last - 1).clamp(min=0)).unsqueeze(2)
        # (past the current token the text is taken to repeat what lies between the two places)
        ahead = torch.arange(self.drafts, device=text.device) % (last.unsqueeze(2) - found).clamp(min=1)
        follow = (found + 1 + ahead).minimum(last.unsqueeze(2))
        return torch.cat([self.dec.tokens.view(-1, 1), text.gather(1, follow.flatten(1))], 1)

    def step(self):
        dec, last = self.dec, self._last()
        tokens = self.propose()
        path, counts, following = dec.accept(dec.draft_step(tokens, self.mask, self.depth, self.drafts), tokens, self.mask)
        # the path's tokens after node 0, then the choice after them, go behind the current token
        i, counts = torch.arange(self.n, device=tokens.device), counts.view(-1, 1)
        taken = tokens.gather(1, path.roll(-1, 1).clamp(min=0).long())
        taken = torch.where(i == counts - 1, following.view(-1, 1), taken)
        scratch = self.text.shape[1] - 1
        self.text.scatter_(1, torch.where(i < counts, (last + 1 + i).clamp(max=scratch), scratch), taken)
        # and their pairs into the index, as far as they are followed (place 0 stands for none)
        places = torch.where(i < counts, (last + i).clamp(max=scratch), 0)
        key = self._bucket(places)
        self.before.scatter_(1, places, torch.where(places > 0, self.places.gather(1, key), 0))
        self.places.scatter_reduce_(1, key, places, "amax")


class BeamSearch:
    """text int64 [sequences, beams, max_seq_len + 1] and scores fp32 [sequences, beams], best first: the beams' tokens (the
    current one at seq_lens; past the end of the cache the last column) and sums of log probabilities."""

    def __init__(self, dec, beams):
        assert beams >= 1 and dec.B % beams == 0, "the decoder's batch must be sequences * beams"
        self.dec, self.beams, self.sequences = dec, beams, dec.B // beams
        device = dec.tokens.device
        self.scores = torch.zeros(self.sequences, beams, device=device)
        self.text = torch.zeros(self.sequences, beams, dec.cfg.max_seq_len + 1, dtype=torch.long, device=device)
        self.reset()

    def _alone(self):
        """All beams are alike: the first one takes part."""
        self.scores.fill_(float("-inf"))
        self.scores[:, 0] = 0

    def reset(self):
        self.dec.reset()
        self.text.zero_()
        self.text[:, :, 0] = self.dec.tokens.view(self.sequences, self.beams)
        self._alone()

    def start(self, prompt, chunk_size=512):
        self.reset()
        logits = self.dec.prefill(prompt.repeat_interleave(self.beams, 0), chunk_size)
        self.text[:, :, :prompt.shape[1]] = prompt.unsqueeze(1)
        self._choose(logits)
        return logits

    def step(self):
        dec = self.dec
        logits = dec.step()
        dec.seq_lens.add_(1)
        self._choose(logits)

    def _choose(self, logits):
        dec = self.dec
        scores, parents, tokens = beam_search_select(logits, self.scores)
        kv_cache_reorder(*dec.caches[:2], dec.block_tables, dec.seq_lens, parents, kv_scales=dec.caches[2])
        self.scores.copy_(scores)
        dec.tokens.copy_(tokens.view(-1))
        at = parents.long().unsqueeze(2)
        self.text.copy_(self.text.gather(1, at.expand_as(self.text)))
        where = dec.seq_lens.long().clamp(max=self.text.shape[2] - 1).view(self.sequences, self.beams, 1)
        self.text.scatter_(2, where, tokens.unsqueeze(2))
