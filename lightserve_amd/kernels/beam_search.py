"""Beam search over a paged KV cache on MI355X: the selection of a step, and the beams' caches after it.

The reference takes the argmax of each step's logits (model/cuda_graph_decode.py:114, :145). A beam search keeps several
candidates per sequence, each a row of its own in the block tables:

    scores, beams, tokens = beam_search_select(logits, scores, num=None)
    kv_cache_reorder(k_cache, v_cache, block_tables, seq_lens, beams, *, kv_scales=None)

beam_search_select takes the logits [batch * K, vocab] (fp32, fp16 or bf16) of a step and the beams' scores fp32 [batch, K] (sums of log
probabilities; -inf for a beam that takes no part, as all but the first in a search's first step) and
returns the num (default K) best of scores[b, k] + log_softmax(logits[b * K + k])[v] of each sequence, best first: scores fp32, beams int32 (the k)
and tokens int64 (the v), all [batch, num]. Equal ones go to the lower k, then the lower v. Sums and scores are held and
compared in 64 bits (sums of different beams are often nearer to each other than 32 bits tell) and rounded once at the end; the
exponentials are 32-bit ones, so that a beam's log-sum is off by up to 2^-23 and candidates of different beams that are nearer
than 2^-22 may stand either way. (So may different logits of one beam whose sums 64 bits round to one number, as beside
a score of -1e30.) A row of logits with NaN or +inf, or nothing above -inf, offers no candidates, nor
does a beam with a score of NaN or -inf; where fewer than num candidates are above -inf, the rest have score -inf, beam 0
and token 0. Up to 64 beams, 64 candidates and 2^20 tokens of a vocabulary, and 2560 chunks of 8192 tokens of one
sequence's beams (64 of 2^18 tokens, 19 of 2^20).

kv_cache_reorder lets beam k of sequence b go on from beam parents[b, k] (int32 [batch, K]; any other number: from itself). Beams b * K ..
b * K + K - 1 are the sequence's rows of block_tables int32 [batch * K, max_blocks] and seq_lens int32 [batch * K]; they have one length, which the
first one's entry gives. Blocks that are complete are shared: the beam's table entries become its parent's (in place).
Of the last, incomplete block the rows are copied into the block that the beam's own table names, so that every beam needs a block of its
own there, and for each block to come; they are written by no other. Which complete blocks no table names any more is for the caller
to find. Caches and kv_scales are as in kv_cache_keep (draft_tree.py): of one layer, or [layers, ...] with
one launch for all. A search over layers kept apart calls it for each, with the tables of before: the call changes them.
"""
import torch

from .. import _lib
from .draft_tree import cache_rows, launch_with_workspace
from .quantized_kv_cache import check_device

MAX_BEAMS, MAX_CANDIDATES = 64, 64  # LSFA_BEAMS_MAX, LSFA_BEAMS_NUM_MAX


def beam_search_select(logits, scores, num=None):
    assert logits.dim() == 2 and logits.dtype in _lib.TORCH_TO_LSFA, "logits must be [batch * beams, vocab] in fp32, fp16 or bf16"
    assert scores.dim() == 2 and scores.dtype == torch.float32, "scores must be fp32 [batch, beams]"
    batch, beams = scores.shape
    rows, vocab = logits.shape
    assert rows == batch * beams, "logits must have a row for each of scores' beams"
    num = beams if num is None else num
    assert 1 <= beams <= MAX_BEAMS and 1 <= num <= MAX_CANDIDATES, f"1 to {MAX_BEAMS} beams and {MAX_CANDIDATES} candidates"
    assert rows == 0 or vocab > 0, "the vocabulary must not be empty"
    if not logits.get_device() == scores.get_device() >= 0:
        check_device((("logits", logits), ("scores", scores)))
    if rows and (logits.stride(1) != 1 or logits.stride(0) < vocab):
        logits = _lib.packed(logits)
    device = logits.device
    out = scores.new_empty((batch, num))
    parents = torch.empty((batch, num), dtype=torch.int32, device=device)
    tokens = torch.empty((batch, num), dtype=torch.int64, device=device)
    if batch > 0:
        scores = scores.contiguous()
        args = _lib.pack(
            _lib.BeamArgs, logits.data_ptr(), scores.data_ptr(), out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), 0, 0,
            max(logits.stride(0), vocab), _lib.TORCH_TO_LSFA[logits.dtype], batch, beams, vocab, num, 0)
        launch_with_workspace(device, args, _lib.beam_workspace_size, _lib.beam)
    return out, parents, tokens


def kv_cache_reorder(k_cache, v_cache, block_tables, seq_lens, parents, *, kv_scales=None):
    assert parents.dtype == torch.int32 and parents.dim() == 2, "parents must be int32 [batch, beams]"
    rows = parents.numel()
    assert parents.shape[1] <= MAX_BEAMS, f"at most {MAX_BEAMS} beams"
    assert block_tables.dim() == 2 and block_tables.shape[0] == rows and (
        rows == 0 or (block_tables.stride(1) == 1 and block_tables.stride(0) >= block_tables.shape[1])), \
        "block_tables must be int32 [batch * beams, max_blocks] with its rows one after another (it is changed in place)"
    assert seq_lens.dtype == torch.int32 and seq_lens.shape == (rows,), "seq_lens must be int32 [batch * beams]"
    cache_rows(_lib.kv_reorder, k_cache, v_cache, kv_scales, block_tables, seq_lens.contiguous(), parents, None)
