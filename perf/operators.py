"""An 8-bit paged KV cache, and attention with a sliding window over paged caches, as cases that a measuring program can time and compare.

Four operators, each reached through a public entry point:

  append   kv_cache_append: the K and V rows of new tokens, quantised to e4m3 with a power-of-two scale a row, into a paged cache
  read     kv_cache_read: cached rows back as packed K and V of 16 or 32 bits
  decode   paged_attention_decode: one new token per sequence against an 8- or 16-bit paged cache, under a sliding window with
           sinks (a few first tokens that stay visible) or none
  chunk    paged_prefill: the same for chunks of new tokens

A row of K or V is the head_dim values of one token and KV head. Its scale s is the least power of two that brings the row's
largest finite magnitude within 448 s (e4m3's largest value); stored is the exponent plus 127, at least 1. Codes are x / s rounded
to nearest even, NaN for infinities and NaN. Where 256 s does not fit the rows' own type, magnitudes are held to 240 s, so that
what a row stands for always fits it. A query at position p sees key j where j <= p and (j > p - window or j < sinks).

listed() names twelve cases; draw() gives others of the same ranges. Sizes are those of this repository's workloads
(lightserve_amd/workloads.py, model/minimal_llama.py) and tests, or generic ones. Lengths are spread evenly from the shortest
to the longest, so that a case's work is known without its inputs.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
# Scale exponent (plus 127) of the topmost rows, whose codes stop at 240.
TOP = {torch.float32: 247, torch.bfloat16: 247, torch.float16: 135}


def listed():
    return [
        # One decode step of eight requests at LLaMA-3-8B's layer shape: the smallest call, latency.
        dict(name="append_step_bf16", op="append", dtype="bf16", sequences=8, shortest=1, longest=1, cached=1500, kv_heads=8,
             dim=128, block=16),
        # Prefill chunks of odd lengths with a head dim between the tile widths.
        dict(name="append_chunks_odd_fp16", op="append", dtype="fp16", sequences=9, shortest=1, longest=777, cached=2100,
             kv_heads=3, dim=80, block=32),
        # Four whole prompts in one prefill.
        dict(name="append_prompts_bf16", op="append", dtype="bf16", sequences=4, shortest=8192, longest=8192, cached=0,
             kv_heads=8, dim=128, block=16),
        # The cached prefixes of a batch, back as packed rows for the packed attention.
        dict(name="read_prefixes_bf16", op="read", dtype="bf16", sequences=8, shortest=1024, longest=8192, kv_heads=8, dim=128,
             block=16),
        # One short, odd-sized sequence.
        dict(name="read_single_fp16", op="read", dtype="fp16", sequences=1, shortest=333, longest=333, kv_heads=3, dim=96,
             block=64),
        # One request's decode step over the 8-bit cache: latency.
        dict(name="decode_single_bf16", op="decode", dtype="bf16", cache="e4m3", sequences=1, shortest=1500, longest=1500,
             heads=32, kv_heads=8, dim=128, block=16, window=0, sinks=0, lse=False),
        # A batch of ordinary requests over the 8-bit cache.
        dict(name="decode_batch_bf16", op="decode", dtype="bf16", cache="e4m3", sequences=32, shortest=1024, longest=8192,
             heads=32, kv_heads=8, dim=128, block=16, window=0, sinks=0, lse=False),
        # Long contexts of which a window stays; the blocks that left it have been given back to the pool.
        dict(name="decode_window_bf16", op="decode", dtype="bf16", cache="e4m3", sequences=64, shortest=8192, longest=131072,
             heads=32, kv_heads=8, dim=128, block=16, window=4096, sinks=4, lse=True),
        # A window over a 16-bit cache, heads in groups of seven, some sequences shorter than the window.
        dict(name="decode_window_odd_fp16", op="decode", dtype="fp16", cache="16 bit", sequences=16, shortest=500,
             longest=14502, heads=14, kv_heads=2, dim=64, block=16, window=1000, sinks=1, lse=False),
        # A batch of prefill chunks against long 8-bit prefixes (the repository's chunked prefill workload).
        dict(name="chunk_batch_bf16", op="chunk", dtype="bf16", cache="e4m3", sequences=8, new_shortest=512, new_longest=512,
             shortest=1024, longest=8192, heads=32, kv_heads=8, dim=128, block=16, window=0, sinks=0, lse=False),
        # One request's odd-sized chunk under a window.
        dict(name="chunk_window_single_bf16", op="chunk", dtype="bf16", cache="e4m3", sequences=1, new_shortest=333,
             new_longest=333, shortest=6011, longest=6011, heads=32, kv_heads=8, dim=128, block=16, window=1024, sinks=4,
             lse=True),
        # Whole prompts longer than the window over a 16-bit cache, every head with keys of its own.
        dict(name="chunk_window_prompts_fp16", op="chunk", dtype="fp16", cache="16 bit", sequences=2, new_shortest=3900,
             new_longest=4096, shortest=0, longest=130, heads=16, kv_heads=16, dim=64, block=32, window=2048, sinks=16,
             lse=False),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "chunk"])
    c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), block=rng.choice([16, 32, 64]))
    kv_heads, dim = rng.choice([1, 2, 3, 8, 16]), rng.choice([64, 80, 96, 112, 128])
    if op in ("append", "read"):
        c["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
        c["sequences"] = _spread(rng, 1, 48)
        most = max(1, min(8192, 20_000_000 // (c["sequences"] * kv_heads * dim)))
        c["longest"] = _spread(rng, 1, most)
        c["shortest"] = rng.randint(0, c["longest"])
        if op == "append":
            c["cached"] = rng.choice([0, _spread(rng, 1, 4000)])
        return c | dict(kv_heads=kv_heads, dim=dim)
    group = rng.choice([1, 2, 3, 4, 7, 8])
    c |= dict(cache=rng.choice(["e4m3", "e4m3", "16 bit"]), heads=kv_heads * group, kv_heads=kv_heads, dim=dim)
    c |= dict(window=_spread(rng, 1, 4096), sinks=rng.choice([0, 1, 4, rng.randint(5, 70)])) if c["cache"] != "e4m3" or rng.random() < 0.6 \
        else dict(window=0, sinks=0)
    c["lse"] = rng.random() < 0.5
    if op == "decode":
        c["sequences"] = _spread(rng, 1, 64)
        most = 65536 if c["window"] else max(64, min(32768, 150_000_000 // (c["sequences"] * kv_heads * dim)))
        c["longest"] = _spread(rng, 1, most)
        c["shortest"] = rng.randint(0, c["longest"])
        return c
    c["sequences"] = _spread(rng, 1, 12)
    c["new_longest"] = _spread(rng, 2, max(2, min(4096, 120_000 // (c["sequences"] * c["heads"]))))
    c["new_shortest"] = rng.randint(0, c["new_longest"])
    c["longest"] = _spread(rng, 1, 8192)
    c["shortest"] = rng.randint(0, c["longest"])
    return c


# ------------------------------------------------------------------ sizes
def _lengths(shortest, longest, n):
    return [longest if n == 1 else shortest + (longest - shortest) * i // (n - 1) for i in range(n)]


def _sizes(case):
    """(new tokens, tokens in the cache once the new ones are there) of each sequence."""
    n = case["sequences"]
    if case["op"] == "append":
        new = _lengths(case["shortest"], case["longest"], n)
        return new, [a + b for a, b in zip(new, _lengths(0, case["cached"], n)[::-1])]
    if case["op"] == "chunk":
        new = _lengths(case["new_shortest"], case["new_longest"], n)
        return new, [a + b for a, b in zip(new, _lengths(case["shortest"], case["longest"], n))]
    lens = _lengths(case["shortest"], case["longest"], n)
    return ([1] * n if case["op"] == "decode" else lens), lens


def _visible(p, window, sinks):
    """Keys that a query at position p sees."""
    if p < 0:
        return 0
    if not window or window > p:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(case):
    new, lens = _sizes(case)
    kv, d = case["kv_heads"], case["dim"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] in ("append", "read"):
        rows = sum(new) * kv
        return {"bytes": rows * (2 * d * (size + 1) + 2), "flops": rows * 4 * d}
    row = 2 * d + 2 if case["cache"] == "e4m3" else 4 * d
    seen = keys = 0
    for n, length in zip(new, lens):
        w, s, first = case["window"], case["sinks"], length - n
        seen += sum(_visible(p, w, s) for p in range(first, length))
        low = max(0, first - w + 1) if w else 0
        keys += length - low + min(s, low) if n else 0
    tokens = sum(new)
    return {"bytes": keys * kv * row + 2 * tokens * case["heads"] * d * size, "flops": 4 * d * case["heads"] * seen}


# ----------------------------------------------------------------- inputs
def _rows(gen, n, heads, dim, dtype, mul):
    """[n, heads, dim] as a projection leaves K or V: normal values, a few channels far larger than the rest."""
    x = torch.randn(n, heads, dim, generator=gen, device="cuda") * mul
    x[:, :, ::dim // 5] *= 6
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    new, lens = _sizes(case)
    n, block, kv, d, dtype = case["sequences"], case["block"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    # Tables over a shuffled pool. Blocks that no query of the call can see any more are not in it (-1).
    have = []
    for a, length in zip(new, lens):
        low = max(0, length - a - window + 1) if window else 0
        have.append([i for i in range(-(-length // block)) if (i + 1) * block > low or i * block < sinks])
    order = torch.randperm(sum(map(len, have)) + 3, generator=host, dtype=torch.int32)
    table = torch.full((n, max([1] + [-(-length // block) for length in lens])), -1, dtype=torch.int32)
    at = 0
    for b, held in enumerate(have):
        table[b, held] = order[at:at + len(held)]
        at += len(held)
    s = dict(case=case, block_tables=table.cuda(), seq_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
             cu=torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32).cuda(), total=sum(new),
             longest=max(lens), longest_new=max(new), dtype=dtype, window=window or None, sinks=sinks)
    blocks = order.numel()
    if case["op"] == "append":
        s["k"], s["v"] = (_rows(gen, s["total"], kv, d, dtype, m) for m in (0.5, 1.0))
        codes = torch.randint(0, 127, (2, blocks, block, kv, d), generator=gen, device="cuda", dtype=torch.uint8)
        s["k_cache"], s["v_cache"] = codes.view(E4M3).unbind(0)
        s["kv_scales"] = torch.randint(110, 130, (blocks, kv, block, 2), generator=gen, device="cuda", dtype=torch.uint8)
        return s
    k, v = (_rows(gen, blocks * block, kv, d, dtype, m) for m in (0.5, 1.0))
    s["kv_scales"] = None
    if case["op"] == "read" or case["cache"] == "e4m3":
        (k, ks), (v, vs) = _quantise(k), _quantise(v)
        s["kv_scales"] = torch.stack([ks, vs], -1).view(blocks, block, kv, 2).transpose(1, 2).contiguous()
    s["k_cache"], s["v_cache"] = k.view(blocks, block, kv, d), v.view(blocks, block, kv, d)
    if case["op"] != "read":
        s["q"] = (torch.randn(s["total"], case["heads"], d, generator=gen, device="cuda") * 0.7).to(dtype)
    return s


# ------------------------------------------------------------ plain forms
def _power(e):
    """2^(e - 127) in fp32, from its bits (torch.ldexp and pow are an ulp off here and there)."""
    return (e.int() << 23).view(torch.float32)


def _quantise(x):
    """e4m3 codes of x [..., head_dim], and the exponents (plus 127) of its rows' scales."""
    f = x.float()
    largest = torch.where(f.isfinite(), f.abs(), 0).amax(-1, keepdim=True)
    mantissa, power = torch.frexp(largest)  # 448 is 0.875 * 2^9
    e = torch.where(largest > 0, power - 9 + (mantissa > 0.875) + 127, 1).clamp(1, 254)
    most = torch.where(e >= TOP[x.dtype], 240.0, 448.0)
    y = torch.where(f.isfinite(), (f * _power(254 - e)).clamp(-most, most), math.nan)
    return y.to(E4M3), e.squeeze(-1).to(torch.uint8)


def _token_places(s):
    """Sequence and index of each token of packed rows."""
    t = torch.arange(s["total"], device="cuda")
    b = torch.bucketize(t, s["cu"][1:].long(), right=True)
    return b, t - s["cu"].long()[b]


def _slots(s, b, position):
    block = s["case"]["block"]
    return s["block_tables"][b, position // block].long() * block + position % block


def _append(s):
    b, i = _token_places(s)
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    slot = _slots(s, b, s["seq_lens"].long()[b] - n[b] + i)
    block = s["case"]["block"]
    (k, ks), (v, vs) = _quantise(s["k"]), _quantise(s["v"])
    s["k_cache"].view(torch.uint8).flatten(0, 1)[slot] = k.view(torch.uint8)
    s["v_cache"].view(torch.uint8).flatten(0, 1)[slot] = v.view(torch.uint8)
    s["kv_scales"][slot // block, :, slot % block] = torch.stack([ks, vs], -1)
    return s["k_cache"], s["v_cache"], s["kv_scales"]


def _rows_at(s, slot):
    """K and V rows of the cache slots, in fp32."""
    k, v = (s[name].view(torch.uint8).flatten(0, 1)[slot].view(E4M3).float() if s["kv_scales"] is not None
            else s[name].flatten(0, 1)[slot].float() for name in ("k_cache", "v_cache"))
    if s["kv_scales"] is None:
        return k, v
    block = s["case"]["block"]
    scale = _power(s["kv_scales"][slot // block, :, slot % block])
    return k * scale[..., :1], v * scale[..., 1:]


def _read(s):
    b, i = _token_places(s)
    k, v = _rows_at(s, _slots(s, b, i))
    return k.to(s["dtype"]), v.to(s["dtype"])


def _attention(s):
    """Over the rows that some query of a sequence may see, padded to the longest."""
    case, lens = s["case"], s["seq_lens"].long()
    decode, window, sinks = case["op"] == "decode", s["window"], s["sinks"]
    B, kv, group, d = case["sequences"], case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    n = torch.ones_like(lens) if decode else (s["cu"][1:] - s["cu"][:-1]).long()
    most = 1 if decode else s["longest_new"]
    at = torch.arange(s["longest"], device="cuda").expand(B, -1)
    if window is not None and sinks + window + most - 1 < s["longest"]:
        low = (lens - n - window + 1).clamp(min=sinks)
        at = torch.cat([torch.arange(sinks, device="cuda").expand(B, -1),
                        low[:, None] + torch.arange(window + most - 1, device="cuda")], 1)
    held = at < lens[:, None]
    slot = _slots(s, torch.arange(B, device="cuda")[:, None], torch.where(held, at, 0))
    k, v = _rows_at(s, torch.where(held, slot, 0).clamp(min=0))
    k, v = torch.where(held[..., None, None], k, 0), torch.where(held[..., None, None], v, 0)
    tb, ti = _token_places(s)
    q = torch.zeros(B, most, case["heads"], d, device="cuda")
    q[tb, ti] = s["q"].float()
    q = q.view(B, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(B, kv, group * most, d)
    p = (lens - n)[:, None] + torch.arange(most, device="cuda")
    seen = held[:, None] & (at[:, None] <= p[..., None])
    if window is not None:
        seen &= (at[:, None] > p[..., None] - window) | (at[:, None] < sinks)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1 / math.sqrt(d)).view(B, kv, group, most, -1)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, kv, group * most, -1), v.transpose(1, 2)).view(B, kv, group, most, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, -1, d)[tb, ti].to(s["dtype"])
    lse = (top + total.log()).view(B, -1, most).transpose(1, 2)[tb, ti]
    return (o, lse if decode else lse.T.contiguous()) if case["lse"] else o


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _append, "read": _read, "decode": _attention, "chunk": _attention}[op](s)
    from lightserve_amd.kernels.paged_attention import paged_attention_decode, paged_prefill
    from lightserve_amd.kernels.quantized_kv_cache import kv_cache_append, kv_cache_read
    cache = s["k_cache"], s["v_cache"]
    if op == "append":
        kv_cache_append(s["k"], s["v"], *cache, s["kv_scales"], s["block_tables"], s["seq_lens"], s["cu"])
        return *cache, s["kv_scales"]
    if op == "read":
        return kv_cache_read(*cache, s["kv_scales"], s["block_tables"], s["cu"], total=s["total"], dtype=s["dtype"])
    how = dict(kv_scales=s["kv_scales"], window=s["window"], sinks=s["sinks"], return_lse=s["case"]["lse"])
    if op == "decode":
        return paged_attention_decode(s["q"], *cache, s["block_tables"], s["seq_lens"], max_seq_len=s["longest"], **how)
    return paged_prefill(s["q"], *cache, s["block_tables"], s["cu"], s["seq_lens"], max_seqlen_q=s["longest_new"], **how)


# ---------------------------------------------------------------- 64 bits
def _two_to(n):
    """2^n in 64 bits for whole numbers n, without a rounding."""
    return (n.long() + 1023 << 52).view(torch.double)


def _exact_codes(x):
    """The e4m3 values (in 64 bits) that rows x stand for once divided by their scales."""
    y = x.double()
    largest = torch.nan_to_num(y, nan=0.0, posinf=0.0, neginf=0.0).abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(largest.clamp(min=1e-300) / 448)).clamp(-126, 127)
    e = torch.where(largest <= 448 * _two_to(e - 1), e - 1, e).clamp(-126, 127)  # log2 near a whole number
    y = y / _two_to(e)
    top = (_two_to(e) * 256 > torch.finfo(x.dtype).max).expand_as(y)
    y = torch.where(top, y.clamp(-240, 240), y)
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = _two_to(torch.where(_two_to(power) > y.abs().clamp(min=2.0 ** -6), power - 1, power) - 3)
    return torch.where(x.isfinite(), torch.round(y / step) * step, math.nan)


def exact(case, seed):
    s = prepare(case, seed)
    block, kv, d = case["block"], case["kv_heads"], case["dim"]
    table, cu, lens = s["block_tables"].tolist(), s["cu"].tolist(), s["seq_lens"].tolist()

    def slots(b, low, high):
        return torch.tensor([table[b][p // block] * block + p % block for p in range(low, high)], device="cuda",
                            dtype=torch.long)

    values = [s[name].double().flatten(0, 1) for name in ("k_cache", "v_cache")]
    if case["op"] == "append":
        for b, length in enumerate(lens):
            at = slots(b, length - (cu[b + 1] - cu[b]), length)
            for value, rows in zip(values, (s["k"], s["v"])):
                value[at] = _exact_codes(rows[cu[b]:cu[b + 1]])
        return *(value.view(s["k_cache"].shape) for value in values), None
    if s["kv_scales"] is not None:
        scale = _two_to(s["kv_scales"].long() - 127)
        values = [value * scale[..., i].transpose(1, 2).flatten(0, 1)[..., None] for i, value in enumerate(values)]
    k, v = values
    if case["op"] == "read":
        at = torch.cat([slots(b, 0, length) for b, length in enumerate(lens)])
        return k[at], v[at]
    window, sinks, group = s["window"], s["sinks"], case["heads"] // kv
    out = torch.zeros(s["total"], case["heads"], d, device="cuda", dtype=torch.double)
    log = torch.full((s["total"], case["heads"]), -math.inf, device="cuda", dtype=torch.double)
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if not n or not length:
            continue
        low = max(0, length - n - window + 1) if window else 0
        places = list(range(min(sinks, low))) + list(range(low, length))
        at = torch.cat([slots(b, 0, min(sinks, low)), slots(b, low, length)])
        j = torch.tensor(places, device="cuda")
        p = torch.arange(length - n, length, device="cuda")
        hidden = j > p[:, None]
        if window:
            hidden |= (j <= p[:, None] - window) & (j >= sinks)
        for h in range(case["heads"]):
            x = s["q"][cu[b]:cu[b + 1], h].double() @ k[at, h // group].T.contiguous() / math.sqrt(d)
            x[hidden] = -math.inf
            log[cu[b]:cu[b + 1], h] = x.logsumexp(1)
            out[cu[b]:cu[b + 1], h] = torch.softmax(x, 1).nan_to_num(0.0) @ v[at, h // group]
    if not case["lse"]:
        return out
    return out, log if case["op"] == "decode" else log.T.contiguous()
