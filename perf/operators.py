"""Attention over a paged 8-bit KV cache and over packed prompts, as measurable cases.

Three operators that a step of a serving loop needs one after the other:

  append   K and V of new tokens into a paged cache of 8-bit codes (``int8`` or ``float8_e4m3fn``) with
           one fp32 scale per block of 16 positions and KV head.  A block that already holds tokens keeps
           the larger of its old scale and the one its new tokens ask for; where the scale grows, the old
           codes are rounded to it.
  decode   attention of one query token per sequence over that cache
  prefill  attention of packed prompts over their own keys and values, each sequence by itself

Scores of decode and prefill: ``s = scale * q.k``, capped to ``cap * tanh(s / cap)`` where a cap is given,
then a bias ``-slope[head] * |i - j|`` where slopes are given.  Query position i sees key position j when
``j <= i`` (``causal``) and ``|i - j| < window``, or when ``j < prefix``; a row that sees nothing is 0.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one pass, ``work`` what a pass cannot do without, ``exact``
the outputs from the definition in 64 bits.  Head counts are those of the other workloads: 32/8, 64/8 and
32/4 query / KV heads and what sharding leaves of them (16/2, 8/1).  K, V and q are N(0, 1), K scaled per
channel by log-normal(0, 0.75): a few channels are outliers.
"""
from __future__ import annotations

import math

import torch

own = False

HEAD_DIM, BLOCK = 128, 16
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
SCALE = HEAD_DIM ** -0.5
SMALLEST = 2.0 ** -100                       # magnitudes below it do not lower a block's scale any further
GEOMETRIES = ((32, 8), (64, 8), (32, 4), (16, 2), (8, 1))
MAX_APPEND_ROWS = 16384 * 8                  # (token, KV head) rows of the largest append
MAX_KV_ROWS = 4 * 8 * 65536                  # (position, KV head) rows of the largest decode step
MAX_PAIRS = 64 * 8192 * 8192 // 2            # (query head, row, key) triples of the largest prefill


def _text(numbers):
    """A list of lengths as a case holds it."""
    return ",".join(str(n) for n in numbers)


def _parsed(case):
    """The case with its lengths as lists of numbers."""
    return {k: [int(n) for n in v.split(",") if n] if k in ("lens", "olds", "news", "prefixes") else v for k, v in case.items()}


def listed():
    return [
        # one new token of each of four sequences: the smallest append of a serving loop
        dict(name="append_decode_tokens", kind="append", codes="int8", dtype="bf16", kv_heads=8, olds="32,37,44,46",
             news="1,1,1,1", layout="own"),
        # a prompt chunk into empty blocks, K and V as views into the projection's output
        dict(name="append_prompt_8k", kind="append", codes="int8", dtype="bf16", kv_heads=8, olds="0", news="8192", layout="qkv"),
        # chunks of several sequences that end and begin inside blocks, fp8 codes
        dict(name="append_chunks_ragged", kind="append", codes="e4m3", dtype="fp16", kv_heads=4,
             olds="0,5,16,131,40,0,77", news="701,1,1500,333,17,15,2048", layout="own"),
        # a short chat turn of one sequence: latency
        dict(name="decode_b1_500", kind="decode", codes="int8", dtype="bf16", heads=32, kv_heads=8, lens="500", softcap=0.0,
             alibi=False, window=0, prefix=0),
        # one long sequence on one GPU of eight
        dict(name="decode_shard_b1_128k", kind="decode", codes="e4m3", dtype="bf16", heads=8, kv_heads=1, lens="131072",
             softcap=0.0, alibi=False, window=0, prefix=0),
        # a batch of different lengths with capped scores
        dict(name="decode_b32_ragged_cap", kind="decode", codes="e4m3", dtype="fp16", heads=32, kv_heads=4,
             lens=_text(1 + (8190 * (i * i + 3 * i)) // (31 * 34) for i in range(32)), softcap=30.0, alibi=False, window=0, prefix=0),
        # a layer with a sliding window that keeps the first tokens, and a bias by distance
        dict(name="decode_b8_window_bias", kind="decode", codes="int8", dtype="bf16", heads=16, kv_heads=2,
             lens=_text(32768 - 911 * i for i in range(8)), softcap=0.0, alibi=True, window=4096, prefix=64),
        # the largest decode step: four sequences at 64k
        dict(name="decode_b4_64k", kind="decode", codes="int8", dtype="bf16", heads=64, kv_heads=8, lens="65536,65536,65536,65536",
             softcap=0.0, alibi=False, window=0, prefix=0),
        # a few short prompts in one step: latency
        dict(name="prefill_short", kind="prefill", dtype="bf16", heads=32, kv_heads=8, lens="5,64,129", causal=True,
             softcap=0.0, alibi=False, window=0, prefixes="", layout="own"),
        # documents of many lengths packed into one step, capped scores
        dict(name="prefill_documents_cap", kind="prefill", dtype="fp16", heads=32, kv_heads=4,
             lens="1999,127,1,640,2777,333,1500,64,900,3101,17,450", causal=True, softcap=50.0, alibi=False, window=0,
             prefixes="", layout="own"),
        # two prompts whose instructions are seen from both sides, local attention, bias by distance
        dict(name="prefill_prefix_window_bias", kind="prefill", dtype="bf16", heads=32, kv_heads=8, lens="6000,4211",
             causal=True, softcap=0.0, alibi=True, window=2048, prefixes="700,0", layout="qkv"),
        # the largest prefill: one prompt of 8k
        dict(name="prefill_8k", kind="prefill", dtype="bf16", heads=64, kv_heads=8, lens="8192", causal=True, softcap=0.0,
             alibi=False, window=0, prefixes="", layout="qkv"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cut(rng, total, n):
    """``n`` positive lengths of very different size that add up to ``total`` (at least ``n``)."""
    weights = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(n)]
    lens = [max(1, int(total * w / sum(weights))) for w in weights]
    lens[0] += max(0, total - sum(lens))
    return lens


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "prefill", "prefill"))
    dtype = rng.choice(("bf16", "fp16"))
    if kind == "append":
        kv = rng.choice((1, 2, 4, 8))
        n = _log_int(rng, 1, 64)
        if rng.random() < 0.4:
            news = [1] * n
        else:
            news = _cut(rng, _log_int(rng, n, 16384), n)
        olds = [rng.choice((0, _log_int(rng, 1, 200))) for _ in news]
        return dict(kind=kind, codes=rng.choice(tuple(CODES)), dtype=dtype, kv_heads=kv, olds=_text(olds), news=_text(news),
                    layout=rng.choice(("own", "qkv")))
    heads, kv = rng.choice(GEOMETRIES)
    softcap = rng.choice((0.0, 0.0, 15.0, 30.0, 50.0))
    alibi = rng.random() < 0.3
    if kind == "decode":
        n = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 1, min(131072, MAX_KV_ROWS // (kv * n)))
        lens = [ctx if rng.random() < 0.3 else _log_int(rng, 1, ctx) for _ in range(n)]
        window = rng.choice((0, 0, _log_int(rng, 16, 8192)))
        return dict(kind=kind, codes=rng.choice(tuple(CODES)), dtype=dtype, heads=heads, kv_heads=kv, lens=_text(lens), softcap=softcap,
                    alibi=alibi, window=window, prefix=rng.choice((0, _log_int(rng, 1, 256))) if window else 0)
    n = _log_int(rng, 1, 24)
    causal, prefixed = rng.random() < 0.85, rng.random() < 0.3
    longest = int(math.sqrt((2 if causal and not prefixed else 1) * MAX_PAIRS / heads))
    lens = _cut(rng, _log_int(rng, n, min(longest, 12000)), n)
    prefixes = [rng.choice((0, _log_int(rng, 1, l))) for l in lens] if prefixed else ()
    return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv, lens=_text(lens), causal=causal, softcap=softcap, alibi=alibi,
                window=rng.choice((0, 0, _log_int(rng, 16, 4096))), prefixes=_text(prefixes), layout=rng.choice(("own", "qkv")))


# ---- inputs -----------------------------------------------------------------------------


def _tokens(gen, tokens, heads, dtype, outliers):
    x = torch.randn(tokens, heads, HEAD_DIM, generator=gen, device="cuda")
    if outliers:
        x = x * torch.exp(0.75 * torch.randn(1, heads, HEAD_DIM, generator=gen, device="cuda"))
    return x.to(dtype)


def _qkv(gen, tokens, heads, kv, dtype, layout):
    """q, K and V of ``tokens`` tokens: tensors of their own, or views into one projection's output."""
    q, k, v = _tokens(gen, tokens, heads, dtype, False), _tokens(gen, tokens, kv, dtype, True), _tokens(gen, tokens, kv, dtype, False)
    if layout == "qkv":
        both = torch.cat([q, k, v], dim=1)
        q, k, v = both[:, :heads], both[:, heads:heads + kv], both[:, heads + kv:]
    return q, k, v


def _tables(gen, lens, spare):
    """Shuffled pages: the block table of sequences of ``lens`` positions, and the number of blocks."""
    need = [max(1, (l + BLOCK - 1) // BLOCK) for l in lens]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=gen, device="cuda")
    table = torch.zeros(len(lens), max(need), dtype=torch.int64, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, blocks


def _filled(gen, kv, blocks, codes, outliers):
    """A cache full of quantised rows: codes ``(kv, slots, 128)``, scales ``(kv, blocks)``."""
    data = torch.empty(kv, blocks * BLOCK, HEAD_DIM, dtype=CODES[codes], device="cuda")
    scales = torch.empty(kv, blocks, device="cuda")
    for h in range(kv):
        x = torch.randn(blocks, BLOCK, HEAD_DIM, generator=gen, device="cuda")
        if outliers:
            x = x * torch.exp(0.75 * torch.randn(1, 1, HEAD_DIM, generator=gen, device="cuda"))
        scales[h] = _block_scale(x.abs().amax(dim=(1, 2)), codes)
        data[h] = _encode(x * (1.0 / scales[h])[:, None, None], codes).view(-1, HEAD_DIM)
    return data, scales


def prepare(case, seed):
    case = _parsed(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dtype, kv = case["kind"], DTYPE[case["dtype"]], case["kv_heads"]
    st = dict(case=case)
    if kind == "append":
        lens = [o + n for o, n in zip(case["olds"], case["news"])]
        st["block_table"], blocks = _tables(gen, lens, 2)
        _, st["key"], st["value"] = _qkv(gen, sum(case["news"]), 2 * kv, kv, dtype, case["layout"])
        st["k_data"], st["k_scales"] = _filled(gen, kv, blocks, case["codes"], True)
        st["v_data"], st["v_scales"] = _filled(gen, kv, blocks, case["codes"], False)
        starts = [0]
        for n in case["news"]:
            starts.append(starts[-1] + n)
        st["query_start_loc"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return st
    heads = case["heads"]
    st["slopes"] = None
    if case["alibi"]:
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")
    if kind == "decode":
        n = len(case["lens"])
        st["block_table"], blocks = _tables(gen, case["lens"], 2)
        st["k_data"], st["k_scales"] = _filled(gen, kv, blocks, case["codes"], True)
        st["v_data"], st["v_scales"] = _filled(gen, kv, blocks, case["codes"], False)
        st["q"] = _tokens(gen, n, heads, dtype, False)
        st["seq_lens"] = torch.tensor(case["lens"], dtype=torch.int32, device="cuda")
        st["prefix_lens"] = torch.full((n,), case["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
        return st
    st["q"], st["k"], st["v"] = _qkv(gen, sum(case["lens"]), heads, kv, dtype, case["layout"])
    starts = [0]
    for n in case["lens"]:
        starts.append(starts[-1] + n)
    st["cu_seqlens"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    st["prefix_lens"] = None
    if case["prefixes"]:
        st["prefix_lens"] = torch.tensor(case["prefixes"], dtype=torch.int32, device="cuda")
    return st


# ---- one pass ---------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if kind == "append":
        (_own_append if own else _plain_append)(state)
        return (_values(state["k_data"], state["k_scales"]), state["k_scales"],
                _values(state["v_data"], state["v_scales"]), state["v_scales"])
    if kind == "decode":
        return (_own_decode if own else _plain_decode)(state)
    return (_own_prefill if own else _plain_prefill)(state)


def _values(data, scales):
    """What the codes of a cache stand for."""
    kv, blocks = scales.shape
    return data.view(kv, blocks, BLOCK, HEAD_DIM).float() * scales[:, :, None, None]


def _own_append(st):
    from jetfire_b200 import ops
    ops.block8_append(st["key"], st["value"], st["query_start_loc"], st["seq_lens"], st["block_table"], st["k_data"],
                      st["k_scales"], st["v_data"], st["v_scales"])


def _own_decode(st):
    from jetfire_b200 import ops
    c = st["case"]
    return ops.block8_decode_attn(st["q"], st["k_data"], st["k_scales"], st["v_data"], st["v_scales"], st["block_table"],
                                  st["seq_lens"], max(c["lens"]), c["heads"], c["kv_heads"], BLOCK, SCALE, softcap=c["softcap"],
                                  alibi_slopes=st["slopes"], window=c["window"] or None, prefix_lens=st["prefix_lens"])


def _own_prefill(st):
    from jetfire_b200 import ops
    c = st["case"]
    return ops.varlen_prefill_attn(st["q"], st["k"], st["v"], st["cu_seqlens"], SCALE, causal=c["causal"],
                                   softcap=c["softcap"], alibi_slopes=st["slopes"], window=c["window"] or None,
                                   prefix_lens=st["prefix_lens"])


# the plain forms: elementary operations in 32 bits


def _block_scale(amax, codes):
    amax = amax.float().clamp(min=SMALLEST)
    if codes == "int8":
        return amax / torch.full_like(amax, 127.0)       # (a number would be multiplied by its inverse: not the quotient)
    # fp8: the smallest power of two that brings the largest magnitude to at most 448 = 1.75 * 2^8
    mantissa, exponent = torch.frexp(amax)               # mantissa in [0.5, 1)
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    return torch.ldexp(torch.ones_like(amax), exponent)


def _encode(scaled, codes):
    top = CODE_MAX[codes]
    scaled = torch.nan_to_num(scaled, nan=0.0, posinf=top, neginf=-top).clamp(-top, top)
    return scaled.round().to(torch.int8) if codes == "int8" else scaled.to(torch.float8_e4m3fn)


def _plain_append(st):
    codes = st["case"]["codes"]
    start, lens = st["query_start_loc"].long(), st["seq_lens"].long()
    token = torch.arange(st["key"].shape[0], device="cuda")
    seq = (token[:, None] >= start[None, 1:]).sum(1)
    pos = lens[seq] - (start[seq + 1] - token)
    block, row = st["block_table"][seq, pos // BLOCK], pos % BLOCK
    for x, data, scales in ((st["key"], st["k_data"], st["k_scales"]), (st["value"], st["v_data"], st["v_scales"])):
        kv, blocks = scales.shape
        x = x.float()
        size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(2)                       # (T, kv)
        amax = torch.zeros(blocks, kv, device="cuda").index_reduce_(0, block, size, "amax").t()
        first = torch.full((blocks,), BLOCK, device="cuda").index_reduce_(0, block, row, "amin")
        touched = first < BLOCK
        keeps = touched & (first > 0) & torch.isfinite(scales) & (scales > 0)
        old = torch.where(keeps, scales, torch.zeros_like(scales))
        new = torch.where(touched, torch.maximum(old, _block_scale(amax, codes)), scales)
        rows = data.view(kv, blocks, BLOCK, HEAD_DIM)
        live = touched[:, None] & (torch.arange(BLOCK, device="cuda")[None] < first[:, None])             # (blocks, 16)
        ratio = torch.where(keeps, old / new, torch.zeros_like(new))
        moved = _encode(rows.float() * ratio[:, :, None, None], codes)
        take = live[None, :, :, None].expand_as(rows)
        # (fp8 has no masked selection: bytes)
        rows.view(torch.int8).copy_(torch.where(take, moved.view(torch.int8), rows.view(torch.int8)))
        scales.copy_(new)
        fresh = _encode(x * (1.0 / new[:, block]).t()[:, :, None], codes)                                 # (T, kv, 128)
        data.view(torch.int8)[:, block * BLOCK + row] = fresh.view(torch.int8).transpose(0, 1)


def _scores(s, i, j, softcap, slopes, causal, window, prefix):
    """Capped, biased and masked scores ``(heads, rows, keys)`` of positions ``i`` and ``j``."""
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    apart = i[:, None] - j[None, :]
    if slopes is not None:
        s = s - slopes[:, None, None] * apart.abs()
    sees = torch.ones_like(apart, dtype=torch.bool)
    if causal:
        sees &= apart >= 0
    if window:
        sees &= apart.abs() < window
    sees |= (j < prefix)[None, :]
    return s.masked_fill(~sees, float("-inf"))


def _weights(s):
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    z = p.sum(-1, keepdim=True)
    lse = (top + torch.log(z)).squeeze(-1)
    return p / torch.where(z == 0, torch.ones_like(z), z), lse


def _plain_decode(st):
    c = st["case"]
    heads, kv, group = c["heads"], c["kv_heads"], c["heads"] // c["kv_heads"]
    out = torch.zeros(len(c["lens"]), heads, HEAD_DIM, device="cuda")
    lse = torch.full((len(c["lens"]), heads), float("-inf"), device="cuda")
    for b, n in enumerate(c["lens"]):
        j = torch.arange(n, device="cuda")
        blocks = st["block_table"][b, j // BLOCK]
        slots = blocks * BLOCK + j % BLOCK
        bytes_k, bytes_v = st["k_data"].view(torch.int8)[:, slots], st["v_data"].view(torch.int8)[:, slots]
        k = bytes_k.view(st["k_data"].dtype).float() * st["k_scales"][:, blocks, None]
        v = bytes_v.view(st["v_data"].dtype).float() * st["v_scales"][:, blocks, None]
        s = SCALE * (st["q"][b].float().view(kv, group, HEAD_DIM) @ k.transpose(1, 2))                    # (kv, group, n)
        s = _scores(s.view(heads, 1, n), j[-1:], j, c["softcap"], st["slopes"], True, c["window"], c["prefix"])
        p, lse_b = _weights(s)
        out[b] = (p.view(kv, group, n) @ v).view(heads, HEAD_DIM)
        lse[b] = lse_b[:, 0]
    return out.to(st["q"].dtype), lse


def _plain_prefill(st):
    c = st["case"]
    heads, kv, group = c["heads"], c["kv_heads"], c["heads"] // c["kv_heads"]
    out = torch.empty(sum(c["lens"]), heads, HEAD_DIM, device="cuda")
    lse = torch.empty(sum(c["lens"]), heads, device="cuda")
    lo = 0
    for b, n in enumerate(c["lens"]):
        i = torch.arange(n, device="cuda")
        prefix = c["prefixes"][b] if c["prefixes"] else 0
        rows = slice(lo, lo + n)
        for g in range(kv):
            hs = slice(g * group, (g + 1) * group)
            q, k, v = st["q"][rows, hs].float().transpose(0, 1), st["k"][rows, g].float(), st["v"][rows, g].float()
            slopes = st["slopes"][hs] if st["slopes"] is not None else None
            p, lse_g = _weights(_scores(SCALE * (q @ k.t()), i, i, c["softcap"], slopes, c["causal"], c["window"], prefix))
            out[rows, hs] = (p @ v).transpose(0, 1)
            lse[rows, hs] = lse_g.t()
        lo += n
    return out.to(st["q"].dtype), lse


# ---- what a pass cannot do without ---------------------------------------------------------


def _seen(n, causal, window, prefix):
    """Pairs (i, j) of a sequence of ``n`` positions in which i sees j."""
    if causal and not window:                     # j <= i, and the prefix's positions behind i
        p = min(prefix, n)
        return n * (n + 1) // 2 + p * (p - 1) // 2
    total = 0
    for i in range(n):
        lo = max(0, i - window + 1) if window else 0
        hi = i if causal else (min(n - 1, i + window - 1) if window else n - 1)
        p = min(prefix, n)
        total += hi - lo + 1 + min(p, lo) + max(0, p - 1 - hi)
    return total


def work(case):
    case = _parsed(case)
    kind, kv = case["kind"], case["kv_heads"]
    if kind == "append":
        rows = sum(case["news"]) * kv * 2                              # of K and V
        old = touched = 0
        for o, n in zip(case["olds"], case["news"]):
            old += o % BLOCK
            touched += (o + n - 1) // BLOCK - o // BLOCK + 1
        return dict(bytes=rows * HEAD_DIM * 3 + 2 * kv * (4 * touched + 2 * HEAD_DIM * old), flops=rows * HEAD_DIM * 3)
    heads = case["heads"]
    if kind == "decode":
        seen = [min(n, case["window"] + min(case["prefix"], max(0, n - case["window"]))) if case["window"] else n for n in case["lens"]]
        cache = sum(2 * kv * (s * HEAD_DIM + 4 * ((s + BLOCK - 1) // BLOCK)) for s in seen)
        return dict(bytes=cache + len(seen) * heads * (4 * HEAD_DIM + 4), flops=4 * HEAD_DIM * heads * sum(seen))
    tokens = sum(case["lens"])
    prefixes = case["prefixes"] or [0] * len(case["lens"])
    pairs = sum(_seen(n, case["causal"], case["window"], p) for n, p in zip(case["lens"], prefixes))
    return dict(bytes=tokens * (HEAD_DIM * 4 * (heads + kv) + 4 * heads), flops=4 * HEAD_DIM * heads * pairs)


# ---- the definition in 64 bits ------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    case = st["case"]
    if case["kind"] == "append":
        return _exact_append(st, case)
    return _exact_decode(st, case) if case["kind"] == "decode" else _exact_prefill(st, case)


def _fl32(x):
    return x.to(torch.float32).to(torch.float64)


def _exact_append(st, case):
    """Sequence by sequence and block by block.  Scales, their reciprocals and the scaled values are fp32
    numbers by definition, so each is rounded to fp32 here too (the 64-bit value before it is exact, or
    a quotient, which no second rounding moves)."""
    top = CODE_MAX[case["codes"]]
    as_codes = (lambda x: x.clamp(-top, top).round()) if case["codes"] == "int8" else \
        (lambda x: x.clamp(-top, top).float().to(torch.float8_e4m3fn).double())
    table = st["block_table"].tolist()
    out = []
    for x, data, scales in ((st["key"], st["k_data"], st["k_scales"]), (st["value"], st["v_data"], st["v_scales"])):
        kv, blocks = scales.shape
        x = x.double()
        code = data.float().double().view(kv, blocks, BLOCK, HEAD_DIM)
        scale = scales.double()
        token = 0
        for b, (old, new) in enumerate(zip(case["olds"], case["news"])):
            pos, end = old, old + new
            while pos < end:
                row, n = pos % BLOCK, min(BLOCK - pos % BLOCK, end - pos)
                if row == 0 and end - pos >= BLOCK:            # all whole blocks at once
                    n = (end - pos) // BLOCK * BLOCK
                ids = torch.tensor(table[b][pos // BLOCK:(pos + n - 1) // BLOCK + 1], device="cuda")
                m = ids.numel()
                rows = x[token:token + n].transpose(0, 1).reshape(kv, m, n // m, HEAD_DIM)
                amax = rows.abs().amax(dim=(2, 3)).clamp(min=SMALLEST)
                if case["codes"] == "int8":
                    want = _fl32(amax / 127.0)
                else:
                    want = torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
                    want = torch.where(want * 448.0 < amax, want * 2.0, torch.where(want * 224.0 >= amax, want / 2.0, want))
                if row:
                    was = scale[:, ids]
                    want = torch.maximum(want, was)
                    ratio = _fl32(was / want)
                    code[:, ids, :row] = as_codes(_fl32(code[:, ids, :row] * ratio[:, :, None, None]))
                code[:, ids, row:row + n // m] = as_codes(_fl32(rows * _fl32(1.0 / want)[:, :, None, None]))
                scale[:, ids] = want
                pos, token = pos + n, token + n
        out += [code * scale[:, :, None, None], scale]
    return tuple(out)


def _attend64(q, k, v, i, j, case, slopes, causal, prefix):
    """One query head: rows ``q`` at positions ``i`` over keys at positions ``j``."""
    s = (q @ k.t()) * SCALE
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    d = (j[None, :] - i[:, None]).double()
    if slopes is not None:
        s += -d.abs() * slopes
    hidden = torch.zeros_like(s, dtype=torch.bool)
    if causal:
        hidden |= d > 0
    if case["window"]:
        hidden |= d.abs() >= case["window"]
    hidden &= (j >= prefix)[None, :]
    s[hidden] = float("-inf")
    lse = torch.logsumexp(s, 1)
    return torch.exp(s - lse[:, None]) @ v, lse


def _exact_decode(st, case):
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(len(case["lens"]), heads, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.full((len(case["lens"]), heads), float("-inf"), dtype=torch.float64, device="cuda")
    for b, n in enumerate(case["lens"]):
        ids = st["block_table"][b, :(n + BLOCK - 1) // BLOCK]
        j = torch.arange(n, device="cuda")
        for g in range(case["kv_heads"]):
            k = (st["k_data"][g].view(-1, BLOCK, HEAD_DIM).view(torch.int8)[ids].view(st["k_data"].dtype).double()
                 * st["k_scales"][g, ids].double()[:, None, None]).view(-1, HEAD_DIM)[:n]
            v = (st["v_data"][g].view(-1, BLOCK, HEAD_DIM).view(torch.int8)[ids].view(st["v_data"].dtype).double()
                 * st["v_scales"][g, ids].double()[:, None, None]).view(-1, HEAD_DIM)[:n]
            for h in range(g * group, (g + 1) * group):
                slope = st["slopes"][h].double() if st["slopes"] is not None else None
                o, l = _attend64(st["q"][b, h:h + 1].double(), k, v, j[-1:], j, case, slope, True, case["prefix"])
                out[b, h], lse[b, h] = o[0], l[0]
    return out, lse


def _exact_prefill(st, case):
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(sum(case["lens"]), heads, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.empty(sum(case["lens"]), heads, dtype=torch.float64, device="cuda")
    lo = 0
    for b, n in enumerate(case["lens"]):
        prefix = case["prefixes"][b] if case["prefixes"] else 0
        at = torch.arange(n, device="cuda")
        for h in range(heads):
            q, k, v = (t.double() for t in (st["q"][lo:lo + n, h], st["k"][lo:lo + n, h // group], st["v"][lo:lo + n, h // group]))
            slope = st["slopes"][h].double() if st["slopes"] is not None else None
            for r in range(0, n, 4096):
                part = slice(r, min(n, r + 4096))
                o, l = _attend64(q[part], k, v, at[part], at, case, slope, case["causal"], prefix)
                out[lo + r:lo + part.stop, h], lse[lo + r:lo + part.stop, h] = o, l
        lo += n
    return out, lse
