"""Three more operators over a paged 8-bit KV cache, as measurable cases.

The cache holds K and V as 8-bit codes (``int8`` or ``float8_e4m3fn``) with one fp32 scale per block of 16 positions
and KV head.  A serving step rotates and appends, then attends:

  rotary   the step's queries and keys are rotated by their positions, K (from fp32, without a rounding in between) and V
           go into the cache; with block bounds, the lowest and highest code of every block and channel
           are kept as ``int8``
  shared   one query token per sequence over a prefix that all sequences share and the sequence's own positions
  sparse   one query token per sequence over the blocks of its cache that score best by their bounds: for every query head the
           query in 8 bits against the bounds, an upper bound of ``q.k`` over the block, the best head of a KV
           head counts; the first and last blocks always

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges, ``prepare`` makes what a program holds before
the call, ``run`` is one pass, ``work`` what a pass cannot do without, ``exact`` the outputs from the definition in 64
bits.  Head counts are those of the other workloads: 32/8, 64/8 and 32/4 query / KV heads and what sharding leaves of
them (16/2, 8/1).  q and V are N(0, 1), K too with channels scaled by log-normal(0, 0.75); for ``sparse`` the keys
of a block have a mean of their own.
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
SMALLEST = 2.0 ** -100                       # magnitudes below it do not lower a scale any further
GEOMETRIES = ((32, 8), (64, 8), (32, 4), (16, 2), (8, 1))
MAX_ROTARY_ROWS = 8192 * 80                  # (token, head) rows of the largest rotation and append
MAX_SHARED = 256 * 64 * 65536                # (sequence, query head, shared position) triples of the largest shared step
MAX_OWN = 256 * 512                          # own positions of all sequences, each counted as the longest
MAX_KV_ROWS = 4 * 8 * 65536                  # (position, KV head) rows of the largest sparse step


def _text(numbers):
    """A list of lengths as a case holds it."""
    return ",".join(str(n) for n in numbers)


def _parsed(case):
    """The case with its lengths as lists of numbers."""
    return {k: [int(n) for n in v.split(",") if n] if k in ("lens", "olds", "news", "owns") else v for k, v in case.items()}


def listed():
    return [
        # one new token of each of four sequences: the smallest append of a serving loop
        dict(name="rotary_decode_tokens", kind="rotary", codes="int8", dtype="bf16", heads=32, kv_heads=8, olds="32,37,44,46", news="1,1,1,1",
             rot=128, interleaved=False, table="fp32", bounds=True, layout="qkv"),
        # a batch of decode tokens, blocks begun to every extent, rotation table in the activations' type
        dict(name="rotary_decode_b64", kind="rotary", codes="e4m3", dtype="bf16", heads=64, kv_heads=8, olds=_text(16 + 7 * i % 45 for i in range(64)),
             news=_text([1] * 64), rot=128, interleaved=False, table="own", bounds=False, layout="own"),
        # a prompt into empty blocks, q, K and V as views into the projection's output, block bounds kept
        dict(name="rotary_prompt_8k", kind="rotary", codes="int8", dtype="bf16", heads=64, kv_heads=8, olds="0", news="8192", rot=128,
             interleaved=False, table="fp32", bounds=True, layout="qkv"),
        # chunks of several sequences that end and begin inside blocks; half of the channels rotated, in neighbouring pairs
        dict(name="rotary_chunks_ragged", kind="rotary", codes="e4m3", dtype="fp16", heads=32, kv_heads=4, olds="0,5,16,131,40,0,77",
             news="701,1,1500,333,17,15,2048", rot=64, interleaved=True, table="fp32", bounds=True, layout="own"),
        # a few samples of one question: latency
        dict(name="shared_b4_2k", kind="shared", codes="int8", dtype="bf16", heads=32, kv_heads=8, prefix=2048, owns="17,20,33,64", softcap=0.0),
        # one system prompt, conversations of many lengths, capped scores
        dict(name="shared_b32_8k_cap", kind="shared", codes="e4m3", dtype="fp16", heads=32, kv_heads=4, prefix=8192 - 16,
             owns=_text(1 + (990 * (i * i + 3 * i)) // (31 * 34) for i in range(32)), softcap=30.0),
        # a long document, many questions about it
        dict(name="shared_b64_32k", kind="shared", codes="int8", dtype="bf16", heads=64, kv_heads=8, prefix=32768, owns=_text(64 + 7 * i for i in range(64)),
             softcap=0.0),
        # the largest: 256 samples over a context of 64k
        dict(name="shared_b256_64k", kind="shared", codes="int8", dtype="bf16", heads=64, kv_heads=8, prefix=65536,
             owns=_text(1 + (i * 37) % 509 for i in range(256)), softcap=0.0),
        # one sequence: latency
        dict(name="sparse_b1_8k", kind="sparse", codes="int8", dtype="bf16", heads=32, kv_heads=8, lens="8000", top=64, first=1, last=2, softcap=0.0),
        # a long sequence on one GPU of eight
        dict(name="sparse_shard_b1_128k", kind="sparse", codes="e4m3", dtype="bf16", heads=8, kv_heads=1, lens="131072", top=256, first=1, last=8,
             softcap=0.0),
        # a batch of different lengths, some below the number of blocks that are kept, capped scores
        dict(name="sparse_b32_ragged_cap", kind="sparse", codes="e4m3", dtype="fp16", heads=32, kv_heads=4,
             lens=_text(1 + (16000 * (i * i + 3 * i)) // (31 * 34) for i in range(32)), top=96, first=2, last=4, softcap=30.0),
        # four long sequences
        dict(name="sparse_b4_64k", kind="sparse", codes="int8", dtype="bf16", heads=64, kv_heads=8, lens="65536,65536,65536,65531", top=128, first=1,
             last=2, softcap=0.0),
    ]


def _log_int(rng, lo, hi):
    if hi <= lo:
        return lo
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))))


def _cut(rng, total, n):
    """``n`` positive lengths of very different size that add up to about ``total``."""
    weights = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(n)]
    return [max(1, int(total * w / sum(weights))) for w in weights]


def draw(rng):
    kind = rng.choice(("rotary", "shared", "sparse"))
    common = dict(kind=kind, codes=rng.choice(tuple(CODES)), dtype=rng.choice(("bf16", "fp16")))
    heads, kv = rng.choice(GEOMETRIES)
    common.update(heads=heads, kv_heads=kv)
    softcap = rng.choice((0.0, 0.0, 15.0, 30.0, 50.0))
    if kind == "rotary":
        most = MAX_ROTARY_ROWS // (heads + 2 * kv)
        n = _log_int(rng, 1, 64)
        news = [1] * n if rng.random() < 0.4 else _cut(rng, _log_int(rng, n, min(16384, most - n)), n)
        olds = [rng.choice((0, _log_int(rng, 1, 400))) for _ in news]
        return dict(common, olds=_text(olds), news=_text(news), rot=rng.choice((128, 128, 96, 64, 32)), interleaved=rng.random() < 0.3,
                    table=rng.choice(("fp32", "fp32", "own")), bounds=rng.random() < 0.5, layout=rng.choice(("own", "qkv")))
    if kind == "shared":
        n = _log_int(rng, 1, 256)
        blocks = _log_int(rng, 1, min(65536, MAX_SHARED // (heads * n)) // BLOCK)
        longest = _log_int(rng, 1, min(4096, MAX_OWN // n))
        owns = [longest if rng.random() < 0.2 else _log_int(rng, 1, longest) for _ in range(n)]
        return dict(common, prefix=blocks * BLOCK, owns=_text(owns), softcap=softcap)
    n = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, min(131072, MAX_KV_ROWS // (kv * n)))
    lens = [ctx if rng.random() < 0.3 else _log_int(rng, 1, ctx) for _ in range(n)]
    top = _log_int(rng, 4, 512)
    first = rng.choice((0, 1, 1, 2))
    return dict(common, lens=_text(lens), top=top, first=first, last=_log_int(rng, 1, min(8, top - first)), softcap=softcap)


# ---- inputs -----------------------------------------------------------------------------


def _tokens(gen, tokens, heads, dtype, outliers):
    x = torch.randn(tokens, heads, HEAD_DIM, generator=gen, device="cuda")
    if outliers:
        x = x * torch.exp(0.75 * torch.randn(1, heads, HEAD_DIM, generator=gen, device="cuda"))
    return x.to(dtype)


def _tables(gen, lens, spare):
    """Shuffled pages: the block table of sequences of ``lens`` positions, what the permutation has left, the number of blocks."""
    need = [max(1, (l + BLOCK - 1) // BLOCK) for l in lens]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=gen, device="cuda")
    table = torch.zeros(len(lens), max(need), dtype=torch.int64, device="cuda")
    counts = torch.tensor(need, device="cuda")
    table[torch.arange(max(need), device="cuda")[None] < counts[:, None]] = perm[:sum(need)]
    return table, perm[sum(need):], blocks


def _filled(gen, kv, blocks, codes, outliers, topic=0.0):
    """A cache full of quantised rows: codes ``(kv, slots, 128)``, scales ``(kv, blocks)``."""
    data = torch.empty(kv, blocks * BLOCK, HEAD_DIM, dtype=CODES[codes], device="cuda")
    scales = torch.empty(kv, blocks, device="cuda")
    for h in range(kv):
        x = torch.randn(blocks, BLOCK, HEAD_DIM, generator=gen, device="cuda")
        if topic:
            x = x + topic * torch.randn(blocks, 1, HEAD_DIM, generator=gen, device="cuda")
        if outliers:
            x = x * torch.exp(0.75 * torch.randn(1, 1, HEAD_DIM, generator=gen, device="cuda"))
        scales[h] = _block_scale(x.abs().amax(dim=(1, 2)), codes)
        data[h] = _encode(x * (1.0 / scales[h])[:, None, None], codes).view(-1, HEAD_DIM)
    return data, scales


def _bounds_of(data, blocks, codes):
    """Lowest and highest code of every block and channel, ``(kv, blocks, 2, 128)`` int8."""
    rows = data.view(data.shape[0], blocks, BLOCK, HEAD_DIM)
    return torch.stack([torch.stack(_bounds(r.float(), codes), dim=1) for r in rows])


def _rotation(positions, rot, dtype):
    """cos and sin of every position's angles side by side, ``(positions, rot)``; far angles need 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq[None]
    return torch.cat([angle.cos(), angle.sin()], dim=1).to(dtype)


def prepare(case, seed):
    case = _parsed(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dtype, heads, kv = case["kind"], DTYPE[case["dtype"]], case["heads"], case["kv_heads"]
    st = dict(case=case)
    if kind == "rotary":
        lens = [o + n for o, n in zip(case["olds"], case["news"])]
        st["block_table"], _, blocks = _tables(gen, lens, 2)
        T = sum(case["news"])
        q, k, v = _tokens(gen, T, heads, dtype, False), _tokens(gen, T, kv, dtype, True), _tokens(gen, T, kv, dtype, False)
        if case["layout"] == "qkv":
            both = torch.cat([q, k, v], dim=1)
            q, k, v = both[:, :heads], both[:, heads:heads + kv], both[:, heads + kv:]
        st["q"], st["key"], st["value"] = q, k, v
        st["k_data"], st["k_scales"] = _filled(gen, kv, blocks, case["codes"], True)
        st["v_data"], st["v_scales"] = _filled(gen, kv, blocks, case["codes"], False)
        st["bounds"] = _bounds_of(st["k_data"], blocks, case["codes"]) if case["bounds"] else None
        starts = [0]
        for n in case["news"]:
            starts.append(starts[-1] + n)
        st["query_start_loc"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["positions"] = torch.tensor([p for o, l in zip(case["olds"], lens) for p in range(o, l)], dtype=torch.int64, device="cuda")
        st["cos_sin"] = _rotation(max(lens), case["rot"], torch.float32 if case["table"] == "fp32" else dtype)
        return st
    if kind == "shared":
        n, shared = len(case["owns"]), case["prefix"] // BLOCK
        st["block_table"], left, blocks = _tables(gen, case["owns"], shared + 2)
        st["shared_table"] = left[:shared].contiguous()
        st["seq_lens"] = torch.tensor([case["prefix"] + o for o in case["owns"]], dtype=torch.int32, device="cuda")
    else:
        n = len(case["lens"])
        st["block_table"], _, blocks = _tables(gen, case["lens"], 2)
        st["seq_lens"] = torch.tensor(case["lens"], dtype=torch.int32, device="cuda")
    st["k_data"], st["k_scales"] = _filled(gen, kv, blocks, case["codes"], True, 0.7 if kind == "sparse" else 0.0)
    st["v_data"], st["v_scales"] = _filled(gen, kv, blocks, case["codes"], False)
    st["q"] = _tokens(gen, n, heads, dtype, False)
    if kind == "sparse":
        st["bounds"] = _bounds_of(st["k_data"], blocks, case["codes"])
    return st


# ---- one pass ---------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if kind == "rotary":
        q = (_own_rotary if own else _plain_rotary)(state)
        out = [q, _values(state["k_data"], state["k_scales"]), state["k_scales"], _values(state["v_data"], state["v_scales"]), state["v_scales"]]
        if state["bounds"] is not None:
            out.append(state["bounds"] * _unit(state["k_scales"], state["case"]["codes"])[:, :, None, None])
        return out
    if kind == "shared":
        return (_own_shared if own else _plain_shared)(state)
    return (_own_sparse if own else _plain_sparse)(state)


def _values(data, scales):
    """What the codes of a cache stand for."""
    kv, blocks = scales.shape
    rows, scales = data.view(kv, blocks, BLOCK, HEAD_DIM), scales[:, :, None, None]
    return rows * scales if data.dtype == torch.int8 else rows.float().mul_(scales)


def _unit(scales, codes):
    """What a bound of 1 stands for: the scale of the codes, for e4m3 448 / 127 of it."""
    return scales if codes == "int8" else scales * torch.full_like(scales, 448.0 / 127.0)


def _own_rotary(st):
    from jetfire_b200 import ops
    return ops.block8_append_rotary(st["q"], st["key"], st["value"], st["positions"], st["cos_sin"], st["query_start_loc"], st["seq_lens"],
                                    st["block_table"], st["k_data"], st["k_scales"], st["v_data"], st["v_scales"],
                                    interleaved=st["case"]["interleaved"], bounds=st["bounds"])


def _own_shared(st):
    from jetfire_b200 import ops
    c = st["case"]
    return ops.block8_shared_prefix_attn(st["q"], st["k_data"], st["k_scales"], st["v_data"], st["v_scales"], st["shared_table"], st["block_table"],
                                         st["seq_lens"], c["prefix"] + max(c["owns"]), c["heads"], c["kv_heads"], BLOCK, SCALE, softcap=c["softcap"])


def _own_sparse(st):
    from jetfire_b200 import ops
    c = st["case"]
    return ops.block8_sparse_decode_attn(st["q"], st["k_data"], st["k_scales"], st["v_data"], st["v_scales"], st["bounds"], st["block_table"],
                                         st["seq_lens"], max(c["lens"]), c["heads"], c["kv_heads"], BLOCK, SCALE, top_blocks=c["top"],
                                         first_blocks=c["first"], last_blocks=c["last"], softcap=c["softcap"])


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


def _bounds(rows, codes):
    """Lowest and highest of codes ``(blocks, 16, 128)`` (as numbers) per block and channel: int8 codes as they are, e4m3 ones in
    units of 448 / 127, rounded outwards."""
    lo, hi = rows.amin(dim=1), rows.amax(dim=1)
    if codes == "e4m3":
        top = torch.full_like(lo, 448.0)
        lo, hi = torch.floor(lo * 127.0 / top), torch.ceil(hi * 127.0 / top)
    return lo.to(torch.int8), hi.to(torch.int8)


def _rotated(x, cos_sin, interleaved):
    """Rows ``(T, heads, 128)`` in fp32, rotated by ``cos_sin (T, rot)``; the channels behind ``rot`` stay."""
    x, rot = x.float(), cos_sin.shape[1]
    c, s = cos_sin[:, None, :rot // 2].float(), cos_sin[:, None, rot // 2:].float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y, z = a * c - b * s, b * c + a * s
    turned = torch.stack([y, z], dim=-1).flatten(-2) if interleaved else torch.cat([y, z], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _plain_rotary(st):
    case = st["case"]
    codes = case["codes"]
    turn = st["cos_sin"][st["positions"]]
    start, lens = st["query_start_loc"].long(), st["seq_lens"].long()
    token = torch.arange(st["key"].shape[0], device="cuda")
    seq = (token[:, None] >= start[None, 1:]).sum(1)
    pos = lens[seq] - (start[seq + 1] - token)
    block, row = st["block_table"][seq, pos // BLOCK], pos % BLOCK
    sides = ((_rotated(st["key"], turn, case["interleaved"]), st["k_data"], st["k_scales"]), (st["value"].float(), st["v_data"], st["v_scales"]))
    touched = last = None
    for x, data, scales in sides:
        kv, blocks = scales.shape
        size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(2)                       # (T, kv)
        amax = torch.zeros(blocks, kv, device="cuda").index_reduce_(0, block, size, "amax").t()
        first = torch.full((blocks,), BLOCK, device="cuda").index_reduce_(0, block, row, "amin")
        last = torch.full((blocks,), -1, device="cuda").index_reduce_(0, block, row, "amax")
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
    if st["bounds"] is not None:
        rows = st["k_data"].view(kv, blocks, BLOCK, HEAD_DIM)[:, touched].float()
        there = (torch.arange(BLOCK, device="cuda")[None] <= last[touched][:, None])[:, :, None]          # (touched blocks, 16, 1)
        for h in range(kv):
            lo, _ = _bounds(torch.where(there, rows[h], torch.full_like(rows[h], CODE_MAX[codes])), codes)
            _, hi = _bounds(torch.where(there, rows[h], torch.full_like(rows[h], -CODE_MAX[codes])), codes)
            st["bounds"][h, touched] = torch.stack([lo, hi], dim=1)
    return _rotated(st["q"], turn, case["interleaved"]).to(st["q"].dtype)


def _block_values(data, scales, g, ids):
    """Values of the blocks ``ids`` (any shape) of KV head g in fp32: ``(*ids.shape, 16, 128)``."""
    rows = data[g].view(-1, BLOCK, HEAD_DIM).view(torch.int8)[ids].view(data.dtype).float()
    return rows * scales[g, ids][..., None, None]


def _capped(s, cap):
    return cap * torch.tanh(s / cap) if cap else s


def _plain_shared(st):
    case = st["case"]
    heads, kv, prefix = case["heads"], case["kv_heads"], case["prefix"]
    group, n = heads // kv, len(case["owns"])
    width = st["block_table"].shape[1] * BLOCK
    out = torch.empty(n, heads, HEAD_DIM, device="cuda")
    lse = torch.empty(n, heads, device="cuda")
    behind = torch.arange(width, device="cuda")[None] >= (st["seq_lens"].long() - prefix)[:, None]        # (n, width)
    for g in range(kv):
        part = slice(g * group, (g + 1) * group)
        k, v = (_block_values(d, s, g, st["shared_table"]).view(-1, HEAD_DIM)
                for d, s in ((st["k_data"], st["k_scales"]), (st["v_data"], st["v_scales"])))
        for lo in range(0, n, 64):
            some = slice(lo, lo + 64)
            ids, q = st["block_table"][some], st["q"][some, part].float()
            ko, vo = (_block_values(d, s, g, ids).view(ids.shape[0], width, HEAD_DIM)
                      for d, s in ((st["k_data"], st["k_scales"]), (st["v_data"], st["v_scales"])))
            both = torch.cat([(q.reshape(-1, HEAD_DIM) @ k.t()).view(-1, group, prefix), q @ ko.transpose(1, 2)], dim=2)
            s = _capped(SCALE * both, case["softcap"])
            s[:, :, prefix:].masked_fill_(behind[some, None], float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            z = p.sum(-1, keepdim=True)
            o = (p[:, :, :prefix].reshape(-1, prefix) @ v).view(-1, group, HEAD_DIM) + p[:, :, prefix:] @ vo
            out[some, part] = o / z
            lse[some, part] = (top + torch.log(z)).squeeze(-1)
    return out.to(st["q"].dtype), lse


def _plain_sparse(st):
    case = st["case"]
    heads, kv, top = case["heads"], case["kv_heads"], case["top"]
    group = heads // kv
    out = torch.empty(len(case["lens"]), heads, HEAD_DIM, device="cuda")
    lse = torch.empty(len(case["lens"]), heads, device="cuda")
    chosen = torch.full((len(case["lens"]), kv, top), -1, dtype=torch.int32, device="cuda")
    for b, length in enumerate(case["lens"]):
        n = (length + BLOCK - 1) // BLOCK
        ids = st["block_table"][b, :n]
        q = st["q"][b].float().view(kv, group, HEAD_DIM)
        if n > top:
            size = q.abs().amax(-1, keepdim=True).clamp(min=SMALLEST)
            step = size / torch.full_like(size, 127.0)
            q8 = torch.round(q / step)
            near = st["bounds"][:, ids].float()                                                           # (kv, n, 2, 128)
            dot = q8.clamp(min=0) @ near[:, :, 1].transpose(1, 2) + q8.clamp(max=0) @ near[:, :, 0].transpose(1, 2)
            score = ((dot * step) * _unit(st["k_scales"][:, ids], case["codes"])[:, None]).amax(1)        # (kv, n)
            score[:, :case["first"]] = float("inf")
            score[:, n - case["last"]:] = float("inf")
            pick = score.sort(dim=1, descending=True, stable=True).indices[:, :top].sort(dim=1).values
        else:
            pick = torch.arange(n, device="cuda").expand(kv, n)
        m = pick.shape[1]
        chosen[b, :, :m] = pick.to(torch.int32)
        behind = (pick[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).view(kv, 1, -1) >= length
        k, v = (torch.stack([_block_values(d, s, g, ids[pick[g]]).view(-1, HEAD_DIM) for g in range(kv)])
                for d, s in ((st["k_data"], st["k_scales"]), (st["v_data"], st["v_scales"])))
        s = _capped(SCALE * (q @ k.transpose(1, 2)), case["softcap"]).masked_fill(behind, float("-inf"))
        most = s.amax(-1, keepdim=True)
        p = torch.exp(s - most)
        z = p.sum(-1, keepdim=True)
        out[b] = ((p @ v) / z).view(heads, HEAD_DIM)
        lse[b] = (most + torch.log(z)).view(heads)
    return out.to(st["q"].dtype), lse, chosen


# ---- what a pass cannot do without --------------------------------------------------------


def work(case):
    case = _parsed(case)
    heads, kv = case["heads"], case["kv_heads"]
    if case["kind"] == "rotary":
        T = sum(case["news"])
        blocks = sum((o + n + BLOCK - 1) // BLOCK - o // BLOCK for o, n in zip(case["olds"], case["news"]))
        size = T * (heads * HEAD_DIM * 4 + 2 * kv * HEAD_DIM * 3 + case["rot"] * (4 if case["table"] == "fp32" else 2) + 8)
        size += blocks * kv * (8 + (2 * HEAD_DIM if case["bounds"] else 0))
        return {"bytes": size, "flops": T * (heads + kv) * case["rot"] * 3 + T * 2 * kv * HEAD_DIM}
    if case["kind"] == "shared":
        n, total = len(case["owns"]), case["prefix"] + sum(case["owns"])
        pairs = heads * (n * case["prefix"] + sum(case["owns"]))
        return {"bytes": total * kv * 2 * HEAD_DIM + total // BLOCK * kv * 8 + n * heads * (HEAD_DIM * 4 + 4), "flops": 4 * HEAD_DIM * pairs}
    size = flops = 0
    for length in case["lens"]:
        n = (length + BLOCK - 1) // BLOCK
        kept = length if n <= case["top"] else case["top"] * BLOCK - (-length) % BLOCK
        size += kept * kv * 2 * HEAD_DIM + min(n, case["top"]) * kv * 8 + heads * (HEAD_DIM * 4 + 4) + 4 * kv * case["top"]
        flops += 4 * HEAD_DIM * heads * kept
        if n > case["top"]:
            size += n * kv * (2 * HEAD_DIM + 4)
            flops += 2 * HEAD_DIM * heads * n
    return {"bytes": size, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    case = st["case"]
    return {"rotary": _exact_rotary, "shared": _exact_shared, "sparse": _exact_sparse}[case["kind"]](st, case)


def _fp32(x):
    """Rounded to a 32-bit number: where the definition says that one is held."""
    return x.float().double()


def _turn64(x, st, case):
    """Channel 2i (or i) of a pair gets ``a cos - b sin``, the other ``b cos + a sin``; products and sums are 32-bit numbers."""
    y, half = x.double(), case["rot"] // 2
    table = st["cos_sin"].double()[st["positions"]][:, None]
    for i in range(half):
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        a, b, c, s = x[..., first].double(), x[..., second].double(), table[..., i], table[..., half + i]
        y[..., first] = _fp32(_fp32(a * c) - _fp32(b * s))
        y[..., second] = _fp32(_fp32(b * c) + _fp32(a * s))
    return y


def _exact_rotary(st, case):
    top = CODE_MAX[case["codes"]]
    q = _turn64(st["q"], st, case)
    outs = [q]
    kv, blocks = st["k_scales"].shape
    lens, news = case["olds"], case["news"]
    for x, data, scales in ((_turn64(st["key"], st, case), st["k_data"], st["k_scales"]), (st["value"].double(), st["v_data"], st["v_scales"])):
        codes = data.view(kv, blocks, BLOCK, HEAD_DIM).double()
        scale = scales.double()
        t = 0
        for s, (old, new) in enumerate(zip(lens, news)):
            ids = st["block_table"][s, old // BLOCK:(old + new + BLOCK - 1) // BLOCK]
            m, r = ids.numel(), old % BLOCK
            rows = torch.zeros(kv, m * BLOCK, HEAD_DIM, dtype=torch.float64, device="cuda")
            rows[:, r:r + new] = x[t:t + new].transpose(0, 1)
            rows = rows.view(kv, m, BLOCK, HEAD_DIM)
            amax = rows.abs().amax(dim=(2, 3)).clamp(min=SMALLEST)
            want = _fp32(amax / 127.0) if case["codes"] == "int8" else torch.exp2(torch.ceil(torch.log2(amax / 448.0)))
            was = torch.zeros_like(want)
            if r:
                was[:, 0] = scale[:, ids[0]]
            now = torch.maximum(was, want)
            fresh = _fp32(rows * _fp32(1.0 / now)[:, :, None, None]).clamp(-top, top)
            fresh = fresh.round() if case["codes"] == "int8" else fresh.float().to(torch.float8_e4m3fn).double()
            there = torch.zeros(m * BLOCK, dtype=torch.bool, device="cuda")
            there[r:r + new] = True
            there = there.view(1, m, BLOCK, 1)
            before = codes[:, ids]
            if r:
                moved = _fp32(before[:, 0, :r] * _fp32(was[:, 0] / now[:, 0])[:, None, None])
                before[:, 0, :r] = moved.round() if case["codes"] == "int8" else moved.float().to(torch.float8_e4m3fn).double()
            codes[:, ids] = torch.where(there, fresh, before)
            scale[:, ids] = now
            t += new
        outs += [codes * scale[:, :, None, None], scale]
        if data is st["k_data"] and st["bounds"] is not None:
            bounds = st["bounds"].double()
            for s, (old, new) in enumerate(zip(lens, news)):
                for at in range(old // BLOCK, (old + new + BLOCK - 1) // BLOCK):
                    i = st["block_table"][s, at]
                    rows = codes[:, i, :min(BLOCK, old + new - at * BLOCK)]
                    lo, hi = rows.min(1).values, rows.max(1).values
                    if case["codes"] == "e4m3":
                        lo, hi = torch.floor(lo * 127 / 448), torch.ceil(hi * 127 / 448)
                    bounds[:, i, 0], bounds[:, i, 1] = lo, hi
            unit = scale if case["codes"] == "int8" else scale * 448 / 127
            kept = bounds * unit[:, :, None, None]
    return outs + ([kept] if st["bounds"] is not None else [])


def _attend64(s, v, cap):
    """Scores ``(rows, keys)`` (-inf: not seen) and values -> outputs and log sums."""
    if cap:
        s = torch.where(torch.isinf(s), s, cap * torch.tanh(s / cap))
    lse = torch.logsumexp(s, dim=-1)
    return torch.exp(s - lse[:, None]) @ v, lse


def _values64(data, scales, g, ids):
    rows = data[g].view(-1, BLOCK, HEAD_DIM).view(torch.int8)[ids].view(data.dtype).double()
    return (rows * scales[g, ids].double()[:, None, None]).reshape(-1, HEAD_DIM)


def _exact_shared(st, case):
    heads, kv, prefix = case["heads"], case["kv_heads"], case["prefix"]
    group, n = heads // kv, len(case["owns"])
    out = torch.empty(n, heads, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.empty(n, heads, dtype=torch.float64, device="cuda")
    for g in range(kv):
        part = slice(g * group, (g + 1) * group)
        k, v = _values64(st["k_data"], st["k_scales"], g, st["shared_table"]), _values64(st["v_data"], st["v_scales"], g, st["shared_table"])
        q = st["q"][:, part].double()
        o1, l1 = [], []
        for lo in range(0, n * group, 512):     # the shared part of all rows, then what is each sequence's own
            o, l = _attend64(SCALE * (q.reshape(-1, HEAD_DIM)[lo:lo + 512] @ k.t()), v, case["softcap"])
            o1.append(o)
            l1.append(l)
        o1, l1 = torch.cat(o1).view(n, group, HEAD_DIM), torch.cat(l1).view(n, group)
        for b, own_len in enumerate(case["owns"]):
            ids = st["block_table"][b, :(own_len + BLOCK - 1) // BLOCK]
            ko, vo = (_values64(d, s, g, ids)[:own_len] for d, s in ((st["k_data"], st["k_scales"]), (st["v_data"], st["v_scales"])))
            o2, l2 = _attend64(SCALE * (q[b] @ ko.t()), vo, case["softcap"])
            both = torch.logaddexp(l1[b], l2)
            out[b, part] = o1[b] * torch.exp(l1[b] - both)[:, None] + o2 * torch.exp(l2 - both)[:, None]
            lse[b, part] = both
    return out, lse


def _exact_sparse(st, case):
    heads, kv, top = case["heads"], case["kv_heads"], case["top"]
    group = heads // kv
    out = torch.empty(len(case["lens"]), heads, HEAD_DIM, dtype=torch.float64, device="cuda")
    lse = torch.empty(len(case["lens"]), heads, dtype=torch.float64, device="cuda")
    chosen = torch.full((len(case["lens"]), kv, top), -1, dtype=torch.int32, device="cuda")

    factor = 1.0 if case["codes"] == "int8" else float(torch.tensor(448.0 / 127.0, dtype=torch.float32))
    for b, length in enumerate(case["lens"]):
        n = (length + BLOCK - 1) // BLOCK
        ids = st["block_table"][b, :n]
        for g in range(kv):
            q = st["q"][b, g * group:(g + 1) * group].double()
            keep = torch.ones(n, dtype=torch.bool, device="cuda")
            if n > top:
                step = _fp32(q.abs().amax(1).clamp(min=SMALLEST) / 127.0)
                q8 = torch.round(_fp32(q / step[:, None]))
                near = st["bounds"][g, ids].double()
                unit = _fp32(st["k_scales"][g, ids].double() * factor)
                score = torch.full((n,), float("-inf"), dtype=torch.float64, device="cuda")
                for h in range(group):
                    best = torch.maximum(q8[h] * near[:, 0], q8[h] * near[:, 1]).sum(1)
                    score = torch.maximum(score, _fp32(_fp32(best * step[h]) * unit))
                at = torch.arange(n, device="cuda")
                score[(at < case["first"]) | (at >= n - case["last"])] = float("inf")
                order = score.argsort(descending=True, stable=True)
                keep = torch.zeros(n, dtype=torch.bool, device="cuda")
                keep[order[:top]] = True
            pick = keep.nonzero().flatten()
            chosen[b, g, :pick.numel()] = pick.to(torch.int32)
            k, v = _values64(st["k_data"], st["k_scales"], g, ids[pick]), _values64(st["v_data"], st["v_scales"], g, ids[pick])
            seen = (pick[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten() < length
            o, l = _attend64(SCALE * (q @ k[seen].t()), v[seen], case["softcap"])
            out[b, g * group:(g + 1) * group], lse[b, g * group:(g + 1) * group] = o, l
    return out, lse, chosen
