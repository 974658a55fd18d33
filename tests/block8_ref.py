"""Plain forms of the 8-bit block cache and of the attention over it, in 64 bits, for the tests."""
from __future__ import annotations

import torch

BLOCK, D = 16, 128
CODE_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def fl32(x):
    return x.to(torch.float32).double()


def scale_for(amax, codes):
    """fp32 scale (as float64) that a largest magnitude asks for."""
    amax = amax.double().clamp(min=2.0 ** -100)
    if codes == torch.int8:
        return fl32(amax / 127.0)
    s = torch.exp2(torch.floor(torch.log2(amax)) - 10)
    for _ in range(4):
        s = torch.where(amax > 448.0 * s, 2 * s, s)
    return s


def encode(x, codes):
    top = CODE_MAX[codes]
    x = torch.nan_to_num(x, nan=0.0, posinf=top, neginf=-top).clamp(-top, top)
    return x.round() if codes == torch.int8 else x.float().to(torch.float8_e4m3fn).double()


def append(key, start, lens, table, code, scale, codes):
    """``key (T, H, 128)`` into ``code (H, blocks, 16, 128)`` / ``scale (H, blocks)`` (float64 CPU tensors of code values
    and scales), in place."""
    H, blocks = scale.shape
    for s in range(len(lens)):
        a, b = int(start[s]), min(int(start[s + 1]), key.shape[0])
        first = int(lens[s]) - (int(start[s + 1]) - a)
        t = a
        while t < b:
            pos = first + t - a
            if pos < 0:
                t += 1
                continue
            r = pos % BLOCK if t == a else 0
            assert t == a or pos % BLOCK == 0 or first < 0
            n = min(BLOCK - pos % BLOCK, b - t)
            blk = pos // BLOCK
            if blk < table.shape[1] and 0 <= int(table[s, blk]) < blocks:
                i = int(table[s, blk])
                x = key[t:t + n].double().transpose(0, 1)                      # (H, n, 128)
                amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax((1, 2))
                old = scale[:, i].clone() if r else torch.zeros(H, dtype=torch.float64)
                old = torch.where(torch.isfinite(old) & (old > 0), old, torch.zeros_like(old))
                new = torch.maximum(old, scale_for(amax, codes))
                if r:
                    code[:, i, :r] = torch.where((new != old)[:, None, None], encode(fl32(code[:, i, :r] * fl32(old / new)[:, None, None]), codes),
                                                 code[:, i, :r])
                code[:, i, r:r + n] = encode(fl32(x * fl32(1.0 / new)[:, None, None]), codes)
                scale[:, i] = new
            t += n


def visible(i, j, causal=True, window=None, prefix=0):
    d = i[:, None] - j[None, :]
    sees = torch.ones_like(d, dtype=torch.bool)
    if causal:
        sees &= d >= 0
    if window is not None:
        sees &= d.abs() < window
    return sees | (j < prefix)[None, :]


def attend(q, k, v, i, j, scale, *, causal=True, window=None, prefix=0, softcap=0.0, slopes=None):
    """``q (H_q, n, 128)`` at positions i, ``k / v (H_kv, m, 128)`` at positions j, all float64 -> out (H_q, n, 128), lse."""
    group = q.shape[0] // k.shape[0]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    s = scale * (q @ k.transpose(1, 2))
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        s = s - slopes.double()[:, None, None] * (i[:, None] - j[None, :]).abs()
    sees = visible(i, j, causal, window, prefix)[None].expand_as(s)
    s = s.masked_fill(~sees, float("-inf"))
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), float("-inf"))
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    p = torch.where(sees, torch.exp(s - m), torch.zeros_like(s))
    z = p.sum(-1, keepdim=True)
    # (a hidden position contributes nothing, whatever its value is: products are formed for seen ones only)
    bad = ~torch.isfinite(v)
    out = p @ torch.where(bad, torch.zeros_like(v), v)
    if bool(bad.any()):
        for h, jj, d in bad.nonzero().tolist():
            out[h, sees[h, :, jj], d] += v[h, jj, d]
    out = torch.where(z > 0, out / torch.where(z > 0, z, torch.ones_like(z)), torch.where(z == 0, torch.zeros_like(out), out / z))
    return out, (m + torch.log(z)).squeeze(-1)
