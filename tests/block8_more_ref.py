"""Plain forms, in 64 bits, of the rotated append, block bounds, shared prefixes and selected blocks over the 8-bit cache."""
from __future__ import annotations

import torch

import block8_ref as R

BLOCK, D = R.BLOCK, R.D


def rotated(x, turn, interleaved):
    """``x (T, H, 128)`` by ``turn (T, rot)`` (NaN rows where a position is not in the table): every product and sum rounded to fp32."""
    y, half = x.double().clone(), turn.shape[1] // 2
    turn = turn.double()[:, None]
    for i in range(half):
        m, n = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b, c, s = x[..., m].double(), x[..., n].double(), turn[..., i], turn[..., half + i]
        y[..., m] = R.fl32(R.fl32(a * c) - R.fl32(b * s))
        y[..., n] = R.fl32(R.fl32(b * c) + R.fl32(a * s))
    return y


def turns(cos_sin, positions):
    got = torch.full((positions.numel(), cos_sin.shape[1]), float("nan"), dtype=torch.float64)
    there = (positions >= 0) & (positions < cos_sin.shape[0])
    got[there] = cos_sin.double()[positions[there].long()]
    return got


def bounds_of(code, rows, codes):
    """``code (H, rows of a block, 128)`` (float64) -> lowest and highest of the first ``rows``, ``(H, 2, 128)``."""
    lo, hi = code[:, :rows].amin(1), code[:, :rows].amax(1)
    if codes == torch.float8_e4m3fn:
        lo, hi = torch.floor(lo * 127 / 448), torch.ceil(hi * 127 / 448)
    return torch.stack([lo, hi], 1)


def table_of(rot, n, dtype=torch.float32):
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(n, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype)


class Cache:
    """A cache on the device and its plain form: codes and scales as float64 on the host."""

    def __init__(self, H, blocks, codes, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.H, self.blocks, self.codes = H, blocks, codes
        x = torch.randn(2, H, blocks, BLOCK, D, generator=g)
        self.code, self.scale = [], []
        for side in range(2):
            s = R.scale_for(x[side].abs().amax((2, 3)), codes)
            self.code.append(R.encode(x[side].double() / s[..., None, None], codes))
            self.scale.append(s)
        self.k_data, self.v_data = (c.to(codes).view(H, blocks * BLOCK, D).to(device) for c in self.code)
        self.k_scales, self.v_scales = (s.float().to(device) for s in self.scale)

    def tensors(self):
        return self.k_data, self.k_scales, self.v_data, self.v_scales

    def same(self):
        """The device's cache holds the plain form's bits."""
        for data, scales, code, scale in ((self.k_data, self.k_scales, self.code[0], self.scale[0]), (self.v_data, self.v_scales, self.code[1], self.scale[1])):
            assert torch.equal(scales.cpu().double(), scale)
            assert torch.equal(data.cpu().double().view(code.shape), code)

    def values(self, side):
        return self.code[side] * self.scale[side][..., None, None]


def choose(q, lo_hi, ks, ids, n, top, first, last, codes, blocks):
    """The blocks chosen for one sequence and KV head: ``q (heads, 128)`` float64, ``lo_hi (blocks, 2, 128)`` and ``ks (blocks,)`` of the
    head, ``ids`` of the sequence's n blocks.  Every step of a score is exact or rounded to fp32."""
    if n <= top:
        return list(range(n))
    ids = ids[:n]
    is_there = (ids >= 0) & (ids < blocks)
    at = ids.clamp(0, blocks - 1)
    unit = R.fl32(ks[at] * (1.0 if codes == torch.int8 else float(torch.tensor(448.0 / 127.0))))
    score = torch.full((n,), float("-inf"), dtype=torch.float64)
    near = lo_hi[at].double()
    for h in range(q.shape[0]):
        if not bool(torch.isfinite(q[h]).all()):
            continue
        step = R.fl32(q[h].abs().max().clamp(min=2.0 ** -100) / 127)
        q8 = torch.round(R.fl32(q[h] / step))
        best = (q8.clamp(max=0) * near[:, 0] + q8.clamp(min=0) * near[:, 1]).sum(1)
        mine = R.fl32(R.fl32(best * step) * unit)
        score = torch.where(torch.isnan(mine), score, torch.maximum(score, mine))
    score[~is_there | torch.isnan(unit)] = float("-inf")
    score[:first] = float("inf")
    score[n - last:] = float("inf")
    forced = torch.zeros(n)
    forced[:first] = forced[n - last:] = 1
    order = sorted(range(n), key=lambda j: (-forced[j].item(), -score[j].item(), j))
    return sorted(order[:top])
