"""Decode attention where the V scales of a sequence are very small or very far apart: the sum of the weights, and with it lse, does
not depend on what the values are.

Tolerances of test_gpu_block8.py.  Scales go from 2^-107 (an int8 block of zeros) to 2^119 (bf16's largest numbers)."""
import pytest
import torch

import block8_ref as R
from test_gpu_block8 import CODES, Decode

pytestmark = pytest.mark.gpu


def _floor(codes):
    return R.scale_for(torch.zeros(()), CODES[codes]).item()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens, heads", [([1], (8, 1)), ([4000], (8, 8)), ([8192], (8, 1)), ([8192, 0, 5000], (16, 1)), ([70000], (4, 2))])
@pytest.mark.parametrize("code", [0, 96])
def test_blocks_of_the_smallest_scale(codes, lens, heads, code):
    """Equal scores over values that are all 0, or all 96 * 2^-107 (96 * 2^-108): lse is the logarithm of the length."""
    c = Decode(lens, *heads, CODES[codes], torch.bfloat16, 81)
    c.q.zero_()
    c.v.fill_(code)
    c.vs.fill_(_floor(codes))
    out, lse = c.run()
    assert torch.isfinite(lse).sum() == sum(n > 0 for n in lens) * heads[0]
    c.check(out, lse)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("high", [0, 40, 100, 118])
@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("lens, heads", [([30], (8, 1)), ([1500], (8, 1)), ([5000], (8, 8)), ([20000, 333], (8, 1))])
def test_blocks_of_zeros_among_others(codes, high, first, lens, heads):
    """Every other block holds zeros, the rest numbers up to 2^high and above: the zeros' positions count like the others."""
    c = Decode(lens, *heads, CODES[codes], torch.bfloat16, 82)
    c.q = (c.q.float() * 0.25).to(c.q.dtype)
    c.vs *= 2.0 ** high
    for row in c.table:
        ids = row[first::2]
        ids = ids[ids >= 0]
        c.v[:, ids] = 0
        c.vs[:, ids] = _floor(codes)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
def test_scales_of_every_size_in_one_sequence(codes):
    c = Decode([6000], 8, 1, CODES[codes], torch.bfloat16, 83)
    c.q = (c.q.float() * 0.25).to(c.q.dtype)
    g = torch.Generator().manual_seed(84)
    c.vs = torch.exp2(torch.randint(-107, 119, c.vs.shape, generator=g).double())
    c.check(*c.run())
