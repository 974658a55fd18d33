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
