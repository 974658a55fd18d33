"""Lengths below zero, down to the lowest number there is, see nothing: of the shared positions and of their own."""
import pytest
import torch

from test_gpu_block8_shared import CODES, Shared

pytestmark = pytest.mark.gpu
LOWEST = -2 ** 31


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("shared, own, n", [(30, 40, 90), (30, 2500, 90), (30, 40, 3)])
def test_lengths_below_zero(shared, own, n, codes):
    """Own tables that would have blocks for them; with few and with many own blocks, and through the decode kernel alone."""
    c = Shared(shared, [own] * n, 8, 8, CODES[codes], torch.bfloat16, 141)
    lens = [(LOWEST, LOWEST + 16 * shared - 1, c.max_S, -1, LOWEST + 5)[i % 5] for i in range(n)]
    a = list(c.device())
    a[7] = torch.tensor(lens, dtype=torch.int32).cuda()
    c.lens = [max(l, 0) for l in lens]
    out, lse = c.run(a)
    c.check(out, lse)
    empty = torch.tensor([l <= 0 for l in lens])
    assert (out[empty.cuda()] == 0).all() and (lse[empty.cuda()] == float("-inf")).all()
