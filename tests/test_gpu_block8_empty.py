"""Decode attention over a table without columns and over a cache without blocks: nothing is seen, so rows are 0 and lse -inf, as for a
length of 0 and for block ids that are none."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("blocks, width", [(4, 0), (0, 3), (0, 0)])
@pytest.mark.parametrize("max_S", [1, 48, 5000])
def test_nothing_to_see(codes, blocks, width, max_S):
    from jetfire_b200 import ops
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    k, v = (torch.zeros(2, blocks * 16, 128, device="cuda").to(codes) for _ in range(2))
    ks, vs = (torch.ones(2, blocks, device="cuda") for _ in range(2))
    table = torch.zeros(3, width, dtype=torch.int32, device="cuda")
    lens = torch.tensor([0, 17, 40], dtype=torch.int32, device="cuda")
    out, lse = ops.block8_decode_attn(q, k, ks, v, vs, table, lens, max_S, 8, 2, 16, 0.1, out=torch.full_like(q, 7.0))
    assert (out == 0).all() and (lse == float("-inf")).all()
