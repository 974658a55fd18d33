"""Attention over more selected blocks than a cluster goes through: pieces of them, and a join."""
import pytest
import torch

from test_gpu_block8_sparse import CODES, Sparse

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens, top, H_q, H_kv", [([12000], 500, 16, 8), ([2500, 0, 1601, 3, 1599, 2000] * 7, 100, 8, 4), ([6000, 900], 200, 40, 1)])
def test_pieces(codes, lens, top, H_q, H_kv):
    c = Sparse(lens, H_q, H_kv, CODES[codes], torch.bfloat16, 161, top=top, softcap=9.0 if H_kv == 1 else 0.0, table_dtype=torch.int32)
    got = c.run()
    c.check(*got)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(c.run(), got))
