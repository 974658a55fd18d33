"""Decode attention over a shared prefix where one product takes all rows: tables of 32 bits, and many query heads for one KV head."""
import pytest
import torch

from test_gpu_block8_shared import CODES, Shared
from test_gpu_block8_shared_rows import BLOCKS, N, OWNS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared_dtype, own_dtype", [(torch.int32, torch.int32), (torch.int32, torch.int64), (torch.int64, torch.int32)])
@pytest.mark.parametrize("codes", CODES)
def test_tables_of_32_bits(shared_dtype, own_dtype, codes):
    """Own tables as views into wider ones, blocks that are not there among both."""
    c = Shared(BLOCKS, OWNS, 16, 8, CODES[codes], torch.bfloat16, 131)
    c.table[:, 5], c.table[:, 11], c.table[3, BLOCKS] = -1, c.blocks, -9
    a = list(c.device())
    a[5] = a[5].to(shared_dtype)
    wide = torch.full((N, a[6].shape[1] + 5), 10 ** 9, dtype=own_dtype, device="cuda")
    wide[:, 2:-3] = a[6]
    a[6] = wide[:, 2:-3]
    c.check(*c.run(a))
    want = c.run()
    assert all(torch.equal(x, y) for x, y in zip(c.run(a), want))


@pytest.mark.parametrize("H_q, H_kv, shared", [(24, 8, 30), (32, 2, 120), (9, 1, 240), (17, 1, 240), (40, 1, 240)])
@pytest.mark.parametrize("codes", CODES)
def test_query_heads_of_a_kv_head(H_q, H_kv, shared, codes):
    c = Shared(shared, OWNS, H_q, H_kv, CODES[codes], torch.float16 if H_q == 17 else torch.bfloat16, 132, softcap=12.0 if H_q == 40 else 0.0,
               table_dtype=torch.int32)
    c.check(*c.run())


@pytest.mark.parametrize("H_q, H_kv", [(32, 2), (40, 1)])
def test_long_parts_of_their_own_with_many_heads(H_q, H_kv):
    c = Shared(300, [(2500, 0, 1, 700)[i % 4] for i in range(80)], H_q, H_kv, torch.int8, torch.bfloat16, 133, table_dtype=torch.int32)
    c.check(*c.run())


def test_sequences_that_end_within_the_shared_positions_with_many_heads():
    owns = [(-480, -479, -100, -1, 0, 5, -17, -352, 33)[i % 9] for i in range(N)]
    c = Shared(120, owns, 32, 2, torch.float8_e4m3fn, torch.bfloat16, 134, table_dtype=torch.int32)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("owns", [[9, 300], [0, -20000], [-36800, 5]])
def test_few_rows_over_a_long_prefix(codes, owns):
    """Two sequences of 40 heads: one row tile, more tiles of positions than thread blocks."""
    c = Shared(2300, owns, 40, 1, CODES[codes], torch.bfloat16, 135, table_dtype=torch.int32)
    c.check(*c.run())
