"""A captured cascade step of a layer with an 8-bit cache is replayed with whatever the sequences share by then."""
import pytest
import torch

from jetfire_b200.adapter import block8 as B8
from test_block8_adapter import D, H_KV, H_Q, _layer, _meta
from test_block8_more_adapter import _fill, _sharing

pytestmark = pytest.mark.gpu
BLOCKS, OWN = 8, [30, 1, 17, 60]


def _step(c, md, q, k, v):
    out = torch.zeros_like(q)
    assert B8.try_block8_attention(impl=c.impl, layer=_layer(), query=q, key=k, value=v, attn_metadata=md, output=out, store=c.store) is out
    return out


@pytest.mark.parametrize("table_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("kept", [0, 3, 8])
def test_a_replay_with_a_shorter_prefix(kept, table_dtype):
    """Of the blocks shared at capture the first ``kept`` still are; the rest of each sequence's are its own."""
    c, other = (_fill(_sharing(4, "cuda", BLOCKS, seed=31), BLOCKS, OWN) for _ in range(2))
    q, k, v = (torch.zeros(4, h * D, dtype=torch.bfloat16, device="cuda") for h in (H_Q, H_KV, H_KV))
    md = _meta(c.lens, [1] * 4, c.table, "cuda")
    md.block_table = md.block_table.to(table_dtype)
    md.use_cascade, md.common_prefix_len = True, 16 * BLOCKS
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = _step(c, md, q, k, v)
    # (blocks that no sequence holds, filled alike in both caches)
    g = torch.Generator().manual_seed(32)
    free = sorted(set(range(c.store.num_blocks)) - set(c.table.flatten().tolist()))
    table, at = c.table.clone(), 0
    for b in range(1, 4):
        for j in range(kept, BLOCKS):
            table[b, j] = free[at]
            at += 1
    new = torch.tensor(free[:at], dtype=torch.long)
    if at:
        for name in ("k_data", "v_data"):
            rows = torch.randint(-127, 128, (H_KV, at, 16, D), generator=g, dtype=torch.int8).cuda()
            for s in (c.store, other.store):
                getattr(s, name).view(H_KV, -1, 16, D)[:, new.cuda()] = rows
        for name in ("k_scales", "v_scales"):
            scales = (torch.rand(H_KV, at, generator=g) * 0.02 + 0.01).cuda()
            for s in (c.store, other.store):
                getattr(s, name)[:, new.cuda()] = scales
    md.block_table.copy_(table)
    tokens = [torch.randn(4, h * D, generator=g).to(torch.bfloat16).cuda() for h in (H_Q, H_KV, H_KV)]
    for x, y in zip((q, k, v), tokens):
        x.copy_(y)
    md.seq_lens.copy_(torch.tensor([n + 1 for n in c.lens], dtype=torch.int32))
    graph.replay()
    eager = _meta(c.lens, [1] * 4, table, "cuda")
    eager.max_seq_len = 640
    want = _step(other, eager, *tokens)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
