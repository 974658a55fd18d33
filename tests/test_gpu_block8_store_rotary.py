"""A store's rotated append, with and without bounds kept, then its decode attention: the same as the ops by themselves."""
import pytest
import torch

import block8_more_ref as M
from jetfire_b200 import ops
from jetfire_b200.adapter.block8 import JetFireBlock8Store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_prompt_and_decode_tokens(codes, top, interleaved):
    H_q, H_kv, n, width = 8, 2, 3, 12
    g = torch.Generator().manual_seed(151)
    table = torch.randperm(n * width, generator=g).view(n, width).int().cuda()
    cos_sin = M.table_of(64, 256).cuda()
    store, other = (JetFireBlock8Store(num_blocks=n * width, num_kv_heads=H_kv, codes=codes, top_blocks=top) for _ in range(2))
    lens = [0] * n
    for news in ([100, 17, 150], [1, 1, 1], [1, 1, 1]):
        T, start = sum(news), torch.tensor([0, news[0], news[0] + news[1], sum(news)], dtype=torch.int32).cuda()
        q, k, v = (torch.randn(T, h, 128, generator=g).bfloat16().cuda() for h in (H_q, H_kv, H_kv))
        pos = torch.cat([torch.arange(l, l + m) for l, m in zip(lens, news)]).cuda()
        lens = [l + m for l, m in zip(lens, news)]
        sl = torch.tensor(lens, dtype=torch.int32).cuda()
        want = ops.block8_append_rotary(q, k, v, pos, cos_sin, start, sl, table, other.k_data, other.k_scales, other.v_data, other.v_scales,
                                        interleaved=interleaved, bounds=other.bounds)
        got = store.append_rotary(q, k, v, pos, cos_sin, start, sl, table, interleaved=interleaved, out=q)
        assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
        assert torch.equal(store.k_data.view(torch.int8), other.k_data.view(torch.int8)) and torch.equal(store.v_scales, other.v_scales)
        assert (store.bounds is None) == (top == 0) and (top == 0 or torch.equal(store.bounds, other.bounds))
        if news[0] == 1:
            out, _ = store.decode(got, sl, table, 16 * width, 128 ** -0.5)
            plain, _ = ops.block8_decode_attn(got, other.k_data, other.k_scales, other.v_data, other.v_scales, table, sl, 16 * width, H_q, H_kv, 16, 128 ** -0.5)
            if top == 0:
                assert torch.equal(out, plain)
            else:      # (of 7, 2 and 10 blocks: the second sequence is attended to as a whole; both results are off by half a step of bf16 and of fp16 weights)
                assert not torch.equal(out, plain)
                assert ((out[1].float() - plain[1].float()).abs() <= 2 ** -7 * plain[1].float().abs() + 2 ** -10 * 5.0).all()
