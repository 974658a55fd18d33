"""Slopes that an implementation holds on the host: a captured decode step does not go there for them."""
import pytest
import torch

from jetfire_b200.adapter import block8 as B8
from test_block8_adapter import D, H_KV, H_Q, Conversation, _impl, _layer, _meta

SLOPES = [0.5, 0.25, 0.125, 0.0625]


def test_slopes_are_brought_into_the_ops_form_once():
    impl = _impl()
    impl.alibi_slopes = torch.tensor(SLOPES, dtype=torch.float64)
    first = B8.score_options(impl, torch.device("cpu"))["alibi_slopes"]
    assert first.dtype == torch.float32 and first.tolist() == SLOPES
    assert B8.score_options(impl, torch.device("cpu"))["alibi_slopes"] is first


@pytest.mark.gpu
def test_a_captured_step_with_slopes_from_the_host():
    c = Conversation(2, "cuda", seed=14, alibi_slopes=torch.tensor(SLOPES))
    impl = _impl()
    impl.alibi_slopes = torch.tensor(SLOPES)
    c.step([30, 14], call=lambda **kw: B8.try_block8_attention(**{**kw, "impl": impl}))
    z = lambda h: torch.zeros(2, h, D, dtype=torch.bfloat16, device="cuda")
    q, k, v, out = z(H_Q), z(H_KV), z(H_KV), z(H_Q)
    md = _meta([30, 14], [1, 1], c.table, "cuda")
    args = dict(layer=_layer(), query=q, key=k, value=v, attn_metadata=md, output=out, store=c.store)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    fresh = _impl()                                       # no step before: an error that says so, and no capture of it
    fresh.alibi_slopes = torch.tensor(SLOPES)
    with torch.cuda.stream(stream):
        with pytest.raises(RuntimeError, match="before one is captured"), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            B8.score_options(fresh, q.device)
        with torch.cuda.graph(graph, stream=stream):
            B8.try_block8_attention(impl=impl, **args)

    def replay(query, key, value, attn_metadata, output, **_):
        with torch.cuda.stream(stream):
            for dst, src in ((q, query), (k, key), (v, value), (md.seq_lens, attn_metadata.seq_lens)):
                dst.copy_(src.reshape(dst.shape))
            graph.replay()
            output.copy_(out.reshape(output.shape))
            stream.synchronize()
        return output

    for _ in range(4):
        assert c.step([1, 1], call=replay) is not None
