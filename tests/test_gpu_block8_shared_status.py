"""A wait that ran out inside the attention over a shared prefix is raised by the op's next call, whatever the sizes of that call.

No wait is made to run out: the note is written as the kernel writes it, into the record it writes to."""
import pytest
import torch

from jetfire_b200 import _lib as L
from jetfire_b200 import ops
from test_gpu_block8_shared import Shared
from test_gpu_varlen_status import _note

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared, owns", [(4, [5, 9]), (30, [7] * 90), (0, [20])])
def test_the_next_call_raises_it_once(shared, owns):
    c = Shared(shared, owns, 8, 8, torch.int8, torch.bfloat16, 121)
    a = c.device()
    want = c.run(a)
    ops.varlen_prefill_status()
    _note()
    with pytest.raises(L.JetFireError, match="block8_shared_prefix_attn") as e:
        c.run(a)
    assert e.value.status == L.JF_ERR_TIMEOUT
    assert all(torch.equal(x, y) for x, y in zip(c.run(a), want))
    ops.varlen_prefill_status()


def test_a_captured_call_leaves_it():
    c = Shared(4, [5, 9], 8, 8, torch.int8, torch.bfloat16, 122)
    a = c.device()
    want = c.run(a)
    torch.cuda.synchronize()
    _note()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        got = c.run(a)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    with pytest.raises(L.JetFireError):
        ops.varlen_prefill_status()
