"""A wait that ran out inside the packed prompts' kernel is not silent: the error it notes is raised once, by the call that asks
for it, by the op's next call, or by the next step of a layer with an 8-bit cache.

No wait is made to run out: the note is written as the kernel writes it, into the record it writes to."""
import ctypes as C
import struct
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from jetfire_b200 import _lib as L
from jetfire_b200 import ops


@pytest.mark.parametrize("device", [-1, 64])
def test_devices_that_are_none(device):
    assert L.lib.jf_varlen_status(device) == L.JF_ERR_ARG and L.lib.jf_varlen_record(device, C.byref(C.c_void_p())) == L.JF_ERR_ARG
    assert L.lib.jf_varlen_record(0, None) == L.JF_ERR_ARG
    with pytest.raises(L.JetFireError):
        ops.varlen_prefill_status(torch.device("cuda", 64))


def _note():
    at = C.c_void_p()
    assert L.lib.jf_varlen_record(torch.cuda.current_device(), C.byref(at)) == L.JF_OK
    C.memmove(at, struct.pack("<Qii", 0x4A46535441545553, L.JF_ERR_TIMEOUT, 0), 16)


def _call(**kw):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(70, h, 128, generator=g).bfloat16().cuda() for h in (4, 2, 2))
    return ops.varlen_prefill_attn(q, k, v, torch.tensor([0, 70], dtype=torch.int32, device="cuda"), 0.1, **kw)


@pytest.mark.gpu
def test_it_is_raised_once():
    want, _ = _call()
    ops.varlen_prefill_status()
    _note()
    with pytest.raises(L.JetFireError, match="varlen_prefill_attn") as e:
        ops.varlen_prefill_status(want.device)
    assert e.value.status == L.JF_ERR_TIMEOUT
    ops.varlen_prefill_status()
    _note()
    with pytest.raises(L.JetFireError, match="varlen_prefill_attn"):
        _call()
    assert torch.equal(_call()[0], want)
    _note()                                              # calls with a record of their own have nothing to do with it
    assert torch.equal(_call(status_record=torch.zeros(16, dtype=torch.uint8, device="cuda"))[0], want)
    with pytest.raises(L.JetFireError):
        ops.varlen_prefill_status()


@pytest.mark.gpu
def test_a_captured_call_leaves_it_to_the_graph_s_owner():
    want, _ = _call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.Generator().manual_seed(1)
    args = [torch.randn(70, h, 128, generator=g).bfloat16().cuda() for h in (4, 2, 2)] + [torch.tensor([0, 70], dtype=torch.int32, device="cuda"), 0.1]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    _note()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        out, _ = ops.varlen_prefill_attn(*args)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    with pytest.raises(L.JetFireError):
        ops.varlen_prefill_status()


@pytest.mark.gpu
def test_the_first_call_of_a_process_may_be_a_captured_one():
    code = """
import torch
from jetfire_b200 import ops
x = [torch.ones(70, h, 128, dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2)]
cu = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, _ = ops.varlen_prefill_attn(*x, cu, 0.1)
graph.replay()
torch.cuda.synchronize()
ops.varlen_prefill_status()
assert (out == 1).all()
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


@pytest.mark.gpu
def test_a_layer_s_next_step_raises_it():
    from test_block8_adapter import Conversation
    c = Conversation(2, "cuda", seed=9)
    assert c.step([30, 12]) is not None
    _note()
    before = list(c.lens)
    with pytest.raises(L.JetFireError):
        c.step([1, 1])
    c.lens = before
    ops.varlen_prefill_status()
