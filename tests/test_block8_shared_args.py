"""What the attention over a shared prefix refuses, without a GPU: C-ABI status codes and the op's checks."""
import ctypes as C

import pytest
import torch

from test_block8_args import L, _args  # noqa: F401  (L: the library, as a fixture)


def _shared(L, blocks=4, table=4096, **kw):
    a = L.Block8SharedArgs()
    a.attn = _args(L, **kw)
    a.attn.workspace_bytes = kw.get("workspace_bytes", L.lib.jf_block8_shared_workspace_bytes(2, 8, 2, 100, 4))
    a.shared_table, a.shared_blocks = table, blocks
    return a


def test_struct_layout(L):
    assert C.sizeof(L.Block8SharedArgs) == C.sizeof(L.Block8AttnArgs) + 8 + 2 * 4


def test_status(L):
    f = lambda **kw: L.lib.jf_block8_shared_attn(C.byref(_shared(L, **kw)), None)
    assert L.lib.jf_block8_shared_attn(None, None) == L.JF_ERR_ARG
    for bad in (dict(blocks=-1), dict(table=None), dict(window=5), dict(prefix_lens=4096), dict(alibi_slopes=4096), dict(codes=2), dict(q_dtype=7), dict(B=-1),
                dict(H_q=7), dict(max_S=0), dict(q=None), dict(block_table=None), dict(out=None), dict(softcap=-1.0), dict(k_data=4104)):
        assert f(**bad) == L.JF_ERR_ARG, bad
    assert f(workspace=None) == L.JF_ERR_WORKSPACE and f(workspace_bytes=64) == L.JF_ERR_WORKSPACE
    assert f(max_blocks=2 ** 27 - 3) == L.JF_ERR_UNSUPPORTED and f(blocks=2 ** 27) == L.JF_ERR_UNSUPPORTED
    assert f(B=0) == L.JF_OK


def test_workspace_bytes(L):
    w = L.lib.jf_block8_shared_workspace_bytes
    assert w(0, 8, 2, 100, 4) == 0 and w(1, 8, 3, 100, 4) == 0 and w(1, 8, 2, 0, 4) == 0 and w(1, 8, 2, 100, -1) == 0
    assert 0 < w(1, 8, 2, 100, 4) <= w(256, 64, 8, 70000, 4096)


def test_the_op_refuses(L):
    from jetfire_b200 import ops
    z = torch.zeros
    data, scales = z(2, 32, 128, dtype=torch.int8), z(2, 2)
    with pytest.raises(RuntimeError, match="CUDA tensor of the current device"):
        ops.block8_shared_prefix_attn(z(1, 4, 128), data, scales, data, scales, z(4, dtype=torch.int64), z(1, 4, dtype=torch.int64), z(1, dtype=torch.int32), 64, 4,
                                      2, 16, 0.1)


@pytest.mark.gpu
def test_the_op_refuses_on_the_device(L):
    from jetfire_b200 import ops
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")
    good = dict(q=z(1, 4, 128, dtype=torch.bfloat16), k_data=z(2, 32, 128, dtype=torch.int8), k_scales=z(2, 2), v_data=z(2, 32, 128, dtype=torch.int8),
                v_scales=z(2, 2), shared_table=z(2, dtype=torch.int64), block_table=z(1, 4, dtype=torch.int64), seq_lens=z(1, dtype=torch.int32), max_S=64,
                H_q=4, H_kv=2, block_size=16, attn_scale=0.1)
    ops.block8_shared_prefix_attn(**good)
    for bad, match in ((dict(shared_table=z(1, 2, dtype=torch.int64)), "shared_table"), (dict(shared_table=z(2)), "shared_table"),
                       (dict(shared_table=z(4, dtype=torch.int64)[::2]), "shared_table"), (dict(shared_table=torch.zeros(2, dtype=torch.int64)), "CUDA"),
                       (dict(softcap=-1.0), "softcap"), (dict(max_S=0), "max_S"), (dict(H_kv=4), "H_kv"), (dict(q=z(1, 5, 128, dtype=torch.bfloat16)), "q must"),
                       (dict(out=z(1, 4, 128)), "out must"), (dict(block_table=z(2, 4, dtype=torch.int64)), "block_table")):
        with pytest.raises(RuntimeError, match=match):
            ops.block8_shared_prefix_attn(**{**good, **bad})
