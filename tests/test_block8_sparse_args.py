"""What the attention over selected blocks refuses, without a GPU: C-ABI status codes and the op's checks."""
import ctypes as C

import pytest
import torch

from test_block8_args import L, _args  # noqa: F401  (L: the library, as a fixture)


def _sparse(L, top=4, first=1, last=2, bounds=4096, chosen=4096, **kw):
    a = L.Block8SparseArgs()
    a.attn = _args(L, **kw)
    a.bounds, a.chosen, a.top_blocks, a.first_blocks, a.last_blocks = bounds, chosen, top, first, last
    return a


def test_struct_layout(L):
    assert C.sizeof(L.Block8SparseArgs) == C.sizeof(L.Block8AttnArgs) + 2 * 8 + 4 * 4


def test_status(L):
    f = lambda **kw: L.lib.jf_block8_sparse_attn(C.byref(_sparse(L, **kw)), None)
    assert L.lib.jf_block8_sparse_attn(None, None) == L.JF_ERR_ARG
    for bad in (dict(top=0), dict(top=-1), dict(first=-1), dict(last=0), dict(first=3), dict(first=2 ** 31 - 1, last=2 ** 31 - 1), dict(bounds=None),
                dict(bounds=4104), dict(chosen=None), dict(chosen=4098), dict(window=5), dict(prefix_lens=4096), dict(alibi_slopes=4096),
                dict(attn_scale=0.0), dict(attn_scale=-1.0), dict(attn_scale=float("nan")), dict(codes=2), dict(q_dtype=7), dict(B=-1), dict(H_q=7),
                dict(max_S=0), dict(q=None), dict(block_table=None), dict(out=None)):
        assert f(**bad) == L.JF_ERR_ARG, bad
    assert f(workspace=None) == L.JF_ERR_WORKSPACE and f(workspace_bytes=64) == L.JF_ERR_WORKSPACE
    assert f(max_S=2 ** 22 + 1, max_blocks=2 ** 20) == L.JF_ERR_UNSUPPORTED
    assert f(B=0) == L.JF_OK


def test_workspace_bytes(L):
    w, dense = L.lib.jf_block8_sparse_workspace_bytes, L.lib.jf_block8_workspace_bytes
    assert w(1, 8, 2, 100, 0) == 0 and w(1, 8, 3, 100, 4) == 0 and w(1, 8, 2, 0, 4) == 0
    # the attention's over the chosen blocks, and four bytes for each block of a row
    up = lambda x: (x + 255) // 256 * 256
    assert w(4, 64, 8, 65536, 128) == up(dense(4, 64, 8, 2048)) + 4 * 8 * 4096 * 4
    assert w(4, 64, 8, 100, 2 ** 31 - 1) == up(dense(4, 64, 8, 100)) + 4 * 8 * 8 * 4


def test_the_op_refuses(L):
    from jetfire_b200 import ops
    z = torch.zeros
    data, scales, bounds = z(2, 32, 128, dtype=torch.int8), z(2, 2), z(2, 2, 2, 128, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA tensor of the current device"):
        ops.block8_sparse_decode_attn(z(1, 4, 128), data, scales, data, scales, bounds, z(1, 4, dtype=torch.int64), z(1, dtype=torch.int32), 64, 4, 2, 16, 0.1,
                                      top_blocks=4)


@pytest.mark.gpu
def test_the_op_refuses_on_the_device(L):
    from jetfire_b200 import ops
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")
    good = dict(q=z(1, 4, 128, dtype=torch.bfloat16), k_data=z(2, 32, 128, dtype=torch.int8), k_scales=z(2, 2), v_data=z(2, 32, 128, dtype=torch.int8),
                v_scales=z(2, 2), bounds=z(2, 2, 2, 128, dtype=torch.int8), block_table=z(1, 4, dtype=torch.int64), seq_lens=z(1, dtype=torch.int32), max_S=64,
                H_q=4, H_kv=2, block_size=16, attn_scale=0.1, top_blocks=4)
    ops.block8_sparse_decode_attn(**good)
    for bad, match in ((dict(top_blocks=2), "top_blocks"), (dict(top_blocks=0), "top_blocks"), (dict(last_blocks=0), "last_blocks"), (dict(first_blocks=-1), "first"),
                       (dict(attn_scale=-0.1), "attn_scale"), (dict(attn_scale=float("nan")), "attn_scale"), (dict(bounds=z(2, 2, 2, 128)), "bounds"),
                       (dict(bounds=z(2, 3, 2, 128, dtype=torch.int8)), "bounds"), (dict(bounds=z(2, 2, 2, 64, dtype=torch.int8)), "bounds"),
                       (dict(softcap=-1.0), "softcap"), (dict(max_S=0), "max_S"), (dict(H_kv=4), "H_kv"), (dict(q=z(1, 5, 128, dtype=torch.bfloat16)), "q must"),
                       (dict(out=z(1, 4, 128)), "out must"), (dict(bounds=torch.zeros(2, 2, 2, 128, dtype=torch.int8)), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            ops.block8_sparse_decode_attn(**{**good, **bad})
    with pytest.raises(ops.JetFireError):
        ops.block8_sparse_decode_attn(**{**good, "workspace": z(16)})
