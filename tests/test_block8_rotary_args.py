"""What the rotated append refuses, without a GPU: C-ABI status codes and the op's checks."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from jetfire_b200.build import build
    build()
    from jetfire_b200 import _lib
    return _lib


def _args(L, **kw):
    a = L.Block8RotaryArgs()
    a.dtype, a.codes, a.H_q, a.H_kv, a.n_seqs, a.max_blocks, a.rot = 0, 0, 8, 2, 1, 4, 128
    a.T, a.table_rows, a.num_blocks, a.bt_stride = 4, 100, 8, 4
    for n in ("query", "key", "value", "positions", "cos_sin", "query_start_loc", "seq_lens", "block_table", "k_data", "k_scales", "v_data", "v_scales",
              "bounds", "query_out"):
        setattr(a, n, 4096)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_struct_layout(L):
    assert C.sizeof(L.Block8RotaryArgs) == 12 * 4 + 10 * 8 + 14 * 8
    assert L.Block8RotaryArgs.T.offset == 48 and L.Block8RotaryArgs.query.offset == 128


def test_status(L):
    f = lambda **kw: L.lib.jf_block8_append_rotary(C.byref(_args(L, **kw)), None)
    assert L.lib.jf_block8_append_rotary(None, None) == L.JF_ERR_ARG
    for bad in (dict(dtype=2), dict(codes=2), dict(H_q=-1), dict(H_q=70000), dict(H_kv=0), dict(T=-1), dict(T=2 ** 31), dict(n_seqs=-1), dict(max_blocks=-1),
                dict(num_blocks=-1), dict(rot=0), dict(rot=8), dict(rot=120), dict(rot=144), dict(table_rows=-1), dict(cos_sin=None), dict(cos_sin=4104),
                dict(positions=None), dict(query=None), dict(query_out=None), dict(query_out=4104), dict(key=None), dict(value=None),
                dict(query_start_loc=None), dict(seq_lens=None), dict(block_table=None), dict(k_data=None), dict(k_data=4100), dict(k_scales=None),
                dict(v_data=None), dict(v_scales=4098), dict(bounds=4100)):
        assert f(**bad) == L.JF_ERR_ARG, bad
    assert f(T=0) == L.JF_OK and f(n_seqs=0) == L.JF_OK          # nothing to do, nothing launched


def test_the_op_refuses(L):
    from jetfire_b200 import ops
    z = torch.zeros
    q, key, start, lens = z(4, 4, 128, dtype=torch.bfloat16), z(4, 2, 128, dtype=torch.bfloat16), z(2, dtype=torch.int32), z(1, dtype=torch.int32)
    data, scales = z(2, 32, 128, dtype=torch.int8), z(2, 2)
    args = (z(4, dtype=torch.int64), z(10, 128), start, lens, z(1, 4, dtype=torch.int64), data, scales, data, scales)
    with pytest.raises(RuntimeError, match="CUDA tensor of the current device"):
        ops.block8_append_rotary(q, key, key, *args)
    with pytest.raises(RuntimeError, match="must be a tensor"):
        ops.block8_append_rotary(None, key, key, *args)
    with pytest.raises(RuntimeError, match="CUDA tensor of the current device"):
        ops.block8_append(key, key, start, lens, args[4], data, scales, data, scales, bounds=z(2, 2, 2, 128, dtype=torch.int8))


@pytest.mark.gpu
def test_the_op_refuses_on_the_device(L):
    from jetfire_b200 import ops
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")
    bf = torch.bfloat16
    good = dict(query=z(4, 4, 128, dtype=bf), key_tok=z(4, 2, 128, dtype=bf), value_tok=z(4, 2, 128, dtype=bf), positions=z(4, dtype=torch.int64),
                cos_sin=z(10, 128), query_start_loc=torch.tensor([0, 4], dtype=torch.int32, device="cuda"),
                seq_lens=torch.tensor([4], dtype=torch.int32, device="cuda"), block_table=z(1, 4, dtype=torch.int64),
                k_data=z(2, 32, 128, dtype=torch.int8), k_scales=z(2, 2), v_data=z(2, 32, 128, dtype=torch.int8), v_scales=z(2, 2))
    ops.block8_append_rotary(**good)
    for bad, match in ((dict(query=z(5, 4, 128, dtype=bf)), "query must be"), (dict(query=z(4, 4, 64, dtype=bf)), "query must be"),
                       (dict(query=z(4, 4, 128, dtype=torch.float16)), "dtype"), (dict(query=z(4, 128, 4, dtype=bf).transpose(1, 2)), "innermost"),
                       (dict(positions=z(3, dtype=torch.int64)), "positions"), (dict(positions=z(4)), "positions"),
                       (dict(positions=z(8, dtype=torch.int64)[::2]), "positions"), (dict(cos_sin=z(10, 120)), "cos_sin"), (dict(cos_sin=z(10, 144)), "cos_sin"),
                       (dict(cos_sin=z(10, 128, dtype=torch.float16)), "cos_sin"), (dict(cos_sin=z(128)), "cos_sin"),
                       (dict(bounds=z(2, 2, 2, 128)), "bounds"), (dict(bounds=z(2, 3, 2, 128, dtype=torch.int8)), "bounds"),
                       (dict(out=z(4, 4, 128)), "out must"), (dict(out=z(3, 4, 128, dtype=bf)), "out must"),
                       (dict(out=z(4 * 4 * 128 + 1, dtype=bf)[1:].view(4, 4, 128)), "out must"), (dict(positions=torch.zeros(4, dtype=torch.int64)), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            ops.block8_append_rotary(**{**good, **bad})
    # a table that is no view 16-byte copies can take is copied
    ops.block8_append_rotary(**{**good, "cos_sin": z(1281)[1:].view(10, 128)})
    ops.block8_append_rotary(**{**good, "cos_sin": z(128, 10).t()})
