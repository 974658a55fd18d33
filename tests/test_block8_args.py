"""What the 8-bit cache's entry points refuse, without a GPU: C-ABI status codes and the ops' checks."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from jetfire_b200.build import build
    build()
    from jetfire_b200 import _lib
    return _lib


def test_struct_layout(L):
    assert C.sizeof(L.Block8AttnArgs) == 12 * 4 + 2 * 8 + 13 * 8
    assert L.Block8AttnArgs.num_blocks.offset == 48 and L.Block8AttnArgs.q.offset == 64


def test_append_status(L):
    f = L.lib.jf_block8_append
    ok = [16, 16, 0, 4, 2, 256, 128, 256, 128, 16, 16, 1, 16, 0, 4, 4, 0, 16, 16, 16, 16, 8, None]
    def call(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return f(*a)
    for bad in (dict(_2=2), dict(_16=2), dict(_3=-1), dict(_4=0), dict(_11=-1), dict(_15=-1), dict(_21=-1), dict(_0=None), dict(_9=None),
                dict(_12=None), dict(_17=None), dict(_17=20), dict(_18=None), dict(_18=18)):
        assert call(**bad) == L.JF_ERR_ARG, bad
    assert call(_3=0) == L.JF_OK and call(_11=0) == L.JF_OK          # nothing to do, nothing launched
    assert call(_3=2 ** 31) == L.JF_ERR_ARG


def _args(L, **kw):
    a = L.Block8AttnArgs()
    a.codes, a.q_dtype, a.B, a.H_q, a.H_kv, a.max_S, a.max_blocks = 0, 0, 2, 8, 2, 100, 8
    a.num_blocks, a.bt_stride, a.attn_scale = 16, 8, 0.1
    for n in ("q", "k_data", "k_scales", "v_data", "v_scales", "block_table", "seq_lens", "out"):
        setattr(a, n, 4096)
    a.workspace, a.workspace_bytes = 4096, L.lib.jf_block8_workspace_bytes(2, 8, 2, 100)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_attn_status(L):
    f = lambda **kw: L.lib.jf_block8_attn(C.byref(_args(L, **kw)), None)
    assert L.lib.jf_block8_attn(None, None) == L.JF_ERR_ARG
    for bad in (dict(codes=2), dict(q_dtype=7), dict(B=-1), dict(H_q=0), dict(H_q=7), dict(H_kv=0), dict(max_S=0), dict(max_blocks=-1),
                dict(window=-1), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(q=None), dict(q=4100),
                dict(k_data=None), dict(k_data=4104), dict(v_scales=None), dict(block_table=None), dict(seq_lens=None), dict(out=None)):
        assert f(**bad) == L.JF_ERR_ARG, bad
    assert f(workspace=None) == L.JF_ERR_WORKSPACE and f(workspace_bytes=64) == L.JF_ERR_WORKSPACE and f(workspace=4100) == L.JF_ERR_WORKSPACE
    assert f(max_blocks=2 ** 28) == L.JF_ERR_UNSUPPORTED
    assert f(B=0) == L.JF_OK


def test_workspace_bytes(L):
    w = L.lib.jf_block8_workspace_bytes
    assert w(0, 8, 2, 100) == 0 and w(1, 8, 3, 100) == 0 and w(1, 8, 2, 0) == 0 and w(2 ** 30, 8, 2, 100000) == 0
    assert 0 < w(1, 8, 2, 1) <= w(4, 64, 8, 131072)


def test_ops_refuse_what_is_no_cuda_tensor_or_no_cache(L):
    from jetfire_b200 import ops
    z = torch.zeros
    key, start, lens, table = z(4, 2, 128, dtype=torch.bfloat16), z(2, dtype=torch.int32), z(1, dtype=torch.int32), z(1, 4, dtype=torch.int64)
    data, scales = z(2, 32, 128, dtype=torch.int8), z(2, 2)
    with pytest.raises(RuntimeError, match="CUDA tensor of the current device"):
        ops.block8_append(key, key, start, lens, table, data, scales, data, scales)
    with pytest.raises(RuntimeError, match="must be a tensor"):
        ops.block8_append(key, None, start, lens, table, None, scales, data, scales)
    with pytest.raises(RuntimeError, match="CUDA tensor of the current device"):
        ops.block8_decode_attn(z(1, 4, 128), data, scales, data, scales, table, lens, 64, 4, 2, 16, 0.1)
    for w in (0, -5):
        with pytest.raises(RuntimeError, match="window"):
            ops.block8_decode_attn(z(1, 4, 128), data, scales, data, scales, table, lens, 64, 4, 2, 16, 0.1, window=w)


@pytest.mark.gpu
def test_ops_refuse_wrong_shapes_and_types(L):
    from jetfire_b200 import ops
    def z(*s, dtype=torch.float32):
        return torch.zeros(*s, dtype=dtype, device="cuda")
    i32, i64, bf = torch.int32, torch.int64, torch.bfloat16
    good = dict(key=z(4, 2, 128, dtype=bf), value=z(4, 2, 128, dtype=bf), start=z(2, dtype=i32), lens=z(1, dtype=i32), table=z(1, 4, dtype=i64),
                kd=z(2, 32, 128, dtype=torch.int8), ks=z(2, 2), vd=z(2, 32, 128, dtype=torch.int8), vs=z(2, 2))
    ops.block8_append(*good.values())
    for kw in (dict(key=z(4, 3, 128, dtype=bf)), dict(value=z(5, 2, 128, dtype=bf)), dict(value=z(4, 2, 128, dtype=torch.float16)),
               dict(key=z(4, 2, 128)), dict(key=z(4, 2, 64, dtype=bf)), dict(start=z(3, dtype=i32)), dict(start=z(2, dtype=i64)),
               dict(lens=z(1, dtype=i64)), dict(lens=z(1, 1, dtype=i32)), dict(table=z(2, 4, dtype=i64)), dict(table=z(1, 4)), dict(table=z(4, dtype=i64)),
               dict(kd=z(2, 32, 128, dtype=torch.uint8)), dict(kd=z(2, 33, 128, dtype=torch.int8)), dict(vd=z(2, 48, 128, dtype=torch.int8)),
               dict(vd=z(2, 32, 128, dtype=torch.float8_e4m3fn)), dict(ks=z(2, 3)), dict(ks=z(2, 2, dtype=bf)), dict(vs=z(2, 4)[:, ::2]),
               dict(kd=z(32, 2, 128, dtype=torch.int8).transpose(0, 1)), dict(ks=torch.zeros(2, 2))):
        with pytest.raises(RuntimeError, match="block8_append"):
            ops.block8_append(*{**good, **kw}.values())
    call = dict(q=z(1, 4, 128, dtype=bf), kd=good["kd"], ks=good["ks"], vd=good["vd"], vs=good["vs"], table=good["table"], lens=good["lens"],
                max_S=64, H_q=4, H_kv=2, block_size=16, scale=0.1)
    ops.block8_decode_attn(*call.values())
    for kw in (dict(q=z(2, 4, 128, dtype=bf)), dict(q=z(1, 4, 128)), dict(H_q=3), dict(H_q=0), dict(H_kv=4), dict(max_S=0), dict(block_size=32),
               dict(table=z(2, 4, dtype=i64)), dict(lens=z(1, dtype=i64))):
        with pytest.raises(RuntimeError):
            ops.block8_decode_attn(*{**call, **kw}.values())
    for kw in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(window=0), dict(alibi_slopes=z(3)), dict(alibi_slopes=z(4, dtype=bf)),
               dict(prefix_lens=z(2, dtype=i32)), dict(prefix_lens=z(1)), dict(out=z(1, 4, 128)), dict(workspace=z(8)),
               dict(out=z(1, 4, 256, dtype=bf)[..., ::2])):
        with pytest.raises(RuntimeError):
            ops.block8_decode_attn(*call.values(), **kw)


# ---- packed prompts -----------------------------------------------------------------------


def _varlen(L, **kw):
    a = L.VarlenAttnArgs()
    a.dtype, a.n_seqs, a.H_q, a.H_kv, a.causal, a.attn_scale, a.T = 0, 2, 8, 2, 1, 0.1, 40
    a.q_stride_t, a.q_stride_h, a.k_stride_t, a.k_stride_h, a.v_stride_t, a.v_stride_h = 1024, 128, 256, 128, 256, 128
    for n in ("q", "k", "v", "cu_seqlens", "out"):
        setattr(a, n, 4096)
    for k, v in kw.items():
        setattr(a, k, v)
    return L.lib.jf_varlen_attn(C.byref(a), None)


def test_varlen_status(L):
    assert C.sizeof(L.VarlenAttnArgs) == 8 * 4 + 7 * 8 + 9 * 8
    assert L.lib.jf_varlen_attn(None, None) == L.JF_ERR_ARG
    for bad in (dict(dtype=3), dict(n_seqs=-1), dict(H_q=0), dict(H_q=7), dict(H_kv=0), dict(window=-1), dict(softcap=-1.0),
                dict(softcap=float("nan")), dict(T=-1), dict(q=None), dict(k=None), dict(v=None), dict(cu_seqlens=None), dict(out=None), dict(q=4104),
                dict(k=4098), dict(v=4100), dict(out=4104), dict(status_record=4100), dict(q_stride_t=1028), dict(k_stride_h=0), dict(v_stride_t=-256)):
        assert _varlen(L, **bad) == L.JF_ERR_ARG, bad
    assert _varlen(L, T=2 ** 31) == L.JF_ERR_UNSUPPORTED
    assert _varlen(L, T=0) == L.JF_OK and _varlen(L, n_seqs=0) == L.JF_OK


@pytest.mark.gpu
def test_varlen_refuses_wrong_shapes_and_types(L):
    from jetfire_b200 import ops
    def z(*s, dtype=torch.bfloat16):
        return torch.zeros(*s, dtype=dtype, device="cuda")
    i32 = torch.int32
    good = dict(q=z(9, 4, 128), k=z(9, 2, 128), v=z(9, 2, 128), cu=torch.tensor([0, 9], dtype=i32, device="cuda"), scale=0.1)
    ops.varlen_prefill_attn(*good.values())
    for kw in (dict(q=z(9, 3, 128)), dict(q=z(9, 4, 64)), dict(k=z(8, 2, 128)), dict(v=z(9, 1, 128)), dict(v=z(9, 2, 128, dtype=torch.float16)),
               dict(q=z(9, 4, 128, dtype=torch.float32)), dict(cu=torch.tensor([0, 9], device="cuda")), dict(cu=torch.tensor([0, 9], dtype=i32)),
               dict(cu=z(1, 2, dtype=i32)), dict(q=torch.zeros(9, 4, 128, dtype=torch.bfloat16))):
        with pytest.raises(RuntimeError):
            ops.varlen_prefill_attn(*{**good, **kw}.values())
    for kw in (dict(window=0), dict(window=-3), dict(softcap=-1.0), dict(softcap=float("nan")), dict(alibi_slopes=z(4)), dict(alibi_slopes=z(3, dtype=torch.float32)),
               dict(prefix_lens=z(2, dtype=i32)), dict(out=z(9, 4, 128, dtype=torch.float16)), dict(out=z(9, 4, 256)[..., ::2]),
               dict(status_record=z(4)), dict(out=z(8, 4, 128))):
        with pytest.raises(RuntimeError):
            ops.varlen_prefill_attn(*good.values(), **kw)
