"""Decode attention over a shared prefix of the 8-bit cache, against the definition in 64 bits with the tolerances of the decode
attention: weights that meet V are fp16, half a step 2^-11 of themselves; scores are sums of 128 fp32 products of exact codes and
a query rounded by 2^-22 of its head's largest element at most, which stands in the exponent below 2^-14."""
import pytest
import torch

import block8_ref as R
from test_gpu_block8 import Decode

pytestmark = pytest.mark.gpu
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Shared(Decode):
    """``owns``: positions behind the shared ones (negative: the sequence ends before)."""

    def __init__(self, shared, owns, H_q, H_kv, codes, dtype, seed, **kw):
        lens = [16 * shared + o for o in owns]
        super().__init__(lens, H_q, H_kv, codes, dtype, seed, **kw)
        self.shared = shared
        self.max_S = max(1, max(lens))
        width = max(self.table.shape[1], shared)
        table = torch.full((len(lens), width), -1, dtype=torch.int64)
        table[:, :self.table.shape[1]] = self.table
        used = torch.randperm(self.blocks, generator=torch.Generator().manual_seed(seed + 7))[:shared]
        assert len(used) == shared
        table[:, :shared] = used      # (the decode attention's plain form knows nothing of sharing)
        free = [i for i in range(self.blocks) if i not in set(used.tolist())]
        at = 0
        for b, o in enumerate(owns):
            for j in range(shared, shared + (max(o, 0) + 15) // 16):
                table[b, j] = free[at]
                at += 1
        self.table = table

    def device(self):
        a = super().device()
        return (*a[:5], a[5][0, :self.shared].contiguous(), a[5][:, self.shared:], *a[6:])

    def run(self, args=None, **kw):
        from jetfire_b200 import ops
        return ops.block8_shared_prefix_attn(*(args or self.device()), softcap=self.kw["softcap"], **kw)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("shared, owns", [(1, [1]), (8, [1, 16, 17]), (7, [5] * 9), (9, [0, 3, 0]), (33, [100, 1, 64, 300]), (64, list(range(1, 33))),
                                          (100, [2] * 70), (500, [40, 3]), (129, [7] * 130)])
def test_lengths(codes, shared, owns):
    c = Shared(shared, owns, 8, 2, CODES[codes], torch.bfloat16, 71)
    c.check(*c.run())


@pytest.mark.parametrize("H_q, H_kv", [(1, 1), (3, 1), (8, 8), (32, 8), (64, 8), (9, 1), (16, 1), (40, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_heads_and_types(H_q, H_kv, dtype):
    for codes in CODES.values():
        c = Shared(40, [5, 0, 33, 16, 1] * 5, H_q, H_kv, codes, dtype, 72, softcap=20.0 if H_q in (9, 64) else 0.0)
        c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("n", [3, 40])
def test_sequences_that_end_within_the_shared_positions(codes, n):
    """Empty ones (padding of a captured batch) among them."""
    c = Shared(20, ([4, -5, -320, 0, -128, -200, -319, 17] * n)[:n], 16, 2, CODES[codes], torch.bfloat16, 73)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("shared", [30, 300])
def test_value_scales_far_apart(codes, shared):
    c = Shared(shared, [50, 20, 9] * 12, 8, 2, CODES[codes], torch.bfloat16, 74, v_spread=6.0)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("n", [2, 40])
def test_blocks_of_zeros_beside_others_count(codes, n):
    """Values of zero have scales near 2^-107: their positions weigh as any others do, in the sum and so in lse."""
    c = Shared(40, [20, 5] * (n // 2), 8, 1, CODES[codes], torch.bfloat16, 75)
    zero = c.table[0, :40:2]
    c.v[:, zero] = 0.0
    c.vs[:, zero] = R.scale_for(torch.zeros(len(zero)), c.codes)
    c.check(*c.run())
    c.v[:] = 0.0
    c.vs[:] = R.scale_for(torch.zeros(1), c.codes)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("order", ["rising", "falling", "spiky"])
def test_scores_that_grow_and_fall_along_the_prefix(codes, order):
    """The reference moves at many places, in a few rows only, by a lot."""
    c = Shared(200, [9, 1, 30] * 20, 8, 2, CODES[codes], torch.float16, 76)
    f = torch.linspace(0.05, 3.0, 200, dtype=torch.float64)
    f = {"rising": f, "falling": f.flip(0), "spiky": torch.where(torch.arange(200) % 37 == 5, 6.0, 0.2).double()}[order]
    c.ks[:, c.table[0, :200]] *= f
    c.ks = R.fl32(c.ks)
    c.check(*c.run())


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0])
@pytest.mark.parametrize("softcap", [0.0, 1e-20, 1e-4, 3.0, 1e20])
def test_scales_and_caps_of_any_size(scale, softcap):
    for codes in CODES.values():
        c = Shared(30, [7, -3, -480] * 15, 8, 2, codes, torch.bfloat16, 77, softcap=softcap)
        c.scale = scale
        c.q = (c.q.float() * 0.5).to(c.q.dtype)
        c.check(*c.run())


@pytest.mark.parametrize("size", [1e-30, 1e-5, 1e4])
def test_queries_of_any_size(size):
    for dtype in (torch.bfloat16, torch.float16):
        if dtype == torch.float16 and size == 1e-30:
            continue
        c = Shared(30, [7, 3] * 20, 8, 2, torch.int8, dtype, 78, q_scale=size)
        c.check(*c.run())


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_no_numbers(bad, n):
    for codes in CODES.values():
        for softcap in (0.0, 5.0):
            c = Shared(30, [7, 3] * (n // 2), 8, 2, codes, torch.bfloat16, 79, softcap=softcap)
            clean = c.q.clone()
            c.q[1, 2, 77] = bad
            out, lse = c.run()
            assert torch.isnan(out[1, 2]).all()
            out[1, 2] = 0
            want = c.run
            c.q = clean
            want, want_lse = c.run()
            want[1, 2] = 0
            lse[1, 2] = want_lse[1, 2]
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("n", [2, 40])
def test_blocks_that_are_not_there(n):
    c = Shared(30, [20, 40] * (n // 2), 8, 2, torch.int8, torch.bfloat16, 80)
    c.table[:, 3] = -1
    c.table[:, 10:19] = c.blocks
    c.table[0, 31] = -5
    c.check(*c.run())
    c.table[:, :30] = -1
    c.check(*c.run())
    c.table[:] = -1
    c.check(*c.run())


@pytest.mark.parametrize("n", [2, 40])
def test_tables_of_32_bits_views_and_lengths(n):
    c = Shared(30, [20, 40] * (n // 2), 8, 2, torch.float8_e4m3fn, torch.float16, 81, table_dtype=torch.int32)
    a = list(c.device())
    wide = torch.full((n, a[6].shape[1] + 9), -7, dtype=torch.int32, device="cuda")
    wide[:, 3:-6] = a[6]
    a[6] = wide[:, 3:-6]
    a[5] = a[5].long()
    c.check(*c.run(a))
    a[7] = torch.tensor(([10 ** 9, -4] * n)[:n], dtype=torch.int32).cuda()       # cut to max_S and to zero
    c.lens = ([c.max_S, 0] * n)[:n]
    for b in range(n):
        c.table[b, 32:] = c.table[1, 32:] if b % 2 else -1
    a[6][:] = c.table[:, 30:].int().cuda()
    c.check(*c.run(a))
    a[8] = c.max_S = 300                                                          # within the shared positions
    c.lens = ([300, 0] * n)[:n]
    c.check(*c.run(a))


@pytest.mark.parametrize("n", [1, 40])
def test_nothing_shared_and_nothing_else(n):
    from jetfire_b200 import ops
    c = Shared(0, [20, 40] * n, 8, 2, torch.int8, torch.bfloat16, 82)
    c.check(*c.run())
    c = Shared(30, [0] * n, 8, 2, torch.int8, torch.bfloat16, 83)
    a = list(c.device())
    a[6] = a[6][:, :0]
    c.check(*c.run(a))
    out, lse = c.run([a[0][:0], *a[1:6], a[6][:0], a[7][:0], *a[8:]])
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    none = [a[0], *(x[:, :0].contiguous() for x in a[1:5]), *a[5:]]
    out, lse = ops.block8_shared_prefix_attn(*none)
    assert (out == 0).all() and (lse == float("-inf")).all()


@pytest.mark.parametrize("n", [2, 40])
def test_caller_owned_output_and_workspace_and_the_same_bits_again(n):
    from jetfire_b200 import ops
    c = Shared(100, [700, 3] * (n // 2), 8, 2, torch.float8_e4m3fn, torch.float16, 84)
    out = torch.full((n, 8, 128), 9.0, dtype=torch.float16, device="cuda")
    ws = torch.full((ops.block8_shared_workspace_bytes(n, 8, 2, c.max_S, 100) + 256,), 255, dtype=torch.uint8, device="cuda")   # (NaN as numbers)
    got = c.run(out=out, workspace=ws)
    assert got[0].data_ptr() == out.data_ptr()
    c.check(*got)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(c.run(), got))


def test_two_calls_at_once_on_two_streams():
    cases = [Shared(300, [17, 90, 300] * 11, 8, 2, torch.int8, torch.bfloat16, 85), Shared(900, [30] * 20, 16, 1, torch.float8_e4m3fn, torch.float16, 86, softcap=9.0)]
    args = [c.device() for c in cases]
    want = [c.run(a) for c, a in zip(cases, args)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(cases[i].run(args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(g, want[i]))
        cases[i].check(*want[i])


@pytest.mark.parametrize("n", [3, 48])
def test_captured_and_replayed_with_other_lengths(n):
    """Two graphs of the same op, replayed in turn while the sequences grow."""
    c = Shared(50, [40 + i % 7 for i in range(n)], 8, 2, torch.int8, torch.bfloat16, 87)
    a = list(c.device())
    graphs, got, stream = [], [], torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            got.append(c.run(a))
    for i in range(4):
        now = [max(0, l - 30 + 10 * i) for l in c.lens]
        a[7].copy_(torch.tensor(now, dtype=torch.int32))
        a[0].copy_(torch.randn(a[0].shape, generator=torch.Generator().manual_seed(i)).to(a[0].dtype))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        d = Shared(50, [l - 800 for l in c.lens], 8, 2, torch.int8, torch.bfloat16, 87)
        d.table, d.lens, d.q, d.max_S = c.table, now, a[0].cpu(), c.max_S
        d.check(*got[i % 2])


@pytest.mark.parametrize("codes", CODES)
def test_the_same_as_the_decode_attention_over_whole_tables(codes):
    """A longer prefix and more rows than the plain form is quick for: against the library's own decode attention, twice its tolerance."""
    from jetfire_b200 import ops
    n, shared, H_q, H_kv = 100, 1000, 32, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    blocks = shared + 4 * n
    code = CODES[codes]
    kd, vd = ((torch.randn(H_kv, blocks * 16, 128, device="cuda", generator=g) * 40).clamp(-127, 127).to(code) for _ in range(2))
    ks, vs = (torch.rand(H_kv, blocks, device="cuda", generator=g) * 0.02 + 0.01 for _ in range(2))
    perm = torch.randperm(blocks, device="cuda", generator=g)
    own = perm[shared:].view(n, 4)
    lens = torch.tensor([16000 + i % 60 for i in range(n)], dtype=torch.int32, device="cuda")
    q = torch.randn(n, H_q, 128, device="cuda", generator=g).bfloat16()
    args = (q, kd, ks, vd, vs)
    rest = (lens, 16064, H_q, H_kv, 16, 128 ** -0.5)
    want, want_lse = ops.block8_decode_attn(*args, torch.cat([perm[:shared].expand(n, shared), own], 1), *rest)
    out, lse = ops.block8_shared_prefix_attn(*args, perm[:shared].contiguous(), own, *rest)
    vmax = (vd.float().abs().amax() * vs.amax()).item()
    tol = 2 * ((2 ** -11 + 2 ** -14) * vmax + 2 ** -8 * want.float().abs())
    assert ((out.float() - want.float()).abs() <= tol).all()
    assert ((lse - want_lse).abs() <= 2 * (2 ** -14 + 2 ** -22 * want_lse.abs())).all()
