"""Decode attention over a shared prefix where the sequences are many enough for one product of all rows: the same checks as of few
sequences, on one row tile of a KV head (90 rows), on a pair and a single one (360 rows) and on three pairs (720 rows)."""
import pytest
import torch

import block8_ref as R
from test_gpu_block8_shared import CODES, Shared

pytestmark = pytest.mark.gpu
N, BLOCKS = 90, 30          # 90 sequences, 8 KV heads, 30 blocks: 21600 blocks if each were to read its own
HEADS = [(8, 8), (32, 8), (64, 8)]
OWNS = [(7 * i) % 50 for i in range(N)]


@pytest.mark.parametrize("H_q, H_kv", HEADS)
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_types_and_codes(H_q, H_kv, codes, dtype):
    c = Shared(BLOCKS, OWNS, H_q, H_kv, CODES[codes], dtype, 91, softcap=15.0 if H_q == 64 else 0.0)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("shared", [28, 31, 32, 33, 40])
def test_tiles_that_end_anywhere(codes, shared):
    c = Shared(shared, OWNS + OWNS[:10], 16, 8, CODES[codes], torch.bfloat16, 92)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("softcap", [0.0, 8.0])
def test_sequences_that_end_within_the_shared_positions(codes, softcap):
    owns = [(-480, -479, -100, -1, 0, 5, -17, -352, 33)[i % 9] for i in range(N)]
    c = Shared(BLOCKS, owns, 32, 8, CODES[codes], torch.bfloat16, 93, softcap=softcap)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("spread", [3.0, 12.0])
def test_value_scales_far_apart(codes, spread):
    c = Shared(BLOCKS, OWNS, 16, 8, CODES[codes], torch.bfloat16, 94, v_spread=spread)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
def test_blocks_of_zeros_beside_others_count(codes):
    c = Shared(BLOCKS, OWNS, 32, 8, CODES[codes], torch.bfloat16, 95)
    zero = c.table[0, :BLOCKS:2]
    c.v[:, zero] = 0.0
    c.vs[:, zero] = R.scale_for(torch.zeros(len(zero)), c.codes)
    c.check(*c.run())
    c.v[:] = 0.0
    c.vs[:] = R.scale_for(torch.zeros(1), c.codes)
    c.check(*c.run())


@pytest.mark.parametrize("order", ["rising", "falling", "spiky"])
def test_scores_that_grow_and_fall_along_the_prefix(order):
    c = Shared(100, OWNS, 32, 8, torch.int8, torch.float16, 96)
    f = torch.linspace(0.05, 3.0, 100, dtype=torch.float64)
    f = {"rising": f, "falling": f.flip(0), "spiky": torch.where(torch.arange(100) % 37 == 5, 6.0, 0.2).double()}[order]
    c.ks[:, c.table[0, :100]] *= f
    c.ks = R.fl32(c.ks)
    c.check(*c.run())


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0])
@pytest.mark.parametrize("softcap", [0.0, 1e-20, 3.0, 1e20])
def test_scales_and_caps_of_any_size(scale, softcap):
    c = Shared(BLOCKS, [o - 40 for o in OWNS], 16, 8, torch.int8, torch.bfloat16, 97, softcap=softcap)
    c.scale = scale
    c.q = (c.q.float() * 0.5).to(c.q.dtype)
    c.check(*c.run())


@pytest.mark.parametrize("size", [1e-30, 1e-5, 1e4])
def test_queries_of_any_size(size):
    c = Shared(BLOCKS, OWNS, 16, 8, torch.float8_e4m3fn, torch.bfloat16, 98, q_scale=size)
    c.check(*c.run())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
def test_queries_that_are_no_numbers(bad, softcap):
    """Their rows are NaN, the others to the bit what they are without them."""
    c = Shared(BLOCKS, OWNS, 32, 8, torch.int8, torch.bfloat16, 99, softcap=softcap)
    want, want_lse = c.run()
    c.q[1, 2, 77] = c.q[80, 31, 0] = bad
    out, lse = c.run()
    for b, h in ((1, 2), (80, 31)):
        assert torch.isnan(out[b, h]).all()
        out[b, h], lse[b, h] = want[b, h], want_lse[b, h]
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_blocks_that_are_not_there_and_scales_of_zero():
    c = Shared(BLOCKS, OWNS, 16, 8, torch.int8, torch.bfloat16, 100)
    c.table[:, 3] = -1
    c.table[:, 10:19] = c.blocks
    c.ks[:, c.table[0, 20]] = 0.0
    c.check(*c.run())
    c.table[:, :BLOCKS] = -1
    c.check(*c.run())
    c.table[:] = -1
    c.check(*c.run())


def test_long_parts_of_their_own():
    """Sequences whose own positions are cut into pieces."""
    c = Shared(40, [(3000, 1, 0, 777, 1500)[i % 5] for i in range(70)], 16, 8, torch.int8, torch.bfloat16, 101)
    c.check(*c.run())


def test_many_results_a_row():
    """One KV head over a long prefix: a row's results are joined by several warps."""
    c = Shared(1100, [3, 40, 0] * 7, 8, 1, torch.float8_e4m3fn, torch.float16, 102)
    c.check(*c.run())


def test_one_sequence_over_a_very_long_prefix():
    c = Shared(20500, [9], 4, 1, torch.int8, torch.bfloat16, 103)
    c.check(*c.run())


def test_no_positions_behind_the_prefix_and_a_cut_at_max_S():
    c = Shared(BLOCKS, [0] * N, 16, 8, torch.int8, torch.bfloat16, 104)
    a = list(c.device())
    a[6] = a[6][:, :0]
    c.check(*c.run(a))
    c = Shared(60, OWNS, 16, 8, torch.int8, torch.bfloat16, 105)
    a = list(c.device())
    a[8] = c.max_S = 500
    c.lens = [min(l, 500) for l in c.lens]
    c.check(*c.run(a))


def test_caller_owned_output_and_workspace_and_the_same_bits_again():
    from jetfire_b200 import ops
    c = Shared(BLOCKS, OWNS, 32, 8, torch.float8_e4m3fn, torch.float16, 106)
    out = torch.full((N, 32, 128), 9.0, dtype=torch.float16, device="cuda")
    ws = torch.full((ops.block8_shared_workspace_bytes(N, 32, 8, c.max_S, BLOCKS) + 256,), 255, dtype=torch.uint8, device="cuda")   # (NaN as numbers)
    got = c.run(out=out, workspace=ws)
    assert got[0].data_ptr() == out.data_ptr()
    c.check(*got)
    for _ in range(5):
        assert all(torch.equal(x, y) for x, y in zip(c.run(), got))


def test_two_calls_at_once_on_two_streams():
    cases = [Shared(BLOCKS, OWNS, 32, 8, torch.int8, torch.bfloat16, 107), Shared(45, OWNS, 8, 8, torch.float8_e4m3fn, torch.float16, 108, softcap=9.0)]
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


def test_captured_behind_an_append_and_replayed_with_other_lengths():
    """Appends of the sequences' tokens in front of it in the same graph: what the kernels read was written just before."""
    from jetfire_b200 import ops
    H_q, H_kv = 16, 8
    c = Shared(BLOCKS, [20 + i % 9 for i in range(N)], H_q, H_kv, torch.int8, torch.bfloat16, 109)
    a = list(c.device())
    key, value = (torch.zeros(N, H_kv, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    start = torch.arange(N + 1, dtype=torch.int32, device="cuda")
    whole = torch.cat([a[5].expand(N, -1), a[6]], 1).contiguous()
    lens = a[7]
    lens.sub_(4)
    k, v = (x.double().view(H_kv, -1, 16, 128).cpu() for x in (a[1], a[3]))
    ks, vs = a[2].double().cpu(), a[4].double().cpu()

    def step():
        lens.add_(1)
        ops.block8_append(key, value, start, lens, whole, a[1], a[2], a[3], a[4])
        return c.run(a)

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    now = [l - 4 for l in c.lens]
    for i in range(3):
        new = [torch.randn(N, h, 128, generator=torch.Generator().manual_seed(10 * i + h)).to(torch.bfloat16) for h in (H_q, H_kv, H_kv + 0)]
        for x, y in zip((a[0], key, value), new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        now = [n + 1 for n in now]
        R.append(new[1], list(range(N + 1)), now, c.table, k, ks, torch.int8)
        R.append(new[2], list(range(N + 1)), now, c.table, v, vs, torch.int8)
        c.q, c.lens, c.k, c.v, c.ks, c.vs = new[0], now, k, v, ks, vs
        c.check(*got)
