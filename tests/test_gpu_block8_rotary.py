"""The rotated append into the 8-bit cache: bit for bit the plain form's queries, codes, scales and bounds."""
import pytest
import torch

import block8_more_ref as M
import block8_ref as R

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16


class Step:
    def __init__(self, news, olds, *, H_q=4, H_kv=2, codes=INT8, dtype=BF16, rot=128, interleaved=False, table=torch.float32, layout="own", seed=0,
                 pad=0, rows=700):
        g = torch.Generator().manual_seed(seed)
        self.news, self.olds, self.codes, self.interleaved = news, olds, codes, interleaved
        lens = [o + n for o, n in zip(olds, news)]
        need = [(l + 15) // 16 for l in lens]
        self.c = M.Cache(H_kv, sum(need) + 3, codes, seed + 1)
        perm = torch.randperm(self.c.blocks, generator=g)
        self.table = torch.full((len(news), max(need) + 1), -1, dtype=torch.int64)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        T = sum(news) + pad
        both = torch.randn(T, H_q + 2 * H_kv, 128, generator=g).mul_(torch.exp(0.5 * torch.randn(1, H_q + 2 * H_kv, 128, generator=g))).to(dtype)
        self.host = both[:, :H_q], both[:, H_q:H_q + H_kv], both[:, H_q + H_kv:]
        dev = both.cuda()
        if layout == "qkv":
            self.qkv = dev[:, :H_q], dev[:, H_q:H_q + H_kv], dev[:, H_q + H_kv:]
        elif layout == "odd":      # rows that start on odd addresses
            self.qkv = tuple(torch.zeros(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(x) for x in self.host)
        else:
            self.qkv = tuple(x.contiguous().cuda() for x in self.host)
        self.start = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.positions = torch.tensor([p for o, l in zip(olds, lens) for p in range(o, l)] + [0] * pad)
        self.cos_sin = M.table_of(rot, rows, table)
        self.bounds = torch.full((H_kv, self.c.blocks, 2, 128), 77, dtype=torch.int8, device="cuda")

    def run(self, bounds=True, **kw):
        from jetfire_b200 import ops
        return ops.block8_append_rotary(*self.qkv, self.positions.cuda(), self.cos_sin.cuda(), self.start.cuda(), self.lens.cuda(), self.table.cuda(),
                                        *self.c.tensors(), interleaved=self.interleaved, bounds=self.bounds if bounds else None, **kw)

    def expect(self, bounds=True):
        """Moves the plain cache on; -> rotated queries, bounds."""
        turn = M.turns(self.cos_sin, self.positions)
        key = M.rotated(self.host[1], turn, self.interleaved)
        R.append(key, self.start, self.lens, self.table, self.c.code[0], self.c.scale[0], self.codes)
        R.append(self.host[2], self.start, self.lens, self.table, self.c.code[1], self.c.scale[1], self.codes)
        want = torch.full((self.c.H, self.c.blocks, 2, 128), 77.0, dtype=torch.float64)
        for s, (o, n) in enumerate(zip(self.olds, self.news)):
            for blk in range(o // 16, (o + n + 15) // 16):
                i = int(self.table[s, blk])
                if 0 <= i < self.c.blocks:
                    want[:, i] = M.bounds_of(self.c.code[0][:, i], min(16, o + n - 16 * blk), self.codes)
        return M.rotated(self.host[0], turn, self.interleaved), want

    def check(self, q, rows=None):
        want, bounds = self.expect()
        rows = rows or slice(None)
        assert torch.equal(q.cpu()[rows], want.float().to(q.dtype)[rows])
        self.c.same()
        assert torch.equal(self.bounds.cpu().double(), bounds)


@pytest.mark.parametrize("codes", [INT8, E4M3])
@pytest.mark.parametrize("dtype, rot, interleaved, table, layout", [
    (BF16, 128, False, torch.float32, "own"), (FP16, 128, True, torch.float32, "qkv"), (BF16, 64, False, BF16, "qkv"), (FP16, 96, False, FP16, "odd"),
    (BF16, 32, True, BF16, "own"), (FP16, 16, False, torch.float32, "odd"), (BF16, 112, True, torch.float32, "odd"), (FP16, 80, False, FP16, "own")])
def test_rotations_types_and_layouts(codes, dtype, rot, interleaved, table, layout):
    s = Step([1, 17, 16, 33, 5, 1], [0, 5, 16, 15, 11, 47], codes=codes, dtype=dtype, rot=rot, interleaved=interleaved, table=table, layout=layout, seed=rot)
    s.check(s.run())


@pytest.mark.parametrize("news, olds", [([1], [0]), ([1] * 40, list(range(40))), ([300], [3]), ([2, 3] * 9, [7, 31] * 9)])
@pytest.mark.parametrize("H_q, H_kv", [(1, 1), (16, 2), (5, 5), (64, 8)])
def test_lengths_and_heads(news, olds, H_q, H_kv):
    s = Step(news, olds, H_q=H_q, H_kv=H_kv, codes=E4M3 if H_q == 16 else INT8, seed=len(news))
    s.check(s.run())


def test_a_large_step_takes_several_heads_a_warp():
    s = Step([1300], [9], H_q=64, H_kv=1, rows=1400)
    s.check(s.run())


def test_large_step_with_an_odd_number_of_heads():
    s = Step([6500], [0], H_q=13, H_kv=1, rows=6500, codes=E4M3, dtype=FP16)
    s.check(s.run())


@pytest.mark.parametrize("codes", [INT8, E4M3])
def test_tokens_one_by_one_grow_scales_and_bounds(codes):
    """Sixteen and more single tokens of growing size into one block: scales grow, earlier codes are rounded again, bounds follow."""
    first = Step([3], [0], codes=codes, seed=5)
    first.table = torch.tensor([[2, 0, 1]])
    first.check(first.run())
    for i in range(3, 20):
        s = Step([1], [i], codes=codes, seed=100 + i)
        s.c, s.table, s.bounds = first.c, first.table, first.bounds
        scale = 2.0 ** (i - 10)
        s.host = tuple((x * scale).to(BF16) for x in s.host)
        s.qkv = tuple(x.cuda().contiguous() for x in s.host)
        before = first.bounds.clone()
        q = s.run()
        want, bounds = s.expect()
        at = int(first.table[0, i // 16])
        before[:, at] = bounds[:, at].to(torch.int8).cuda()
        assert torch.equal(q.cpu(), want.float().to(BF16))
        s.c.same()
        assert torch.equal(s.bounds, before)


def test_no_numbers():
    """NaN and infinities: 0 and the largest code, neither in the scale; products with them are no numbers either."""
    for codes in (INT8, E4M3):
        s = Step([40], [3], codes=codes, rot=64)
        for x in s.host:
            x[2, 0, 3], x[5, 0, 100], x[7, 0, 90], x[20, 0, 40] = float("nan"), float("inf"), float("-inf"), float("inf")
        s.qkv = tuple(x.contiguous().cuda() for x in s.host)
        q = s.run()
        want, bounds = s.expect()
        want = want.float().to(BF16)
        assert torch.equal(torch.isnan(q.cpu()), torch.isnan(want)) and torch.equal(torch.nan_to_num(q.cpu(), 0.5), torch.nan_to_num(want, 0.5))
        s.c.same()
        assert torch.equal(s.bounds.cpu().double(), bounds)


def test_positions_outside_of_the_table():
    s = Step([20, 2], [0, 4], rot=64, H_q=2)
    s.positions[3], s.positions[9], s.positions[21] = 700, -1, 2 ** 40
    q = s.run().cpu()
    want, bounds = s.expect()
    want = want.float().to(BF16)
    assert torch.isnan(q[3, :, :64]).all() and torch.equal(q[3, :, 64:], s.host[0][3, :, 64:])
    assert torch.equal(torch.nan_to_num(q, 9.0), torch.nan_to_num(want, 9.0))
    s.c.same()
    assert torch.equal(s.bounds.cpu().double(), bounds)


def test_rows_behind_the_last_sequence_stay():
    s = Step([3, 2], [0, 30], pad=6)
    out = torch.full((11, 4, 128), 5.0, dtype=BF16, device="cuda")
    q = s.run(out=out)
    assert q.data_ptr() == out.data_ptr() and (q[5:] == 5.0).all()
    s.check(q, slice(0, 5))


def test_in_place_with_32_bit_positions_and_table():
    from jetfire_b200 import ops
    s = Step([9, 1], [14, 2])
    q = s.qkv[0]
    got = ops.block8_append_rotary(*s.qkv, s.positions.int().cuda(), s.cos_sin.cuda(), s.start.cuda(), s.lens.cuda(), s.table.int().cuda(), *s.c.tensors(),
                                   bounds=s.bounds, out=q)
    assert got.data_ptr() == q.data_ptr()
    s.check(got)


def test_blocks_that_are_not_there_are_skipped():
    s = Step([40, 20], [0, 0])
    s.table[0, 1], s.table[1, 0] = -1, s.c.blocks
    s.check(s.run())


def test_empty_calls():
    from jetfire_b200 import ops
    s = Step([4], [0])
    q, k, v = (x[:0] for x in s.qkv)
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    args = (s.cos_sin.cuda(), zero, zero[:1], s.table.cuda(), *s.c.tensors())
    assert ops.block8_append_rotary(q, k, v, s.positions[:0].cuda(), *args).shape == (0, 4, 128)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = torch.full_like(s.qkv[0], 3.0)
    ops.block8_append_rotary(*s.qkv, s.positions.cuda(), s.cos_sin.cuda(), zero[:1], none, s.table[:0].cuda(), *s.c.tensors(), out=out)
    assert (out == 3.0).all()
    # a table without columns: the queries are rotated all the same
    got = ops.block8_append_rotary(*s.qkv, s.positions.cuda(), s.cos_sin.cuda(), s.start.cuda(), s.lens.cuda(), s.table[:, :0].cuda(), *s.c.tensors())
    assert torch.equal(got.cpu(), M.rotated(s.host[0], M.turns(s.cos_sin, s.positions), False).float().to(BF16))
    # ... and a table of angles without rows turns all into NaN
    got = ops.block8_append_rotary(*s.qkv, s.positions.cuda(), s.cos_sin[:0].cuda(), s.start.cuda(), s.lens.cuda(), s.table[:, :0].cuda(), *s.c.tensors())
    assert torch.isnan(got).all()
    s.c.same()


@pytest.mark.parametrize("codes", [INT8, E4M3])
def test_bounds_of_the_append_without_a_rotation(codes):
    from jetfire_b200 import ops
    s = Step([18, 1, 7], [3, 20, 0], codes=codes, layout="qkv")
    ops.block8_append(s.qkv[1], s.qkv[2], s.start.cuda(), s.lens.cuda(), s.table.cuda(), *s.c.tensors(), bounds=s.bounds)
    s.cos_sin = torch.cat([torch.ones(700, 64), torch.zeros(700, 64)], 1)
    _, bounds = s.expect()
    s.c.same()
    assert torch.equal(s.bounds.cpu().double(), bounds)


def test_captured_and_on_another_stream():
    """A captured call is replayed with other tokens in the same memory."""
    from jetfire_b200 import ops
    a, b = Step([1] * 6, [3, 15, 16, 0, 40, 31], seed=1), Step([1] * 6, [3, 15, 16, 0, 40, 31], seed=1)
    args = (a.positions.cuda(), a.cos_sin.cuda(), a.start.cuda(), a.lens.cuda(), a.table.cuda(), *a.c.tensors())
    out = torch.zeros_like(a.qkv[0])
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.block8_append_rotary(*a.qkv, *args, bounds=a.bounds, out=out)
    for x, y in zip(a.qkv, b.qkv):
        y.mul_(-1.5)
        x.copy_(y)
    b.host = tuple(x.cpu() for x in b.qkv)
    graph.replay()
    torch.cuda.synchronize()
    want, bounds = b.expect()
    assert torch.equal(out.cpu(), want.float().to(BF16)) and torch.equal(a.bounds.cpu().double(), bounds)
    for x, y in zip(a.c.tensors(), (b.c.code[0], b.c.scale[0], b.c.code[1], b.c.scale[1])):
        assert torch.equal(x.cpu().double().view(y.shape), y)
