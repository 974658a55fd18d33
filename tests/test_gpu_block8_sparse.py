"""Attention over selected blocks of the 8-bit cache: the choice exactly, the outputs against the definition in 64 bits over the
chosen blocks, with the tolerances of the decode attention (it is that arithmetic)."""
import pytest
import torch

import block8_more_ref as M
import block8_ref as R
from test_gpu_block8 import Decode

pytestmark = pytest.mark.gpu
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Sparse(Decode):
    def __init__(self, lens, H_q, H_kv, codes, dtype, seed, *, top, first=1, last=2, softcap=0.0, **kw):
        super().__init__(lens, H_q, H_kv, codes, dtype, seed, softcap=softcap, **kw)
        self.top, self.first, self.last = top, first, last
        self.bounds = torch.stack([M.bounds_of(self.k[:, i], 16, codes) for i in range(self.blocks)], 1).to(torch.int8)

    def expected(self):
        out = torch.zeros(len(self.lens), self.H_q, 128, dtype=torch.float64)
        lse = torch.full((len(self.lens), self.H_q), float("-inf"), dtype=torch.float64)
        self.chosen = torch.full((len(self.lens), self.H_kv, self.top), -1, dtype=torch.int32)
        k, v, G = self.k * self.ks[..., None, None], self.v * self.vs[..., None, None], self.H_q // self.H_kv
        for b, length in enumerate(self.lens):
            length = min(max(length, 0), self.max_S)
            n = (length + 15) // 16
            for g in range(self.H_kv):
                heads = slice(g * G, (g + 1) * G)
                pick = M.choose(self.q[b, heads].double(), self.bounds[g], self.ks[g], self.table[b], n, self.top, self.first, self.last, self.codes,
                                self.blocks)
                self.chosen[b, g, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
                j = torch.tensor([p * 16 + r for p in pick for r in range(16) if p * 16 + r < length], dtype=torch.long)
                ids = self.table[b][j // 16]
                j, ids = j[(ids >= 0) & (ids < self.blocks)], ids[(ids >= 0) & (ids < self.blocks)]
                if len(j):
                    o, l = R.attend(self.q[b, heads].double()[:, None], k[g, ids, j % 16][None], v[g, ids, j % 16][None], torch.tensor([length - 1]), j,
                                    self.scale, softcap=self.kw["softcap"])
                    out[b, heads], lse[b, heads] = o[:, 0], l[:, 0]
        return out, lse

    def device(self):
        a = super().device()
        return (*a[:5], self.bounds.cuda(), *a[5:])

    def run(self, args=None, **kw):
        from jetfire_b200 import ops
        return ops.block8_sparse_decode_attn(*(args or self.device()), top_blocks=self.top, first_blocks=self.first, last_blocks=self.last,
                                             softcap=self.kw["softcap"], **kw)

    def check(self, out, lse, chosen):
        super().check(out, lse)
        assert torch.equal(chosen.cpu(), self.chosen)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens, top", [([1], 4), ([0, 64, 65, 80], 4), ([49, 48, 47, 33], 3), ([700, 3, 0, 257], 8), ([2049], 20), ([20000], 64),
                                       ([16 * 1000 + 5, 16 * 999], 998)])
def test_lengths(codes, lens, top):
    c = Sparse(lens, 8, 2, CODES[codes], torch.bfloat16, 51, top=top)
    c.check(*c.run())


@pytest.mark.parametrize("H_q, H_kv", [(1, 1), (3, 1), (8, 8), (64, 8), (9, 1), (16, 1), (40, 1), (24, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_heads_and_types(H_q, H_kv, dtype):
    for codes in CODES.values():
        c = Sparse([1500, 900], H_q, H_kv, codes, dtype, 52, top=10, softcap=20.0 if H_q == 64 else 0.0)
        c.check(*c.run())


@pytest.mark.parametrize("top, first, last", [(1, 0, 1), (2, 1, 1), (6, 4, 2), (7, 0, 7), (7, 0, 1), (30, 3, 9), (94, 1, 1), (95, 0, 5)])
def test_first_and_last_blocks(top, first, last):
    c = Sparse([1505, 300, 1500], 8, 2, torch.int8, torch.bfloat16, 53, top=top, first=first, last=last)
    c.check(*c.run())


@pytest.mark.parametrize("n, H_kv", [(8192, 1), (5000, 2), (3000, 8)])
def test_rows_shared_by_clusters(n, H_kv):
    c = Sparse([n * 16 - 3], 4 * H_kv, H_kv, torch.int8, torch.bfloat16, 54, top=200)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens", [[16 * 2000], [16 * 100, 16 * 700]])
def test_equal_scores_go_to_the_lower_blocks(codes, lens):
    """All keys alike; then a few values only, many blocks each."""
    c = Sparse(lens, 4, 1, CODES[codes], torch.bfloat16, 55, top=70)
    c.k[:] = c.k[:, :1, :1]
    c.ks[:] = c.ks[:, :1]
    c.bounds = torch.stack([M.bounds_of(c.k[:, i], 16, c.codes) for i in range(c.blocks)], 1).to(torch.int8)
    c.check(*c.run())
    c.ks *= 2.0 ** torch.randint(0, 3, c.ks.shape, generator=torch.Generator().manual_seed(1))
    c.check(*c.run())


@pytest.mark.parametrize("spread", [0, 20, 60])
def test_scores_of_any_size_and_sign(spread):
    """K scales far apart, queries against the keys: scores below zero, ranges that take several rounds."""
    for sign in (1, -1):
        c = Sparse([16 * 1500, 16 * 300 + 1], 4, 1, torch.int8, torch.bfloat16, 56, top=33)
        g = torch.Generator().manual_seed(2)
        c.k = torch.randint(40, 128, c.k.shape, generator=g).double()
        c.q = (c.q.abs() * sign * 2.0 ** -spread).to(c.q.dtype)
        c.ks = R.fl32(c.ks * torch.exp2(spread * torch.rand(c.ks.shape, generator=g, dtype=torch.float64)))
        c.bounds = torch.stack([M.bounds_of(c.k[:, i], 16, c.codes) for i in range(c.blocks)], 1).to(torch.int8)
        c.check(*c.run())


def test_bounds_are_all_that_the_choice_goes_by():
    c = Sparse([16 * 600], 8, 2, torch.int8, torch.float16, 57, top=40)
    c.bounds = torch.randint(-128, 128, c.bounds.shape, generator=torch.Generator().manual_seed(3)).to(torch.int8)
    c.check(*c.run())


def test_blocks_that_are_not_there_and_scales_that_are_no_numbers():
    c = Sparse([16 * 300 + 7, 16 * 50], 4, 1, torch.int8, torch.bfloat16, 58, top=20)
    c.table[0, 5:280] = -1                   # fewer scores than places: of the rest the first
    c.table[1, 7] = c.blocks
    c.ks[0, c.table[0, 290]] = 0.0
    c.check(*c.run())
    c = Sparse([16 * 300], 4, 1, torch.int8, torch.bfloat16, 59, top=20)
    c.ks[0, c.table[0, 100:200]] = float("nan")
    c.check(*c.run())
    c = Sparse([16 * 300], 4, 1, torch.int8, torch.bfloat16, 59, top=20)
    c.table[:] = -1                          # nothing at all
    c.check(*c.run())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads", [[1], [0, 1, 2, 3]])
def test_queries_that_are_no_numbers(bad, heads):
    """They do not count in the choice; their own rows are NaN."""
    c = Sparse([16 * 100], 4, 1, torch.int8, torch.bfloat16, 60, top=9)
    clean = c.q.clone()
    c.q[0, heads, 5] = bad
    out, lse, chosen = c.run()
    c.expected()
    assert torch.equal(chosen.cpu(), c.chosen)
    assert torch.isnan(out[0, heads]).all()
    rest = [h for h in range(4) if h not in heads]
    if rest:
        want, _ = c.expected()
        c.q = clean
        assert (out[0, rest].double().cpu() - want[0, rest]).abs().max() < 0.05


def test_zero_queries_choose_the_first():
    c = Sparse([16 * 100], 4, 1, torch.float8_e4m3fn, torch.bfloat16, 61, top=9)
    c.q.zero_()
    c.check(*c.run())


def test_tables_of_32_bits_views_lengths_and_max_S():
    c = Sparse([1500, 900], 8, 2, torch.int8, torch.bfloat16, 62, top=10, table_dtype=torch.int32)
    a = list(c.device())
    wide = torch.full((2, c.table.shape[1] + 9), -7, dtype=torch.int32, device="cuda")
    wide[:, 3:-6] = a[6]
    a[6] = wide[:, 3:-6]
    c.check(*c.run(a))
    a[7] = torch.tensor([10 ** 9, -4], dtype=torch.int32).cuda()      # cut to max_S and to zero
    c.lens = [1500, 0]
    c.check(*c.run(a))
    a[8], c.max_S, c.lens = 1000, 1000, [1000, 0]
    c.check(*c.run(a))


def test_no_sequences_no_blocks_and_no_columns():
    from jetfire_b200 import ops
    c = Sparse([300], 4, 1, torch.int8, torch.bfloat16, 63, top=5)
    a = list(c.device())
    out, lse, chosen = c.run([a[0][:0], *a[1:6], a[6][:0], a[7][:0], *a[8:]])
    assert out.shape == (0, 4, 128) and chosen.shape == (0, 1, 5)
    out, lse, chosen = c.run([*a[:6], a[6][:, :0], *a[7:]])
    assert (out == 0).all() and (lse == float("-inf")).all() and (chosen == -1).all()
    none = [a[0], a[1][:, :0], a[2][:, :0], a[3][:, :0], a[4][:, :0], a[5][:, :0], *a[6:]]
    out, lse, chosen = ops.block8_sparse_decode_attn(*[x.contiguous() if torch.is_tensor(x) else x for x in none], top_blocks=5)
    assert (out == 0).all() and (lse == float("-inf")).all() and chosen.cpu().tolist() == [[[0, 1, 2, 17, 18]]]


def test_caller_owned_output_and_workspace_and_the_same_bits_again():
    from jetfire_b200 import ops
    c = Sparse([15000, 700], 8, 2, torch.float8_e4m3fn, torch.float16, 64, top=60)
    out = torch.full((2, 8, 128), 9.0, dtype=torch.float16, device="cuda")
    ws = torch.empty(ops.block8_sparse_workspace_bytes(2, 8, 2, c.max_S, 60) + 256, dtype=torch.uint8, device="cuda")
    got = c.run(out=out, workspace=ws)
    assert got[0].data_ptr() == out.data_ptr()
    c.check(*got)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(c.run(), got))


def test_two_calls_at_once_on_two_streams():
    cases = [Sparse([3000, 17, 900], 8, 2, torch.int8, torch.bfloat16, 65, top=12), Sparse([20000], 16, 1, torch.float8_e4m3fn, torch.float16, 66, top=100)]
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


@pytest.mark.parametrize("codes", CODES)
def test_a_decode_loop_in_a_graph(codes):
    """Rotated append with bounds, then the sparse attention: captured once, replayed while the sequences grow past the number of chosen
    blocks; a cache that begins empty."""
    from jetfire_b200 import ops
    code, top, H_q, H_kv, B = CODES[codes], 4, 4, 2, 3
    c = Sparse([200, 200, 200], H_q, H_kv, code, torch.bfloat16, 67, top=top)
    cos_sin = M.table_of(128, 256)
    k, v = (torch.zeros_like(c.k) for _ in range(2))
    ks, vs = (torch.zeros_like(c.ks) for _ in range(2))
    to = lambda x: x.float().to(code).view(H_kv, -1, 128).cuda()
    kd, vd, ksd, vsd, bounds = to(k), to(v), ks.float().cuda(), vs.float().cuda(), torch.zeros_like(c.bounds).cuda()
    table, start = c.table.cuda(), torch.arange(B + 1, dtype=torch.int32).cuda()
    lens0 = [30, 62, 100]
    g = torch.Generator().manual_seed(9)
    T = sum(lens0)
    prompt = [torch.randn(T, h, 128, generator=g).to(torch.bfloat16) for h in (H_q, H_kv, H_kv)]
    starts = [0, 30, 92, 192]
    positions = torch.cat([torch.arange(n) for n in lens0])
    ops.block8_append_rotary(*(x.cuda() for x in prompt), positions.cuda(), cos_sin.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(),
                             torch.tensor(lens0, dtype=torch.int32).cuda(), table, kd, ksd, vd, vsd, bounds=bounds)
    R.append(M.rotated(prompt[1], M.turns(cos_sin, positions), False), starts, lens0, c.table, k, ks, code)
    R.append(prompt[2], starts, lens0, c.table, v, vs, code)
    lens, pos, turn = torch.tensor(lens0, dtype=torch.int32).cuda(), torch.tensor(lens0).cuda(), cos_sin.cuda()
    q, key, value = (torch.zeros(B, h, 128, dtype=torch.bfloat16, device="cuda") for h in (H_q, H_kv, H_kv))

    def step():
        lens.add_(1)
        turned = ops.block8_append_rotary(q, key, value, pos, turn, start, lens, table, kd, ksd, vd, vsd, bounds=bounds)
        pos.add_(1)
        return turned, ops.block8_sparse_decode_attn(turned, kd, ksd, vd, vsd, bounds, table, lens, 200, H_q, H_kv, 16, c.scale, top_blocks=top)

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        turned, got = step()
    now = list(lens0)
    for i in range(20):
        new = [torch.randn(B, h, 128, generator=g).to(torch.bfloat16) for h in (H_q, H_kv, H_kv)]
        for x, y in zip((q, key, value), new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        turns = M.turns(cos_sin, torch.tensor(now))
        now = [n + 1 for n in now]
        R.append(M.rotated(new[1], turns, False), list(range(B + 1)), now, c.table, k, ks, code)
        R.append(new[2], list(range(B + 1)), now, c.table, v, vs, code)
        assert torch.equal(kd.cpu().double().view(k.shape), k) and torch.equal(ksd.cpu().double(), ks) and torch.equal(vd.cpu().double().view(v.shape), v)
        c.q = M.rotated(new[0], turns, False).float().to(torch.bfloat16)
        assert torch.equal(turned.cpu(), c.q)
        c.k, c.v, c.ks, c.vs, c.lens, c.bounds = k, v, ks, vs, now, bounds.cpu()
        for b, n in enumerate(now):       # bounds hold what the blocks hold, up to the last position
            for blk in range((n + 15) // 16):
                at = c.table[b, blk]
                assert torch.equal(c.bounds[:, at].double(), M.bounds_of(k[:, at], min(16, n - blk * 16), code))
        c.check(*got)


def test_a_row_longer_than_shared_memory():
    """50000 blocks: the choice exactly, the outputs as the decode attention gives them over a table of the chosen blocks."""
    from jetfire_b200 import ops
    n, top = 50000, 300
    g = torch.Generator(device="cuda").manual_seed(6)
    kd, vd = (torch.randint(-127, 128, (1, n * 16, 128), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
    ks, vs = (torch.rand(1, n, device="cuda", generator=g) * 0.02 + 0.001 for _ in range(2))
    rows = kd.view(1, n, 16, 128)
    bounds = torch.stack([rows.amin(2), rows.amax(2)], 2)
    table = torch.randperm(n, device="cuda", generator=g)[None]
    q = torch.randn(1, 4, 128, device="cuda", generator=g).bfloat16()
    lens = torch.tensor([n * 16 - 5], dtype=torch.int32, device="cuda")
    out, lse, chosen = ops.block8_sparse_decode_attn(q, kd, ks, vd, vs, bounds, table, lens, n * 16, 4, 1, 16, 0.05, top_blocks=top)
    pick = M.choose(q[0].double().cpu(), bounds[0].cpu(), ks[0].double().cpu(), table[0].cpu(), n, top, 1, 2, torch.int8, n)
    assert chosen[0, 0].tolist() == pick
    want, want_lse = ops.block8_decode_attn(q, kd, ks, vd, vs, table[:, chosen[0, 0].long()].contiguous(), lens - (n - top) * 16, top * 16, 4, 1, 16, 0.05)
    tol = 2 * ((2 ** -11 + 2 ** -14) * 127 * 0.021 + 2 ** -8 * want.float().abs())
    assert ((out.float() - want.float()).abs() <= tol).all() and (lse - want_lse).abs().max() <= 2 ** -12
