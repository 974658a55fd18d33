"""The cache of 8-bit codes: append bit for bit, decode attention against the definition in 64 bits.

Tolerances.  Decode: the weights that meet V are fp16, off by at most half a step, 2^-11 of themselves, so the output
is off by at most 2^-11 * sum p|v| / sum p <= 2^-11 * max|v| of the sequence; scores are sums of 128 fp32 products
(exact codes times q) scaled in fp32: an error of 2^-20 * |q||k| stands in the exponent.  With |s| <= 40 here that is
below 2^-14 of a weight.  On top comes the rounding to the output type, eps / 2 of the value.  lse: 2^-14 + 2^-22 * |lse|."""
import pytest
import torch

import block8_ref as R

pytestmark = pytest.mark.gpu
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _tables(lens, max_blocks, seed, spare=3):
    g = torch.Generator().manual_seed(seed)
    need = [(l + 15) // 16 for l in lens]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=g)
    table = torch.full((len(lens), max_blocks), -1, dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, blocks


def _values(data, blocks):
    return data.cpu().float().double().view(data.shape[0], blocks, 16, 128)


def _cache(H, blocks, codes, seed):
    """Random codes and scales; the rows are whatever a cache may hold."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(H, blocks, 16, 128, generator=g)
    s = R.scale_for(x.abs().amax((2, 3)), codes)
    c = R.encode(R.fl32(x.double() * R.fl32(1 / s)[..., None, None]), codes)
    return c, s


def _device(c, s, codes):
    return c.float().to(codes).view(c.shape[0], -1, 128).cuda().contiguous(), s.float().cuda()


def _append_both(olds, news, H, codes, dtype, seed, *, key=None, layout="own", table_dtype=torch.int64, pad=0, poison=None):
    from jetfire_b200 import ops
    lens = [o + n for o, n in zip(olds, news)]
    max_blocks = max(1, max((l + 15) // 16 for l in lens))
    table, blocks = _tables(lens, max_blocks, seed)
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    T = start[-1] + pad
    g = torch.Generator().manual_seed(seed + 1)
    sides, tensors = [], []
    for side in range(2):
        x = torch.randn(T, H, 128, generator=g) * torch.exp(torch.randn(1, H, 128, generator=g)) if key is None else key[side]
        x = x.to(dtype)
        if poison is not None:
            x = poison(x, side)
        c, s = _cache(H, blocks, codes, seed + 2 + side)
        dev = x.cuda()
        if layout == "qkv":      # a view into a wider tensor
            wide = torch.zeros(T, 2 * H + 3, 128, dtype=dtype, device="cuda")
            wide[:, H + 1:2 * H + 1] = dev
            dev = wide[:, H + 1:2 * H + 1]
        elif layout == "odd":    # rows that are not 16-byte aligned
            wide = torch.zeros(T, H, 131, dtype=dtype, device="cuda")
            wide[:, :, 1:129] = dev
            dev = wide[:, :, 1:129]
        elif layout == "heads":  # (H, T, 128) memory order
            dev = dev.transpose(0, 1).contiguous().transpose(0, 1)
        d, ds = _device(c, s, codes)
        sides.append((x, c, s))
        tensors.append((dev, d, ds))
    start_t, lens_t = torch.tensor(start, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    ops.block8_append(tensors[0][0], tensors[1][0], start_t.cuda(), lens_t.cuda(), table.to(table_dtype).cuda(), tensors[0][1],
                      tensors[0][2], tensors[1][1], tensors[1][2])
    torch.cuda.synchronize()
    for (x, c, s), (_, d, ds) in zip(sides, tensors):
        R.append(x, start, lens, table, c, s, codes)
        assert torch.equal(ds.cpu().double(), s)
        assert torch.equal(_values(d, blocks), c)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("olds, news", [
    ([0], [1]), ([5], [1]), ([15], [1]), ([16], [1]), ([0], [16]), ([3], [13]), ([3], [14]), ([0], [700]), ([7], [333]),
    ([1, 0, 30, 31, 32, 33], [1, 1, 1, 1, 1, 1]), ([0, 9, 16, 250], [0, 40, 0, 3]), ([2, 5, 8], [17, 1, 64]),
])
def test_append_is_the_definition_bit_for_bit(codes, dtype, olds, news):
    _append_both(olds, news, 3, CODES[codes], dtype, 11)


@pytest.mark.parametrize("layout", ["qkv", "odd", "heads"])
@pytest.mark.parametrize("codes", CODES)
def test_append_of_strided_rows(layout, codes):
    _append_both([4, 0, 31], [20, 5, 1], 2, CODES[codes], torch.bfloat16, 12, layout=layout, table_dtype=torch.int32)


@pytest.mark.parametrize("codes", CODES)
def test_append_many_sequences(codes):
    _append_both([i % 40 for i in range(97)], [(i * 7) % 5 for i in range(97)], 1, CODES[codes], torch.bfloat16, 13)
    _append_both([i for i in range(300)], [1] * 300, 2, CODES[codes], torch.float16, 14, pad=9)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_of_extreme_values(codes, dtype):
    """Zeros, the smallest and largest numbers, infinities and NaN, rows in front that were never written."""
    def poison(x, side):
        x = x.clone()
        x[0:16] = 0
        x[16:32] = torch.finfo(dtype).tiny * 2.0 ** -5
        x[32] = torch.finfo(dtype).max
        x[48, 0, 3], x[49, 1, 5], x[50, 0, 7] = float("inf"), float("-inf"), float("nan")
        x[64:80, 1] = float("nan")
        x[80:96, 0] = float("inf")
        return x
    _append_both([0], [100], 2, CODES[codes], dtype, 15, poison=poison)


def test_append_leaves_the_rest_alone_and_skips_bad_blocks():
    from jetfire_b200 import ops
    H, blocks = 2, 4
    for codes in CODES.values():
        key = torch.randn(40, H, 128, device="cuda", dtype=torch.bfloat16)
        d, v = (torch.full((H, blocks * 16, 128), 3, dtype=torch.int8, device="cuda").view(codes) for _ in range(2))
        ks, vs = (torch.full((H, blocks), 7.5, device="cuda") for _ in range(2))
        start = torch.tensor([0, 20, 36], dtype=torch.int32, device="cuda")
        lens = torch.tensor([20, 10, ], dtype=torch.int32, device="cuda")        # the second: 6 positions below 0
        table = torch.tensor([[1, 99], [-1, 2]], dtype=torch.int64, device="cuda")
        ops.block8_append(key, key, start, lens, table, d, ks, v, vs)
        for data, scales in ((d, ks), (v, vs)):
            raw = data.view(torch.int8).view(H, blocks, 16, 128)
            for blk in (0, 2, 3):
                assert (raw[:, blk] == 3).all() and (scales[:, blk] == 7.5).all()
            assert (scales[:, 1] != 7.5).all() and (raw[:, 1] != 3).any()


def test_append_nothing():
    from jetfire_b200 import ops
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")
    d, s = z(2, 32, 128, dtype=torch.int8), torch.ones(2, 2, device="cuda")
    ops.block8_append(z(0, 2, 128, dtype=torch.bfloat16), z(0, 2, 128, dtype=torch.bfloat16), z(1), z(0), z(0, 4, dtype=torch.int64),
                      d, s, d.clone(), s.clone())
    ops.block8_append(z(3, 2, 128, dtype=torch.bfloat16), z(3, 2, 128, dtype=torch.bfloat16), z(3), z(2), z(2, 4, dtype=torch.int64),
                      d, s, d.clone(), s.clone())
    assert (s == 1).all() and (d == 0).all()


# ---- decode ------------------------------------------------------------------------------


class Decode:
    def __init__(self, lens, H_q, H_kv, codes, dtype, seed, *, softcap=0.0, alibi=False, window=None, prefix=None, table_dtype=torch.int64,
                 q_scale=1.0, v_spread=0.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H_q, self.H_kv, self.codes, self.dtype = lens, H_q, H_kv, codes, dtype
        self.max_S = max(1, max(lens))
        self.table, self.blocks = _tables(lens, (self.max_S + 15) // 16, seed)
        self.table_dtype = table_dtype
        self.k, self.ks = _cache(H_kv, self.blocks, codes, seed + 1)
        self.v, self.vs = _cache(H_kv, self.blocks, codes, seed + 2)
        if v_spread:
            self.vs = R.fl32(self.vs * torch.exp2(v_spread * torch.randn(self.vs.shape, generator=g)).double())
        self.q = (torch.randn(len(lens), H_q, 128, generator=g) * q_scale).to(dtype)
        self.scale = 128 ** -0.5 / q_scale
        self.kw = dict(softcap=softcap, window=window)
        self.slopes = torch.tensor([2.0 ** (-8 * (h + 1) / H_q) for h in range(H_q)]) if alibi else None
        self.prefix = prefix

    def expected(self):
        out = torch.zeros(len(self.lens), self.H_q, 128, dtype=torch.float64)
        lse = torch.full((len(self.lens), self.H_q), float("-inf"), dtype=torch.float64)
        k, v = self.k * self.ks[..., None, None], self.v * self.vs[..., None, None]
        for b, n in enumerate(self.lens):
            ids = self.table[b, :(n + 15) // 16]
            j = torch.arange(n)
            ok = (ids >= 0) & (ids < self.blocks)
            j = j[ok[j // 16]]
            if not len(j):
                continue
            kb, vb = (x[:, ids.clamp(0, self.blocks - 1)].reshape(self.H_kv, -1, 128)[:, j] for x in (k, v))
            o, l = R.attend(self.q[b].double()[:, None], kb, vb, torch.tensor([n - 1]), j, self.scale, prefix=(self.prefix[b] if self.prefix else 0),
                            slopes=self.slopes, **self.kw)
            out[b], lse[b] = o[:, 0], l[:, 0]
        return out, lse

    def device(self):
        kd, ks = _device(self.k, self.ks, self.codes)
        vd, vs = _device(self.v, self.vs, self.codes)
        return (self.q.cuda(), kd, ks, vd, vs, self.table.to(self.table_dtype).cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(),
                self.max_S, self.H_q, self.H_kv, 16, self.scale)

    def options(self):
        return dict(alibi_slopes=self.slopes.cuda() if self.slopes is not None else None,
                    prefix_lens=torch.tensor(self.prefix, dtype=torch.int32).cuda() if self.prefix else None, **self.kw)

    def check(self, out, lse):
        want, want_lse = self.expected()
        vmax = (self.v.abs() * self.vs[..., None, None]).amax().item()
        tol = (2 ** -11 + 2 ** -14) * vmax + torch.finfo(self.dtype).eps / 2 * want.abs() + torch.finfo(self.dtype).tiny
        err = (out.double().cpu() - want).abs()
        assert (err <= tol).all(), f"out: {(err / tol).max():.3g} of the tolerance"
        none = torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse.cpu()), none)
        assert ((lse.double().cpu() - want_lse).abs()[~none] <= 2 ** -14 + 2 ** -22 * want_lse.abs()[~none]).all()

    def run(self, **kw):
        from jetfire_b200 import ops
        return ops.block8_decode_attn(*self.device(), **self.options(), **kw)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [100], [0, 1, 0], [127, 128, 129], [500], [1000, 3, 0, 257], [2049], [20000]])
def test_decode_lengths(codes, lens):
    c = Decode(lens, 8, 2, CODES[codes], torch.bfloat16, 21)
    c.check(*c.run())


@pytest.mark.parametrize("H_q, H_kv", [(1, 1), (3, 1), (8, 8), (32, 8), (64, 8), (9, 1), (32, 2), (16, 1), (40, 1), (24, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_head_layouts(H_q, H_kv, dtype):
    for codes in CODES.values():
        c = Decode([333, 40], H_q, H_kv, codes, dtype, 22, table_dtype=torch.int32)
        c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("options", [
    dict(softcap=5.0), dict(softcap=0.5), dict(softcap=1000.0), dict(alibi=True), dict(window=1), dict(window=16), dict(window=100),
    dict(window=5000), dict(window=100, prefix=[7, 64, 1000, 1]), dict(window=33, prefix=[0, 16, 200, 1], alibi=True, softcap=20.0),
    dict(prefix=[5, 5, 5, 1])])
def test_decode_masks_and_biases(codes, options):
    c = Decode([700, 650, 300, 1], 12, 4, CODES[codes], torch.bfloat16, 23, **options)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
def test_decode_many_sequences(codes):
    c = Decode([(i * 37) % 400 for i in range(70)], 8, 4, CODES[codes], torch.float16, 24)
    c.check(*c.run())
    c = Decode([5000] + [3] * 20, 8, 8, CODES[codes], torch.bfloat16, 25)
    c.check(*c.run())


@pytest.mark.parametrize("B, H_q, H_kv, longest", [(1, 8, 8, 60), (1, 8, 8, 130), (1, 16, 8, 500), (1, 16, 8, 1030), (2, 8, 1, 900), (9, 8, 8, 700),
                                                  (40, 8, 8, 300), (3, 32, 2, 2000), (70, 4, 4, 700)])
def test_decode_clusters_of_every_size(B, H_q, H_kv, longest):
    """Short sequences are shared by the blocks of a cluster: one, two, four or eight of them, also more than there are blocks of
    positions."""
    for codes in CODES.values():
        c = Decode([longest] + [(i * 97) % (longest + 1) for i in range(1, B)], H_q, H_kv, codes, torch.bfloat16, 39, softcap=8.0 if B == 2 else 0.0)
        c.check(*c.run())


@pytest.mark.parametrize("q_scale", [1e-30, 1e-5, 1e4, 1e30])
def test_decode_queries_of_any_size(q_scale):
    """bf16 queries far outside fp16's range go through a power of two."""
    c = Decode([300], 8, 2, torch.int8, torch.bfloat16, 26, q_scale=q_scale)
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lens", [[40], [3000]])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_decode_queries_that_are_no_numbers(codes, lens, value):
    """One element of one head: that head's row is NaN, the others are as ever."""
    c = Decode(lens, 8, 2, CODES[codes], torch.bfloat16, 35)
    c.q[0, 3, 77] = value
    out, lse = c.run()
    assert torch.isnan(out[0, 3]).all() and torch.isnan(lse[0, 3])
    c.q[0, 3, 77] = 0.0
    want, want_lse = c.expected()
    out[0, 3], lse[0, 3] = want[0, 3].to(out.dtype).cuda(), want_lse[0, 3].float().cuda()
    c.check(out, lse)


@pytest.mark.parametrize("codes", CODES)
def test_decode_block_scales_far_apart(codes):
    c = Decode([900, 64], 8, 2, CODES[codes], torch.bfloat16, 27, v_spread=6.0)
    c.check(*c.run())


def test_decode_many_small_weights_add_up():
    """One position takes the maximum, 20000 others 2^-20 of its weight each: together they are a part of the sum that an
    fp16 weight relative to the maximum alone would lose."""
    n = 20001
    c = Decode([n], 8, 1, torch.int8, torch.float16, 28)
    c.k.zero_()
    c.v.fill_(100.0)
    c.ks.fill_(1.0)
    c.vs.fill_(1.0)
    c.q.zero_()
    c.q[:, :, 0] = 1.0
    c.scale = 0.1
    c.k[0, c.table[0, 3], 5, 0] = 100.0
    c.k[0, :, :, 0] -= 39.0                     # 13.9 below: e^-13.9 = 2^-20
    c.k[0, c.table[0, 3], 5, 0] = 100.0
    c.v[0, c.table[0, 3], 5] = -100.0
    c.check(*c.run())


def test_decode_skips_blocks_that_are_none():
    c = Decode([200, 40, 16], 8, 2, torch.int8, torch.bfloat16, 29)
    c.table[0, 3], c.table[0, 12], c.table[1, 0], c.table[2, 0] = -1, 10 ** 12, c.blocks, -5
    c.check(*c.run())


@pytest.mark.parametrize("codes", CODES)
def test_rows_behind_the_end_do_not_count(codes):
    """Whatever the unwritten rows of a last block hold, and scales of blocks outside a window."""
    from jetfire_b200 import ops
    c = Decode([37, 210], 8, 2, CODES[codes], torch.bfloat16, 30, window=50)
    a = list(c.device())
    for data in (a[1], a[3]):
        rows = data.view(torch.int8).view(2, c.blocks, 16, 128)
        rows[:, c.table[0, 2], 5:] = 0x7F
        rows[:, c.table[1, 13], 2:] = -1
    for s in (a[2], a[4]):
        s[:, c.table[1, 0]] = float("nan")
        s[:, c.table[1, 5]] = float("inf")
    c.check(*ops.block8_decode_attn(*a, **c.options()))


def test_decode_lengths_are_cut_to_max_S_and_the_table():
    from jetfire_b200 import ops
    c = Decode([100, 64], 8, 2, torch.int8, torch.bfloat16, 31)
    a = list(c.device())
    a[6] = torch.tensor([10 ** 9, 64], dtype=torch.int32).cuda()
    c.check(*ops.block8_decode_attn(*a[:7], 100, *a[8:]))
    a[6] = torch.tensor([100, -3], dtype=torch.int32).cuda()
    out, lse = ops.block8_decode_attn(*a)
    assert (out[1] == 0).all() and (lse[1] == float("-inf")).all()


def test_append_then_decode_in_a_graph_on_another_stream():
    """The two as a decode loop uses them: captured once, replayed with other inputs; repeats give the same bits."""
    from jetfire_b200 import ops
    H, lens0 = 2, [30, 5, 64]
    c = Decode([l + 4 for l in lens0], 8, H, torch.int8, torch.bfloat16, 32)
    q, kd, ks, vd, vs, table, _, max_S, *rest = c.device()
    lens = torch.tensor(lens0, dtype=torch.int32).cuda()
    start = torch.arange(4, dtype=torch.int32).cuda()
    key, value = torch.zeros(3, H, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, H, 128, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        lens.add_(1)
        ops.block8_append(key, value, start, lens, table, kd, ks, vd, vs)
        return ops.block8_decode_attn(q, kd, ks, vd, vs, table, lens, max_S, *rest)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step()
        lens.sub_(1)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out, lse = step()
        R_lens = list(lens0)
        for i in range(3):
            g = torch.Generator().manual_seed(100 + i)
            kt, vt = (torch.randn(3, H, 128, generator=g).to(torch.bfloat16) * (1 + 3 * i) for _ in range(2))
            key.copy_(kt)
            value.copy_(vt)
            if i == 0:     # the warm-up's rows of zeros went there: blocks and scales as they are now
                c.k, c.v = _values(kd, c.blocks), _values(vd, c.blocks)
                c.ks, c.vs = ks.cpu().double(), vs.cpu().double()
            graph.replay()
            stream.synchronize()
            R_lens = [l + 1 for l in R_lens]
            for x, code, scale in ((kt, c.k, c.ks), (vt, c.v, c.vs)):
                R.append(x, [0, 1, 2, 3], R_lens, c.table, code, scale, torch.int8)
            c.lens = R_lens
            assert torch.equal(_values(kd, c.blocks), c.k) and torch.equal(vs.cpu().double(), c.vs)
            c.check(out, lse)
            again = ops.block8_decode_attn(q, kd, ks, vd, vs, table, lens, max_S, *rest)
            assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_decode_caller_owned_output_and_workspace():
    from jetfire_b200 import ops
    c = Decode([1500, 700], 8, 2, torch.float8_e4m3fn, torch.float16, 33)
    out = torch.full((2, 8, 128), 9.0, dtype=torch.float16, device="cuda")
    ws = torch.empty(ops.block8_workspace_bytes(2, 8, 2, c.max_S) + 256, dtype=torch.uint8, device="cuda")
    got, lse = c.run(out=out, workspace=ws)
    assert got.data_ptr() == out.data_ptr()
    c.check(out, lse)


def test_cache_larger_than_32_bits():
    """Blocks whose bytes lie past 2^32 of the cache."""
    from jetfire_b200 import ops
    blocks = (1 << 32) // (16 * 128) // 2 + 40
    kd, vd = (torch.zeros(2, blocks * 16, 128, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(2, blocks, device="cuda") for _ in range(2))
    table = torch.tensor([[blocks - 1, blocks - 7, 3]], device="cuda")
    key, value = (torch.randn(40, 2, 128, device="cuda").bfloat16() for _ in range(2))
    start, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 40], [40]))
    ops.block8_append(key, value, start, lens, table, kd, ks, vd, vs)
    c = Decode([40], 4, 2, torch.int8, torch.bfloat16, 34)
    ids = table[0].cpu()
    pick = lambda d: d.view(2, blocks, 16, 128)[:, table[0]].cpu().double()
    c.k, c.v, c.ks, c.vs = pick(kd), pick(vd), ks[:, table[0]].cpu().double(), vs[:, table[0]].cpu().double()
    kk, ss = torch.zeros(2, 3, 16, 128, dtype=torch.float64), torch.ones(2, 3, dtype=torch.float64)
    R.append(key.cpu(), [0, 40], [40], torch.tensor([[0, 1, 2]]), kk, ss, torch.int8)
    assert torch.equal(kk[:, :, :8], c.k[:, :, :8]) and torch.equal(ss, c.ks)
    c.table, c.blocks = torch.tensor([[0, 1, 2]]), 3
    c.check(*ops.block8_decode_attn(c.q.cuda(), kd, ks, vd, vs, table, lens, 48, 4, 2, 16, c.scale))


def test_two_calls_at_once_on_two_streams():
    cases = [Decode([3000, 17, 900], 8, 2, torch.int8, torch.bfloat16, 36), Decode([20000], 16, 1, torch.float8_e4m3fn, torch.float16, 37, softcap=5.0)]
    from jetfire_b200 import ops
    args, options = [c.device() for c in cases], [c.options() for c in cases]
    want = [ops.block8_decode_attn(*a, **o) for a, o in zip(args, options)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.block8_decode_attn(*args[i], **options[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
        cases[i].check(*want[i])


@pytest.mark.parametrize("options", [dict(softcap=1e-20), dict(softcap=1e-4), dict(softcap=1e20), dict(softcap=3.0, alibi=True)])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0])
def test_decode_scales_and_caps_of_any_size(options, scale):
    for codes in CODES.values():
        c = Decode([500, 30], 8, 2, codes, torch.bfloat16, 38, **options)
        c.scale = scale
        c.q = (c.q.float() * 0.5).to(c.q.dtype)
        c.check(*c.run())
