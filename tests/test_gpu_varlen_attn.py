"""Attention of packed prompts against the definition in 64 bits.

Tolerances.  Weights are rounded to q's type before they meet V: off by at most eps / 2 of themselves, so the output by
eps / 2 * sum p|v| / sum p <= eps / 2 * max|v|; scores are sums of 128 products in fp32, |s| <= 60 here, so their
error moves a weight by less than 2^-13 (2^-23 * 128 * |q||k| scale / 2 and 2^-22 * |s| together), 2^-13 * max|v| of the output.
The result is rounded once more: eps / 2 of its value.  lse: 2^-13 + 2^-21 * |lse|."""
import pytest
import torch

import block8_ref as R

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, lens, H_q, H_kv, dtype, seed, *, causal=True, window=None, softcap=0.0, alibi=False, prefix=None, layout="own", pad=0,
                 front=0, scale=128 ** -0.5, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.dtype, self.front = lens, dtype, front
        T = front + sum(lens) + pad
        self.q = (torch.randn(T, H_q, 128, generator=g) * spread).to(dtype)
        self.k = (torch.randn(T, H_kv, 128, generator=g) * torch.exp(0.5 * torch.randn(1, H_kv, 128, generator=g))).to(dtype)
        self.v = torch.randn(T, H_kv, 128, generator=g).to(dtype)
        self.scale, self.layout = scale, layout
        self.kw = dict(causal=causal, window=window, softcap=softcap)
        self.slopes = torch.tensor([2.0 ** (-8 * (h + 1) / H_q) for h in range(H_q)]) if alibi else None
        self.prefix = prefix

    def start(self):
        s = [self.front]
        for n in self.lens:
            s.append(s[-1] + n)
        return s

    def device(self):
        ts = [t.cuda() for t in (self.q, self.k, self.v)]
        if self.layout == "qkv":
            both = torch.cat(ts, 1)
            a, b = self.q.shape[1], self.k.shape[1]
            ts = [both[:, :a], both[:, a:a + b], both[:, a + b:]]
        elif self.layout == "heads":
            ts = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in ts]
        elif self.layout == "odd":
            wide = [torch.zeros(*t.shape[:2], 131, dtype=t.dtype, device="cuda") for t in ts]
            for w, t in zip(wide, ts):
                w[..., 3:] = t
            ts = [w[..., 3:] for w in wide]
        return (*ts, torch.tensor(self.start(), dtype=torch.int32).cuda(), self.scale)

    def run(self, **kw):
        from jetfire_b200 import ops
        return ops.varlen_prefill_attn(*self.device(), alibi_slopes=self.slopes.cuda() if self.slopes is not None else None,
                                       prefix_lens=torch.tensor(self.prefix, dtype=torch.int32).cuda() if self.prefix else None, **self.kw, **kw)

    def check(self, out, lse, skip=()):
        out, lse, eps = out.cpu().double(), lse.cpu().double(), torch.finfo(self.dtype).eps
        for b, (lo, n) in enumerate(zip(self.start(), self.lens)):
            if n == 0 or b in skip:
                continue
            dev = "cuda" if n > 600 else "cpu"
            q, k, v = (t[lo:lo + n].to(dev).double().transpose(0, 1) for t in (self.q, self.k, self.v))
            i = torch.arange(n, device=dev)
            want, want_lse = R.attend(q, k, v, i, i, self.scale, prefix=self.prefix[b] if self.prefix else 0,
                                      slopes=self.slopes.to(dev) if self.slopes is not None else None, **self.kw)
            want, want_lse = want.transpose(0, 1).cpu(), want_lse.t().cpu()
            got, fin = out[lo:lo + n], torch.isfinite(want)
            assert torch.equal(torch.isfinite(got), fin)
            assert torch.equal(got[~fin].nan_to_num(7.0), want[~fin].nan_to_num(7.0))
            vmax = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax().item()
            tol = (eps / 2 + 2 ** -13) * vmax + eps / 2 * want.abs()
            err = (got - want).abs()
            worst = (err / tol)[fin].max().item() if fin.any() else 0.0
            assert worst <= 1.0, f"sequence {b}: {worst:.3g} of the tolerance at {(err / tol).nan_to_num(0).argmax().item()}"
            ok = torch.isfinite(want_lse)
            assert ((lse[lo:lo + n] - want_lse).abs()[ok] <= 2 ** -13 + 2 ** -21 * want_lse[ok].abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[1], [16], [127], [128], [129], [255], [256], [257], [384], [700], [5, 64, 129], [0, 3, 0, 0, 400, 1, 0], [1] * 40, [2100]])
def test_lengths(dtype, lens):
    for causal in (True, False):
        c = Case(lens, 2, 1, dtype, 41, causal=causal)
        c.check(*c.run())


@pytest.mark.parametrize("H_q, H_kv", [(1, 1), (8, 8), (32, 8), (9, 3), (16, 1), (40, 2)])
def test_head_layouts(H_q, H_kv):
    c = Case([200, 77], H_q, H_kv, torch.bfloat16, 42)
    c.check(*c.run())


OPTIONS = [dict(window=1), dict(window=2), dict(window=64), dict(window=128), dict(window=129), dict(window=300), dict(window=5000),
           dict(softcap=2.0), dict(softcap=30.0), dict(softcap=1000.0), dict(alibi=True), dict(prefix=[100, 0, 1]), dict(prefix=[600, 129, 50]),
           dict(prefix=[300, 5, 1000], window=40), dict(prefix=[513, 128, 7], window=200, alibi=True, softcap=20.0)]


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_masks_and_biases(options, causal, dtype):
    c = Case([900, 333, 50], 4, 2, dtype, 43, causal=causal, **options)
    c.check(*c.run())


@pytest.mark.parametrize("layout", ["qkv", "heads", "odd"])
def test_strided_inputs(layout):
    c = Case([300, 20], 4, 2, torch.bfloat16, 44, layout=layout)
    c.check(*c.run())


@pytest.mark.parametrize("softcap", [0.0, 3.0, 0.01])
@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales(scale, softcap, alibi):
    c = Case([400], 2, 1, torch.float16, 45, scale=scale, spread=0.5, softcap=softcap, alibi=alibi)
    c.check(*c.run())


@pytest.mark.parametrize("scale", [128 ** -0.5, -(128 ** -0.5)])
@pytest.mark.parametrize("softcap", [4.0, 6.0, 9.0, 14.0, 40.0])
def test_caps_about_the_scores_size(softcap, scale):
    """Largest scores from a seventh of the cap to beyond it: tiles of every branch of the cap's arithmetic.  (Its relative error of
    6.7e-7 moves a score of at most 40 by less than 2^-15.)"""
    for dtype in (torch.bfloat16, torch.float16):
        c = Case([700], 2, 1, dtype, 53, softcap=softcap, scale=scale)
        c.check(*c.run())


@pytest.mark.parametrize("softcap", [1e-20, 1e-4, 1e20])
def test_caps_of_any_size(softcap):
    c = Case([300], 2, 1, torch.bfloat16, 52, softcap=softcap)
    c.check(*c.run())


def test_many_sequences_of_one_step():
    c = Case([(i * 53) % 300 for i in range(75)], 4, 2, torch.bfloat16, 46)
    c.check(*c.run())
    c = Case([3000] + [7] * 40 + [1100], 2, 1, torch.float16, 47, window=700)
    c.check(*c.run())


def test_references_that_move():
    """Keys whose scores grow along the row: the running reference moves at every tile."""
    c = Case([1500], 2, 1, torch.bfloat16, 48, causal=False)
    c.k = (c.k.float() * torch.linspace(0.02, 3.0, 1500)[:, None, None]).to(c.dtype)
    c.check(*c.run())


@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("options", [dict(), dict(window=100), dict(prefix=[0, 200, 0], window=50), dict(causal=False)])
def test_what_a_row_does_not_see_has_no_influence(value, options):
    """Infinities and NaN in keys and values of neighbours, of later positions, of positions outside a window."""
    c = Case([300, 500, 40], 2, 1, torch.bfloat16, 49, pad=60, front=10, **options)
    for t in (c.k, c.v):
        t[:10], t[-60:] = value, value             # rows of no sequence
    c.q[:10], c.q[-60:] = value, value
    c.v[310 + 333, 0, 5] = value                   # rows of the second sequence that see position 333 get it, the others do not
    c.v[310 + 450, 0, 77] = value
    out = torch.full((c.q.shape[0], 2, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    got, lse = c.run(out=out)
    assert got.data_ptr() == out.data_ptr()
    c.check(got, lse)
    assert (out[:10] == 5).all() and (out[-60:] == 5).all()


@pytest.mark.parametrize("shift", [8, 16, 24])
def test_an_output_on_any_multiple_of_16_bytes(shift):
    c = Case([130, 33], 4, 2, torch.bfloat16, 51)
    T, H, _ = c.q.shape
    whole = torch.full((T * H * 128 + 32,), 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = c.run(out=whole[shift:shift + T * H * 128].view(T, H, 128))
    c.check(out, lse)
    assert (whole[:shift] == 7.0).all() and (whole[shift + T * H * 128:] == 7.0).all()


def test_keys_that_are_no_numbers_reach_only_who_sees_them():
    c = Case([400], 2, 1, torch.float16, 50)
    c.k[250] = float("nan")
    out, lse = c.run()
    assert torch.isnan(out[250:]).all() and torch.isfinite(out[:250]).all()
    c.lens = [250]
    c.check(out[:250], lse[:250])


def test_nothing_to_do():
    from jetfire_b200 import ops
    z = lambda T: torch.zeros(T, 2, 128, dtype=torch.bfloat16, device="cuda")
    out, lse = ops.varlen_prefill_attn(z(0), z(0), z(0), torch.zeros(1, dtype=torch.int32, device="cuda"), 0.1)
    assert out.shape == (0, 2, 128) and lse.shape == (0, 2)
    own = torch.full((5, 2, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.varlen_prefill_attn(z(5), z(5), z(5), torch.zeros(4, dtype=torch.int32, device="cuda"), 0.1, out=own)
    assert (own == 3).all()


def test_captured_and_replayed_on_another_stream_with_the_same_bits():
    from jetfire_b200 import ops
    c = Case([500, 129, 64], 8, 2, torch.bfloat16, 51, window=300)
    a = c.device()
    record = torch.zeros(2, dtype=torch.int64, device="cuda")
    want = ops.varlen_prefill_attn(*a, window=300)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            out, lse = ops.varlen_prefill_attn(*a, window=300, status_record=record)
        for _ in range(3):
            out.zero_()
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    ops.decode_status_of_copy(record.cpu())
    c.check(out, lse)


def test_two_calls_at_once_on_two_streams():
    from jetfire_b200 import ops
    cases = [Case([900, 333], 8, 2, torch.bfloat16, 53), Case([1500], 4, 1, torch.bfloat16, 54, window=200, softcap=10.0)]
    args = [c.device() for c in cases]
    kw = [dict(), dict(window=200, softcap=10.0)]
    want = [ops.varlen_prefill_attn(*a, **k) for a, k in zip(args, kw)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.varlen_prefill_attn(*args[i], **kw[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
        cases[i].check(*want[i])
