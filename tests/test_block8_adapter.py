"""Layers with an 8-bit cache behind the attention backend: routing on CPU with the ops replaced by their plain forms, and
whole steps on the GPU -- prompts, decode tokens, both together -- against the definition in 64 bits."""
from types import SimpleNamespace

import pytest
import torch

import block8_ref as R
from jetfire_b200.adapter import block8 as B8
from jetfire_b200.adapter import config as jcfg
from jetfire_b200.adapter import jetfire_backend as jb

H_Q, H_KV, D = 4, 2, 128


def _impl(**kw):
    return SimpleNamespace(scale=D ** -0.5, sliding_window=(-1, -1), alibi_slopes=None, logits_soft_cap=0, attn_type="decoder", **kw)


def _layer(name="l"):
    return SimpleNamespace(num_heads=H_Q, num_kv_heads=H_KV, head_size=D, layer_name=name)


def _meta(olds, news, table, device, **kw):
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    lens = [o + n for o, n in zip(olds, news)]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    return SimpleNamespace(num_actual_tokens=start[-1], max_query_len=max(news), max_seq_len=max(lens), query_start_loc=t(start), seq_lens=t(lens),
                           block_table=table.to(device), use_cascade=False, causal=True, **kw)


def _plain_ops(monkeypatch, calls):
    """The three ops as plain torch on the CPU, recorded."""
    def append(key, value, start, lens, table, kd, ks, vd, vs):
        calls.append(("append", key.shape[0]))
        for x, d, s in ((key, kd, ks), (value, vd, vs)):
            c, sc = d.double().view(H_KV, -1, 16, D), s.double()
            R.append(x, start, lens, table, c, sc, torch.int8)
            d.copy_(c.view(H_KV, -1, D).to(torch.int8))
            s.copy_(sc.float())

    def decode(q, kd, ks, vd, vs, table, lens, max_S, H_q, H_kv, block_size, scale, *, softcap=0.0, alibi_slopes=None, window=None, **_):
        calls.append(("decode", q.shape[0], int(max_S), window, softcap))
        k, v = (d.double().view(H_KV, -1, 16, D) * s.double()[..., None, None] for d, s in ((kd, ks), (vd, vs)))
        out = torch.zeros_like(q)
        for b in range(q.shape[0]):
            n = int(lens[b])
            ids = table[b, :(n + 15) // 16].long()
            o, _ = R.attend(q[b].double()[:, None], k[:, ids].reshape(H_KV, -1, D)[:, :n], v[:, ids].reshape(H_KV, -1, D)[:, :n],
                            torch.tensor([n - 1]), torch.arange(n), scale, window=window, softcap=softcap, slopes=alibi_slopes)
            out[b] = o[:, 0].to(q.dtype)
        return out, None

    def prefill(q, k, v, cu, scale, *, causal=True, window=None, softcap=0.0, alibi_slopes=None, out=None, **_):
        calls.append(("prefill", q.shape[0], len(cu) - 1, window, softcap))
        got = torch.empty_like(q) if out is None else out
        for lo, hi in zip(cu[:-1].tolist(), cu[1:].tolist()):
            i = torch.arange(hi - lo)
            o, _ = R.attend(*(x[lo:hi].double().transpose(0, 1) for x in (q, k, v)), i, i, scale, causal=causal, window=window, softcap=softcap,
                            slopes=alibi_slopes)
            got[lo:hi] = o.transpose(0, 1).to(q.dtype)
        return got, None

    monkeypatch.setattr(B8.ops, "block8_append", append)
    monkeypatch.setattr(B8.ops, "block8_decode_attn", decode)
    monkeypatch.setattr(B8.ops, "varlen_prefill_attn", prefill)


class Conversation:
    """Sequences that grow step by step; the oracle keeps their quantised cache."""

    def __init__(self, n, device, codes=torch.int8, max_blocks=40, seed=0, **impl):
        self.n, self.device, self.codes = n, device, codes
        self.gen = torch.Generator().manual_seed(seed)
        self.table = torch.randperm(n * max_blocks, generator=self.gen).view(n, max_blocks).to(torch.int32)
        self.lens = [0] * n
        self.store = B8.JetFireBlock8Store(num_blocks=n * max_blocks, num_kv_heads=H_KV, codes="int8" if codes == torch.int8 else "e4m3", device=device)
        self.impl = _impl()
        for k, v in impl.items():
            setattr(self.impl, k, v)
        z = lambda *s: torch.zeros(*s, dtype=torch.float64)
        self.side = [(z(H_KV, n * max_blocks, 16, D), z(H_KV, n * max_blocks)) for _ in range(2)]

    def step(self, news, flat=True, call=None, **meta):
        olds = list(self.lens)
        T = sum(news)
        q, k, v = (torch.randn(T, h, D, generator=self.gen).to(torch.bfloat16) for h in (H_Q, H_KV, H_KV))
        md = _meta(olds, news, self.table, self.device, **meta)
        out = torch.full((T, H_Q * D) if flat else (T, H_Q, D), 7.0, dtype=torch.bfloat16, device=self.device)
        done = (call or B8.try_block8_attention)(impl=self.impl, layer=_layer(), query=q.to(self.device), key=k.to(self.device), value=v.to(self.device),
                                                 attn_metadata=md, output=out, store=self.store)
        self.lens = [o + n for o, n in zip(olds, news)]
        start = md.query_start_loc.tolist()
        for x, (c, s) in zip((k, v), self.side):
            R.append(x, start, self.lens, self.table, c, s, self.codes)
        if done is None:
            return None
        assert done is out
        win = self.impl.sliding_window[0] + 1 if self.impl.sliding_window[0] >= 0 else None
        kw = dict(window=win, softcap=float(self.impl.logits_soft_cap or 0), slopes=self.impl.alibi_slopes)
        for b in range(self.n):
            if news[b] == 0:
                continue
            rows, n = slice(start[b], start[b + 1]), self.lens[b]
            if news[b] == 1:
                ids = self.table[b, :(n + 15) // 16].long()
                kk, vv = ((c * s[..., None, None])[:, ids].reshape(H_KV, -1, D)[:, :n] for c, s in self.side)
                o, _ = R.attend(q[rows].double().transpose(0, 1), kk, vv, torch.tensor([n - 1]), torch.arange(n), self.impl.scale, **kw)
            else:
                i = torch.arange(n)
                o, _ = R.attend(*(x[rows].double().transpose(0, 1) for x in (q, k, v)), i, i, self.impl.scale, **kw)
            got = out[rows].reshape(-1, H_Q, D).double().cpu()
            want = o.transpose(0, 1)
            # weights rounded to 8 bits (prompts) or 11, the result to 8: half a step of each, of values below 5
            assert ((got - want).abs() <= 2 ** -8 * 5.0 + 2 ** -8 * want.abs()).all()
        return out


STEPS = [[20, 5, 33], [1, 1, 1], [1, 1, 1], [1, 0, 1]]


@pytest.mark.parametrize("flat", [True, False])
def test_prompts_then_tokens(monkeypatch, flat):
    calls = []
    _plain_ops(monkeypatch, calls)
    c = Conversation(3, "cpu")
    for news in STEPS:
        assert c.step(news, flat) is not None
    assert calls[0] == ("append", 58) and calls[1][:3] == ("prefill", 58, 3)
    assert [x[0] for x in calls[2:]] == ["append", "decode"] * 3
    assert calls[3][1:3] == (3, 34)                      # three rows, bounded by the metadata's longest sequence


def test_prompts_and_tokens_in_one_step(monkeypatch):
    calls = []
    _plain_ops(monkeypatch, calls)
    c = Conversation(4, "cpu", seed=1)
    c.step([9, 17, 0, 0])
    calls.clear()
    c.step([1, 1, 8, 30], num_decodes=2, num_prefills=2, num_decode_tokens=2, num_prefill_tokens=38, jetfire_prefill_has_context=False)
    assert [x[0] for x in calls] == ["append", "decode", "prefill"] and calls[1][1] == 2 and calls[2][1:3] == (38, 2)
    calls.clear()
    d = Conversation(4, "cpu", seed=2)
    d.step([4, 0, 6, 0])
    calls.clear()
    d.step([1, 12, 1, 5])                                 # interleaved, without the scheduler's counts
    assert [x[0] for x in calls] == ["append", "decode", "prefill"] and calls[1][1] == 2 and calls[2][1:3] == (17, 2)


def test_the_implementation_s_settings_are_passed_on(monkeypatch):
    calls = []
    _plain_ops(monkeypatch, calls)
    c = Conversation(2, "cpu", seed=3, sliding_window=(11, 0), logits_soft_cap=20.0, alibi_slopes=torch.tensor([0.5, 0.25, 0.125, 0.0625]))
    c.step([40, 18])
    c.step([1, 1])
    assert calls[1][3:] == (12, 20.0) and calls[3][3:] == (12, 20.0)


def test_steps_that_are_handed_back_are_appended(monkeypatch):
    calls = []
    _plain_ops(monkeypatch, calls)
    c = Conversation(2, "cpu", seed=4)
    c.step([10, 10])
    for news, kw in (([5, 1], {}), ([1, 1], dict(cascade=True)), ([1, 1], dict(causal=False))):
        calls.clear()
        call = None
        if kw:
            def call(attn_metadata, **a):
                attn_metadata.use_cascade, attn_metadata.causal = "cascade" in kw, kw.get("causal", True)
                return B8.try_block8_attention(attn_metadata=attn_metadata, **a)
        assert c.step(news, call=call) is None
        assert [x[0] for x in calls] == ["append"]
    assert c.step([1, 1]) is not None                     # and the next step sees them


def test_configuration_and_stores(monkeypatch):
    for raw, want in (("", None), ("off", None), ("int8", "int8"), ("E4M3", "e4m3")):
        monkeypatch.setenv("JETFIRE_BLOCK8", raw)
        jcfg.reset_jetfire_config()
        assert jcfg.get_jetfire_config().block8 == want
    monkeypatch.setenv("JETFIRE_BLOCK8", "int4")
    jcfg.reset_jetfire_config()
    with pytest.raises(ValueError, match="JETFIRE_BLOCK8"):
        jcfg.get_jetfire_config()
    monkeypatch.delenv("JETFIRE_BLOCK8")
    jcfg.reset_jetfire_config()
    from jetfire_b200.adapter.registry import install_layer_stores
    layers = {"a": SimpleNamespace(num_kv_heads=2, head_size=128), "b": SimpleNamespace(num_kv_heads=2, head_size=64)}
    got = install_layer_stores(layers, num_blocks=8, device="cpu", cfg=jcfg.JetFireConfig(block8="e4m3"))
    assert list(got) == ["a"] and isinstance(got["a"], B8.JetFireBlock8Store) and got["a"].k_data.dtype == torch.float8_e4m3fn
    assert got["a"].k_data.shape == (2, 128, 128) and got["a"].k_scales.shape == (2, 8) and jb.get_layer_store("a") is got["a"]
    for bad in (dict(head_dim=64), dict(block_size=32), dict(codes="int4")):
        with pytest.raises(ValueError):
            B8.JetFireBlock8Store(num_blocks=2, num_kv_heads=1, device="cpu", **bad)
    jb._STORES.pop("a")


class _Native:
    """What the mixin falls back to."""
    def forward(self, layer, query, key, value, kv_cache, attn_metadata, output=None, **kw):
        self.native = getattr(self, "native", 0) + 1
        return output

    def do_kv_cache_update(self, layer, key, value, kv_cache, slot_mapping):
        self.updates = getattr(self, "updates", 0) + 1


class _Impl(jb.JetFireAttentionImplMixin, _Native):
    pass


def _through_the_backend(c):
    impl = _Impl()
    for k, v in vars(c.impl).items():
        setattr(impl, k, v)
    jb.register_layer_store("l", c.store)

    def call(impl=impl, layer=None, query=None, key=None, value=None, attn_metadata=None, output=None, store=None):
        impl.do_kv_cache_update(layer, key, value, None, torch.zeros(query.shape[0], dtype=torch.int64))
        return impl.forward(layer, query, key, value, None, attn_metadata, output=output)
    return impl, (lambda **kw: call(**{**kw, "impl": impl}))


def test_the_backend_routes_layers_with_an_8_bit_cache(monkeypatch):
    calls = []
    _plain_ops(monkeypatch, calls)
    c = Conversation(2, "cpu", seed=5)
    impl, call = _through_the_backend(c)
    try:
        c.step([12, 7], call=call)
        c.step([1, 1], call=call)
        assert not hasattr(impl, "native") and impl.updates == 2       # the native cache is kept as well
        assert impl.forward(_layer(), None, None, None, None, None, output="x") == "x" and impl.native == 1     # a profiling run
    finally:
        jb._STORES.pop("l")


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("impl", [dict(), dict(sliding_window=(30, 0), logits_soft_cap=15.0, alibi_slopes=torch.tensor([0.5, 0.25, 0.125, 0.0625]))])
def test_a_run_of_steps_on_the_gpu(codes, impl):
    """Prompts, tokens, prompts and tokens together, many tokens: through the backend's own methods."""
    c = Conversation(3, "cuda", codes, seed=6, **impl)
    _, call = _through_the_backend(c)
    try:
        assert c.step([150, 0, 33], call=call) is not None
        assert c.step([1, 64, 1], call=call) is not None
        for _ in range(20):
            assert c.step([1, 1, 1], call=call) is not None
        torch.cuda.synchronize()
        for (d, s), (want, want_s) in zip(((c.store.k_data, c.store.k_scales), (c.store.v_data, c.store.v_scales)), c.side):
            assert torch.equal(s.cpu().double(), want_s) and torch.equal(d.cpu().float().double().view(want.shape), want)
    finally:
        jb._STORES.pop("l")


@pytest.mark.gpu
def test_a_captured_decode_step_is_replayed_with_longer_sequences():
    c = Conversation(2, "cuda", seed=7)
    c.step([30, 14])
    z = lambda h: torch.zeros(2, h, D, dtype=torch.bfloat16, device="cuda")
    q, k, v, out = z(H_Q), z(H_KV), z(H_KV), z(H_Q)
    md = _meta([30, 14], [1, 1], c.table, "cuda")
    kept = [t.clone() for t in (c.store.k_data, c.store.v_data, c.store.k_scales, c.store.v_scales)]
    args = dict(impl=c.impl, layer=_layer(), query=q, key=k, value=v, attn_metadata=md, output=out, store=c.store)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        B8.try_block8_attention(**args)
        stream.synchronize()
        for t, was in zip((c.store.k_data, c.store.v_data, c.store.k_scales, c.store.v_scales), kept):
            t.copy_(was)
        with torch.cuda.graph(graph, stream=stream):
            B8.try_block8_attention(**args)

    def replay(query, key, value, attn_metadata, output, **_):
        with torch.cuda.stream(stream):
            for dst, src in ((q, query), (k, key), (v, value), (md.seq_lens, attn_metadata.seq_lens)):
                dst.copy_(src.reshape(dst.shape))
            graph.replay()
            output.copy_(out.reshape(output.shape))
            stream.synchronize()
        return output

    for _ in range(30):                                   # past the lengths of the capture and over block bounds
        assert c.step([1, 1], call=replay) is not None


@pytest.mark.gpu
def test_the_packed_path_s_prompts_can_go_to_the_same_kernel():
    """``native_varlen_prefill`` as the ``prefill_attention`` of a mixed step agrees with the plain attention."""
    from jf_testlib import causal_prefill_attention
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(300, h, D, generator=g).to(torch.bfloat16).cuda() for h in (H_Q, H_KV, H_KV))
    cu = torch.tensor([0, 100, 103, 300], dtype=torch.int32, device="cuda")
    outs = []
    for f in (causal_prefill_attention, B8.native_varlen_prefill):
        wide = torch.zeros(301, H_Q, D, dtype=torch.bfloat16, device="cuda")
        f(q=q, k=k, v=v, out=wide[1:], cu_seqlens=cu, max_seqlen=197, impl=_impl(), layer=_layer(), attn_metadata=SimpleNamespace(causal=True))
        outs.append(wide[1:].float())
    assert ((outs[0] - outs[1]).abs() <= 2 ** -8 * (5.0 + outs[0].abs() * 2)).all()
