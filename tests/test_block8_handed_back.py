"""Layers and steps that the 8-bit path does not serve go to the native attention, or are refused, instead of being served wrongly.
On the CPU, with the ops replaced by their plain forms."""
from types import SimpleNamespace

import pytest
import torch

from jetfire_b200.adapter import block8 as B8
from jetfire_b200.adapter import config as jcfg
from jetfire_b200.adapter import jetfire_backend as jb
from jetfire_b200.adapter.registry import install_layer_stores
from test_block8_adapter import D, H_KV, H_Q, Conversation, _impl, _layer, _meta, _plain_ops, _through_the_backend

NOT_SERVED = [dict(sinks=torch.zeros(H_Q)), dict(kv_sharing_target_layer_name="model.layers.0.attn"), dict(attn_type="encoder"),
              dict(attn_type=SimpleNamespace(name="ENCODER_DECODER"))]


@pytest.mark.parametrize("settings", NOT_SERVED)
def test_layers_with_other_terms_or_another_cache(monkeypatch, settings):
    """A per-head term in the softmax's denominator, a layer that reads another layer's cache, attention that is no decoder's: nothing
    is appended and the native attention runs, for prompts and for tokens."""
    calls = []
    _plain_ops(monkeypatch, calls)
    c = Conversation(2, "cpu", seed=11, **settings)
    impl, call = _through_the_backend(c)
    try:
        for news in ([7, 4], [1, 1]):
            T = sum(news)
            q, k, v = (torch.zeros(T, h * D, dtype=torch.bfloat16) for h in (H_Q, H_KV, H_KV))
            out = torch.full((T, H_Q * D), 7.0, dtype=torch.bfloat16)
            assert call(layer=_layer(), query=q, key=k, value=v, attn_metadata=_meta([0, 0], news, c.table, "cpu"), output=out) is out
            assert (out == 7.0).all()
        assert not calls and impl.native == 2
    finally:
        jb._STORES.pop("l")


@pytest.mark.parametrize("settings", NOT_SERVED)
@pytest.mark.parametrize("on", ["layer", "impl"])
def test_such_layers_get_no_cache(settings, on):
    layer = SimpleNamespace(num_kv_heads=2, head_size=128)
    for k, v in settings.items():
        setattr(layer, k, v)
    if on == "impl":
        layer = SimpleNamespace(num_kv_heads=2, head_size=128, impl=_impl(**{k: v for k, v in settings.items() if k != "attn_type"}))
        layer.impl.attn_type = settings.get("attn_type", "decoder")
    other = SimpleNamespace(num_kv_heads=2, head_size=128, impl=_impl())
    got = install_layer_stores({"x": layer, "y": other}, num_blocks=4, device="cpu", cfg=jcfg.JetFireConfig(block8="int8"))
    assert list(got) == ["y"] and jb.get_layer_store("x") is None
    jb._STORES.pop("y")


def _step(store, layer, impl=None, **kw):
    H_q, H_kv, D = layer.num_heads, layer.num_kv_heads, layer.head_size
    q, k, v = (torch.zeros(3, h * D, dtype=torch.bfloat16) for h in (H_q, H_kv, H_kv))
    md = _meta([0], [3], torch.zeros(1, 2, dtype=torch.int32), "cpu")
    return B8.try_block8_attention(impl=impl or _impl(), layer=layer, query=q, key=k, value=v, attn_metadata=md,
                                   output=torch.zeros(3, H_q * D, dtype=torch.bfloat16), store=store, **kw)


@pytest.mark.parametrize("wrong", [dict(head_size=64), dict(num_kv_heads=4)])
def test_a_layer_that_does_not_fit_its_cache_is_an_error(monkeypatch, wrong):
    """It would stay empty beside a layer that never reads it."""
    calls = []
    _plain_ops(monkeypatch, calls)
    store = B8.JetFireBlock8Store(num_blocks=2, num_kv_heads=H_KV, device="cpu")
    layer = SimpleNamespace(**{**vars(_layer()), **wrong})
    with pytest.raises(ValueError, match="8-bit cache"):
        _step(store, layer)
    assert not calls


def test_an_output_that_is_to_be_quantised_goes_to_the_native_attention(monkeypatch):
    """It would be written without its scale."""
    calls = []
    _plain_ops(monkeypatch, calls)
    c = Conversation(1, "cpu", seed=12)
    impl, _ = _through_the_backend(c)
    try:
        q, k, v = (torch.zeros(3, h * D, dtype=torch.bfloat16) for h in (H_Q, H_KV, H_KV))
        for scale in (dict(output_scale=torch.ones(1)), dict(output_block_scale=torch.ones(1))):
            out = torch.full((3, H_Q * D), 7.0).to(torch.float8_e4m3fn)
            assert impl.forward(_layer(), q, k, v, None, _meta([0], [3], c.table, "cpu"), output=out, **scale) is out
            assert (out.float() == 7.0).all()
        assert not calls and impl.native == 2
    finally:
        jb._STORES.pop("l")


@pytest.mark.parametrize("causal, window, want", [
    (True, (-1, -1), dict(causal=True, window=None)), (True, (9, 0), dict(causal=True, window=10)), (True, (9, -1), dict(causal=True, window=10)),
    (False, (-1, -1), dict(causal=False, window=None)), (False, (9, 9), dict(causal=False, window=10)), (False, (9, 0), dict(causal=True, window=10)),
    (False, (-1, 0), dict(causal=True, window=None)), (False, (9, -1), None), (False, (-1, 5), None), (False, (9, 4), None), (True, 10, dict(causal=True, window=10)),
    (False, 10, dict(causal=False, window=10)), (False, None, dict(causal=False, window=None))])
def test_windows_of_prompts_are_the_pair_s_two_sides(monkeypatch, causal, window, want):
    """(left, right): positions seen before and behind one's own, -1 for all.  What the op has no form for is refused."""
    seen = {}
    monkeypatch.setattr(B8.ops, "varlen_prefill_attn", lambda q, *a, out=None, **kw: (seen.update(kw), (q, None))[1])
    q, k, v = (torch.zeros(3, h, D, dtype=torch.bfloat16) for h in (H_Q, H_KV, H_KV))
    impl = _impl()
    impl.sliding_window = window
    args = dict(q=q, k=k, v=v, out=torch.zeros_like(q), cu_seqlens=torch.tensor([0, 3], dtype=torch.int32), max_seqlen=3, impl=impl, layer=_layer(),
                attn_metadata=SimpleNamespace(causal=causal))
    if want is None:
        with pytest.raises(ValueError, match="sliding_window"):
            B8.native_varlen_prefill(**args)
    else:
        B8.native_varlen_prefill(**args)
        assert {k: seen[k] for k in ("causal", "window")} == want
