"""Cascade steps and chosen blocks of layers with an 8-bit cache: routing on the CPU with the ops replaced by plain forms, whole steps on the GPU
against the definition in 64 bits."""
from types import SimpleNamespace

import pytest
import torch

import block8_more_ref as M
import block8_ref as R
from jetfire_b200.adapter import block8 as B8
from jetfire_b200.adapter import config as jcfg
from jetfire_b200.adapter import jetfire_backend as jb
from jetfire_b200.adapter.registry import install_layer_stores
from test_block8_adapter import D, H_KV, H_Q, Conversation, _impl, _layer, _meta, _plain_ops


def _more_plain_ops(monkeypatch, calls):
    _plain_ops(monkeypatch, calls)
    decode = B8.ops.block8_decode_attn

    def shared(q, kd, ks, vd, vs, shared_table, table, lens, max_S, *rest, **options):
        calls.append(("shared", shared_table.tolist(), tuple(table.shape), sorted(options)))
        return decode(q, kd, ks, vd, vs, torch.cat([shared_table.expand(table.shape[0], -1), table], 1), lens, max_S, *rest, **options)

    def sparse(q, kd, ks, vd, vs, bounds, table, lens, max_S, *rest, top_blocks, first_blocks, last_blocks, **options):
        calls.append(("sparse", top_blocks, first_blocks, last_blocks, sorted(options)))
        return (*decode(q, kd, ks, vd, vs, table, lens, max_S, *rest, **options), None)

    append = B8.ops.block8_append

    def append_kept(*a, bounds=None):
        calls.append(("bounds", bounds is not None))
        return append(*a)

    monkeypatch.setattr(B8.ops, "block8_append", append_kept)
    monkeypatch.setattr(B8.ops, "block8_shared_prefix_attn", shared)
    monkeypatch.setattr(B8.ops, "block8_sparse_decode_attn", sparse)


def _cascade(common):
    def call(attn_metadata, **a):
        attn_metadata.use_cascade, attn_metadata.common_prefix_len = True, common
        return B8.try_block8_attention(attn_metadata=attn_metadata, **a)
    return call


def _sharing(n, device, blocks, top=0, codes=torch.int8, **kw):
    """A conversation whose sequences have the same first blocks, filled once for all."""
    c = Conversation(n, device, codes=codes, **kw)
    c.table[:, :blocks] = c.table[0, :blocks]
    c.store = B8.JetFireBlock8Store(num_blocks=n * 40, num_kv_heads=H_KV, codes="int8" if codes == torch.int8 else "e4m3", device=device, top_blocks=top)
    return c


def _fill(c, blocks, own):
    """The shared blocks as a prompt of the first sequence, then each one's own positions as prompts behind them (appended, handed back)."""
    first = [16 * blocks] + [0] * (c.n - 1)
    c.step(first)
    c.lens = [16 * blocks] * c.n
    assert c.step(own) is None
    return c


def test_cascade_steps_of_decode_tokens_are_served(monkeypatch):
    calls = []
    _more_plain_ops(monkeypatch, calls)
    c = _fill(_sharing(3, "cpu", 4, seed=21), 4, [5, 9, 2])
    calls.clear()
    assert c.step([1, 1, 1], call=_cascade(64 + 7)) is not None       # (whole blocks of it)
    names = [x[0] for x in calls]
    assert names == ["bounds", "append", "shared", "decode"] and calls[0][1] is False
    assert calls[2][1] == c.table[0, :4].tolist() and calls[2][2] == (3, 36) and calls[2][3] == ["softcap"]


@pytest.mark.parametrize("common, news", [(0, [1, 1]), (15, [1, 1]), (64, [3, 1])])
def test_other_cascade_steps_are_handed_back(monkeypatch, common, news):
    calls = []
    _more_plain_ops(monkeypatch, calls)
    c = _fill(_sharing(2, "cpu", 4, seed=22), 4, [5, 9])
    calls.clear()
    assert c.step(news, call=_cascade(common)) is None
    assert [x[0] for x in calls] == ["bounds", "append"]


@pytest.mark.parametrize("settings", [dict(sliding_window=(20, 0)), dict(alibi_slopes=torch.full((H_Q,), 0.1))])
def test_layers_with_a_window_or_a_bias_go_through_the_decode_attention(monkeypatch, settings):
    calls = []
    _more_plain_ops(monkeypatch, calls)
    for top in (0, 4):
        c = _sharing(2, "cpu", 4, top=top, seed=23, **settings)
        _fill(c, 4, [5, 9])
        calls.clear()
        assert c.step([1, 1], call=_cascade(64)) is not None
        assert [x[0] for x in calls] == ["bounds", "append", "decode"] and calls[0][1] is (top > 0)


def test_a_store_that_chooses(monkeypatch):
    calls = []
    _more_plain_ops(monkeypatch, calls)
    c = _sharing(2, "cpu", 0, top=5, seed=24)
    c.step([100, 3])
    assert c.step([1, 1]) is not None
    assert [x for x in calls if x[0] == "sparse"] == [("sparse", 5, 1, 2, ["softcap"])] and all(x[1] for x in calls if x[0] == "bounds")
    assert c.store.bounds.shape == (H_KV, 80, 2, 128)
    calls.clear()
    c.impl.scale = -c.impl.scale                         # (scores are for positive scales)
    assert c.step([1, 1]) is not None
    assert not [x for x in calls if x[0] == "sparse"]


def test_configuration(monkeypatch):
    monkeypatch.setenv("JETFIRE_BLOCK8", "int8")
    for raw, want in (("", 0), ("0", 0), ("3", 3), ("128", 128)):
        monkeypatch.setenv("JETFIRE_BLOCK8_TOP", raw)
        jcfg.reset_jetfire_config()
        assert jcfg.get_jetfire_config().block8_top == want
    for raw in ("1", "2", "-4", "x"):
        monkeypatch.setenv("JETFIRE_BLOCK8_TOP", raw)
        jcfg.reset_jetfire_config()
        with pytest.raises(ValueError, match="JETFIRE_BLOCK8_TOP"):
            jcfg.get_jetfire_config()
    monkeypatch.setenv("JETFIRE_BLOCK8", "off")
    monkeypatch.setenv("JETFIRE_BLOCK8_TOP", "64")
    jcfg.reset_jetfire_config()
    with pytest.raises(ValueError, match="JETFIRE_BLOCK8"):
        jcfg.get_jetfire_config()
    monkeypatch.undo()
    jcfg.reset_jetfire_config()
    with pytest.raises(ValueError, match="top_blocks"):
        B8.JetFireBlock8Store(num_blocks=2, num_kv_heads=1, device="cpu", top_blocks=2)
    layer = SimpleNamespace(num_kv_heads=2, head_size=128, impl=_impl())
    got = install_layer_stores({"z": layer}, num_blocks=4, device="cpu", cfg=jcfg.JetFireConfig(block8="e4m3", block8_top=6))
    assert got["z"].top_blocks == 6 and got["z"].bounds.shape == (2, 4, 2, 128)
    jb._STORES.pop("z")


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_cascade_steps_on_the_device(codes):
    c = _fill(_sharing(5, "cuda", 12, codes=codes, seed=25), 12, [30, 1, 17, 90, 16])
    for _ in range(3):
        assert c.step([1] * 5, call=_cascade(16 * 12)) is not None      # (checks the rows itself)
    assert c.step([1] * 5) is not None


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_chosen_blocks_on_the_device(codes):
    """As many blocks as there are: the whole sequence; fewer: those of the plain choice."""
    c = _sharing(3, "cuda", 0, top=40, codes=codes, seed=26)
    c.step([300, 17, 100])
    assert c.step([1, 1, 1]) is not None
    c.store.top_blocks = 6
    q = torch.randn(3, H_Q, D, generator=c.gen).to(torch.bfloat16)
    lens = torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    out, _ = c.store.decode(q.cuda(), lens, c.table.cuda(), 640, c.impl.scale, softcap=0.0, window=None, alibi_slopes=None)
    code, scale = c.side[0]
    G = H_Q // H_KV
    for b, length in enumerate(c.lens):
        n = (length + 15) // 16
        for g in range(H_KV):
            bounds = c.store.bounds[g].cpu()
            for blk in range(n):
                i = int(c.table[b, blk])
                assert torch.equal(bounds[i].double(), M.bounds_of(code[:, i], min(16, length - 16 * blk), codes)[g])
            heads = slice(g * G, (g + 1) * G)
            pick = M.choose(q[b, heads].double(), bounds, scale[g], c.table[b].long(), n, 6, 1, 2, codes, scale.shape[1])
            j = torch.tensor([p * 16 + r for p in pick for r in range(16) if p * 16 + r < length])
            ids = c.table[b].long()[j // 16]
            kk, vv = ((x * s[..., None, None])[g, ids, j % 16][None] for x, s in c.side)
            o, _ = R.attend(q[b, heads].double()[:, None], kk, vv, torch.tensor([length - 1]), j, c.impl.scale)
            # weights of half a step 2^-11 and scores below 2^-14 of one, then bf16
            tol = (2 ** -11 + 2 ** -14) * vv.abs().max() + 2 ** -8 * o.abs()
            assert ((out[b, heads].double().cpu() - o[:, 0]).abs() <= tol[:, 0]).all()


@pytest.mark.gpu
def test_a_cascade_step_in_a_graph():
    """Decode tokens over a shared prefix: captured, replayed with longer sequences."""
    c = _fill(_sharing(4, "cuda", 8, seed=27), 8, [30, 1, 17, 60])
    q, k, v = (torch.zeros(4, h * D, dtype=torch.bfloat16, device="cuda") for h in (H_Q, H_KV, H_KV))
    out = torch.zeros_like(q)
    md = _meta(c.lens, [1] * 4, c.table, "cuda")
    md.use_cascade, md.common_prefix_len = True, 128
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        assert B8.try_block8_attention(impl=c.impl, layer=_layer(), query=q, key=k, value=v, attn_metadata=md, output=out, store=c.store) is out
    other = _fill(_sharing(4, "cuda", 8, seed=27), 8, [30, 1, 17, 60])
    for i in range(3):
        new = [torch.randn(4, h * D, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda() for h in (H_Q, H_KV, H_KV)]
        for x, y in zip((q, k, v), new):
            x.copy_(y)
        lens = [n + i + 1 for n in c.lens]
        md.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        eager = _meta([n - 1 for n in lens], [1] * 4, other.table, "cuda")
        eager.use_cascade, eager.common_prefix_len = True, 128
        eager.max_seq_len = 640
        want = torch.zeros_like(out)
        B8.try_block8_attention(impl=c.impl, layer=_layer(), query=new[0], key=new[1], value=new[2], attn_metadata=eager, output=want, store=other.store)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(c.store.k_data, other.store.k_data)
