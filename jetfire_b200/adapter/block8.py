"""Layers whose keys and values are kept in 8 bits, without a host mirror and its correction.

For layers that need more than the 2 to 4 bits of the release modes.  ``JetFireBlock8Store`` holds a
layer's cache (codes, one scale per block of 16 positions and KV head); ``try_block8_attention``
serves a step of it: every new token is appended, sequences with one query token attend over the
cache (``ops.block8_decode_attn``), prompts attend over the step's own keys and values
(``ops.varlen_prefill_attn``), both with the implementation's score cap, distance bias and window.  A decode step of
sequences that share a prefix (vLLM's cascade steps) reads the prefix once for all of them (``ops.block8_shared_prefix_attn``); a store made
for it keeps block bounds and lets a decode token attend to its best blocks only (``ops.block8_sparse_decode_attn``; a choice of the
user's, ``JETFIRE_BLOCK8_TOP``).

Nothing of the decode part waits on the host: a step of decode sequences can be captured in a graph.  What they share is known on the
host only and may be another prefix when the graph is replayed, so a captured cascade step goes through every sequence's whole table.
"""
from __future__ import annotations

import torch

from .. import ops
from .config import BLOCK8_CODES, BLOCK8_FIRST, BLOCK8_LAST
from .mixed_batch import split_mixed_batch


class JetFireBlock8Store:
    """Cache of one layer: ``k_data / v_data (H_kv, num_blocks * 16, 128)`` int8 or float8_e4m3fn, ``k_scales /
    v_scales (H_kv, num_blocks)`` float32.  ``top_blocks``: blocks that a decode token attends to (0: all); the store then keeps
    ``bounds (H_kv, num_blocks, 2, 128)`` int8 to choose them by."""

    def __init__(self, *, num_blocks: int, num_kv_heads: int, head_dim: int = 128, codes: str = "int8", device="cuda",
                 block_size: int = 16, top_blocks: int = 0):
        if top_blocks != 0 and top_blocks < BLOCK8_FIRST + BLOCK8_LAST:
            raise ValueError(f"top_blocks must be 0 or at least {BLOCK8_FIRST + BLOCK8_LAST}, got {top_blocks}")
        if head_dim != 128 or block_size != 16:
            raise ValueError("the 8-bit cache is built for head_dim 128 and block_size 16")
        if codes not in BLOCK8_CODES:
            raise ValueError(f"codes must be one of {BLOCK8_CODES}, got {codes!r}")
        self.codes, self.head_dim, self.block_size = codes, head_dim, block_size
        self.num_blocks, self.num_kv_heads = int(num_blocks), int(num_kv_heads)
        self.num_slots = self.num_blocks * block_size
        self.device = torch.device(device)
        data = dict(dtype=ops.BLOCK8_DTYPES[codes], device=self.device)
        self.k_data = torch.zeros(self.num_kv_heads, self.num_slots, head_dim, **data)
        self.v_data = torch.zeros(self.num_kv_heads, self.num_slots, head_dim, **data)
        self.k_scales = torch.zeros(self.num_kv_heads, self.num_blocks, dtype=torch.float32, device=self.device)
        self.v_scales = torch.zeros(self.num_kv_heads, self.num_blocks, dtype=torch.float32, device=self.device)
        self.top_blocks = int(top_blocks)
        self.bounds = torch.zeros(self.num_kv_heads, self.num_blocks, 2, head_dim, dtype=torch.int8, device=self.device) if top_blocks else None

    def append(self, key, value, query_start_loc, seq_lens, block_table) -> None:
        """``key / value (T, H_kv, 128)``: the new tokens of a step, ``seq_lens`` counting them already."""
        kept = dict(bounds=self.bounds) if self.bounds is not None else {}
        ops.block8_append(key, value, query_start_loc, seq_lens, block_table, self.k_data, self.k_scales, self.v_data, self.v_scales, **kept)

    def append_rotary(self, query, key, value, positions, cos_sin, query_start_loc, seq_lens, block_table, *, interleaved=False, out=None):
        """``append`` of keys that are rotated by their positions on the way; returns the rotated queries (``ops.block8_append_rotary``)."""
        return ops.block8_append_rotary(query, key, value, positions, cos_sin, query_start_loc, seq_lens, block_table, self.k_data, self.k_scales,
                                        self.v_data, self.v_scales, interleaved=interleaved, bounds=self.bounds, out=out)

    def decode(self, q, seq_lens, block_table, max_S, scale, *, shared_blocks=0, **options):
        """Attention of one query token per sequence: over the best blocks where the store chooses (``ops.block8_sparse_decode_attn``), else with
        the first ``shared_blocks`` blocks of the first row, the same for all sequences, read once (``ops.block8_shared_prefix_attn``),
        else over everything (``ops.block8_decode_attn``, which also serves layers with a window or a bias by distance)."""
        cache = (q, self.k_data, self.k_scales, self.v_data, self.v_scales)
        sizes = (seq_lens, max_S, int(q.shape[1]), self.num_kv_heads, self.block_size, scale)
        if any(options.get(name) is not None for name in ("window", "alibi_slopes", "prefix_lens")):
            return ops.block8_decode_attn(*cache, block_table, *sizes, **options)
        options = {k: v for k, v in options.items() if v is not None}
        if self.top_blocks and scale > 0:
            out, lse, _ = ops.block8_sparse_decode_attn(*cache, self.bounds, block_table, *sizes, top_blocks=self.top_blocks, first_blocks=BLOCK8_FIRST,
                                                        last_blocks=BLOCK8_LAST, **options)
            return out, lse
        if shared_blocks and q.shape[0]:
            return ops.block8_shared_prefix_attn(*cache, block_table[0, :shared_blocks], block_table[:, shared_blocks:], *sizes, **options)
        return ops.block8_decode_attn(*cache, block_table, *sizes, **options)


def score_options(impl, device) -> dict:
    """The implementation's score cap, slopes and window as the ops' arguments.  A window is a pair (left, right) as
    vLLM's FlashAttentionImpl holds it, -1 for none; a causal one sees its own position and ``left`` before it."""
    window = getattr(impl, "sliding_window", None)
    if window is not None:
        left = int(window[0]) if isinstance(window, (tuple, list)) else int(window) - 1
        window = left + 1 if left >= 0 else None
    slopes = getattr(impl, "alibi_slopes", None)
    if slopes is not None and (slopes.device != device or slopes.dtype != torch.float32 or not slopes.is_contiguous()):
        # brought over once and kept where they came from: a captured step cannot wait for the host
        if device.type == "cuda" and slopes.device.type == "cpu" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("alibi_slopes are on the host: run a step before one is captured")
        slopes = impl.alibi_slopes = slopes.to(device=device, dtype=torch.float32).contiguous()
    return dict(softcap=float(getattr(impl, "logits_soft_cap", None) or 0.0), window=window, alibi_slopes=slopes)


def served(impl) -> bool:
    """Whether a layer's attention is one of queries over the layer's own keys and values, with no terms but those of ``score_options``: a
    decoder's, without a per-head term in the softmax's denominator (``sinks``) and without another layer's cache in place of its own."""
    attn_type = getattr(impl, "attn_type", None)
    attn_type = getattr(attn_type, "name", attn_type)
    return (attn_type is None or str(attn_type).upper() == "DECODER") and getattr(impl, "sinks", None) is None \
        and getattr(impl, "kv_sharing_target_layer_name", None) is None


def native_varlen_prefill(*, q, k, v, out, cu_seqlens, max_seqlen, impl, layer, attn_metadata) -> None:
    """Attention of a step's prompts by this library's own kernel: a ``prefill_attention`` for ``try_jetfire_mixed``.  Raises if a
    wait inside an earlier one ran out (``ops.varlen_prefill_status``)."""
    direct = out.is_contiguous() and out.data_ptr() % 16 == 0
    causal, window = bool(getattr(attn_metadata, "causal", True)), getattr(impl, "sliding_window", None)
    if not causal and isinstance(window, (tuple, list)):     # (left, right): the op sees as far to both sides, or nothing behind
        left, right = (int(w) for w in window)
        causal = right == 0
        if not causal and max(left, -1) != max(right, -1):
            raise ValueError(f"prompts that see {left} positions before and {right} behind their own (sliding_window) are not served")
    got, _ = ops.varlen_prefill_attn(q, k, v, cu_seqlens, float(impl.scale), causal=causal, out=out if direct else None,
                                     **score_options(impl, q.device))
    if not direct:
        out.copy_(got)


def _int32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def try_block8_attention(*, impl, layer, query, key, value, attn_metadata, output, store: JetFireBlock8Store):
    """One step of a layer with an 8-bit cache: append, then attention.  ``query (T, H_q, D)`` or ``(T, H_q * D)``, ``key`` /
    ``value`` likewise with the KV heads, ``output`` like ``query``.  Returns ``output``, or None when the step's attention
    is not one this path serves and the caller's native attention has to.  The tokens are appended all the same where a later step
    may be served -- after prompts with cached context, several query tokens over a cache, cascade steps other than of decode tokens -- and
    not in a layer that never is (``served``)."""
    H_q, H_kv, D = int(layer.num_heads), int(layer.num_kv_heads), int(layer.head_size)
    T = int(attn_metadata.num_actual_tokens)
    if T == 0 or not served(impl):
        return None
    if D != store.head_dim or H_kv != store.num_kv_heads:
        raise ValueError(f"the layer's 8-bit cache has {store.num_kv_heads} heads of {store.head_dim}, the layer {H_kv} of {D}")
    capturing = query.is_cuda and torch.cuda.is_current_stream_capturing()
    if query.is_cuda and not capturing:
        ops.varlen_prefill_status(query.device)        # an error of an earlier step's prompts, as far as it has arrived
    n = int(attn_metadata.seq_lens.numel())
    q = query[:T].reshape(T, H_q, D)
    k, v = key[:T].reshape(T, H_kv, D), value[:T].reshape(T, H_kv, D)
    start, lens, table = _int32(attn_metadata.query_start_loc[:n + 1]), _int32(attn_metadata.seq_lens), attn_metadata.block_table[:n]
    store.append(k, v, start, lens, table)
    shared = 0      # blocks that all sequences begin with
    if getattr(attn_metadata, "use_cascade", False):
        shared = min(int(getattr(attn_metadata, "common_prefix_len", 0) or 0) // store.block_size, int(table.shape[1]))
        if shared == 0 or int(attn_metadata.max_query_len) != 1:
            return None
        if capturing:      # (replayed with sequences that share something else, or nothing: everything is in their tables too)
            shared = 0
    if int(getattr(impl, "dcp_world_size", 1) or 1) > 1 or not bool(getattr(attn_metadata, "causal", True)):
        return None
    options = score_options(impl, q.device)
    width = int(table.shape[1]) * store.block_size

    def decode_rows(rows, q_rows, lens_rows, table_rows):
        # (a captured step is replayed with other lengths: up to what the table holds)
        longest = width if capturing else min(int(attn_metadata.max_seq_len), width)
        out, _ = store.decode(q_rows, lens_rows, table_rows, max(longest, 1), float(impl.scale), shared_blocks=shared, **options)
        out = out.reshape(out.shape[0], *output.shape[1:])
        if isinstance(rows, slice):
            output[rows].copy_(out)
        else:
            output.index_copy_(0, rows, out)

    if int(attn_metadata.max_query_len) == 1:
        if T < n:      # some sequences have no token: whose a row is, worked out on the device
            seqs = torch.searchsorted(start[1:], torch.arange(T, device=q.device, dtype=torch.int32), right=True).clamp_(max=n - 1)
            decode_rows(slice(0, T), q, lens.index_select(0, seqs), table.index_select(0, seqs))
        else:          # (rows behind the sequences are padding)
            decode_rows(slice(0, n), q[:n], lens, table)
        return output
    if capturing:
        return None                                # which rows are prompts is read from the device
    counts = [getattr(attn_metadata, name, None) for name in ("num_decodes", "num_prefills", "num_decode_tokens", "num_prefill_tokens")]
    if all(c is not None for c in counts) and getattr(attn_metadata, "jetfire_prefill_has_context", None) is False:
        nd, npre, ndt, npt = (int(c) for c in counts)
        if nd != ndt:
            return None
        dec, pre = slice(0, nd), slice(ndt, ndt + npt)
        cu = start[nd:nd + npre + 1] - ndt
        dec_lens, dec_table, longest = lens[:nd], table[:nd], int(attn_metadata.max_query_len)
    else:
        sp = split_mixed_batch(start.tolist(), lens.tolist())
        if sp.prefill_with_context:
            return None
        dev = q.device
        dec, pre = (torch.tensor(r, device=dev, dtype=torch.long) for r in (sp.decode_rows, sp.prefill_rows))
        cu = torch.tensor(sp.prefill_cu, device=dev, dtype=torch.int32)
        seqs = torch.tensor(sp.decode_seqs, device=dev, dtype=torch.long)
        dec_lens, dec_table, longest = lens.index_select(0, seqs), table.index_select(0, seqs), sp.max_prefill_len
        nd, npt = len(sp.decode_rows), len(sp.prefill_rows)
    if nd:
        decode_rows(dec, q[dec], dec_lens, dec_table)
    if npt:
        out = torch.empty(npt, H_q, D, dtype=output.dtype, device=output.device)
        native_varlen_prefill(q=q[pre], k=k[pre], v=v[pre], out=out, cu_seqlens=cu.contiguous(), max_seqlen=longest, impl=impl, layer=layer,
                              attn_metadata=attn_metadata)
        out = out.reshape(npt, *output.shape[1:])
        if isinstance(pre, slice):
            output[pre].copy_(out)
        else:
            output.index_copy_(0, pre, out)
    return output
