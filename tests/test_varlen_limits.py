"""The largest calls that the packed-prompt kernel takes, by its waits, which give up after two seconds: work items are found by going through
all sequences level by level, and the next but one is not put down before an item is done."""
import ctypes as C

import pytest

from jetfire_b200 import _lib as L

LIMIT, MULTIPROCESSORS, CHUNK_US = 1 << 18, 148, 0.27   # 131072 sequences beside one of 20000 rows: 157 * 4096 chunks of 32 in 175 ms


def _status(n_seqs, **kw):
    a = L.VarlenAttnArgs()
    a.dtype, a.n_seqs, a.H_q, a.H_kv, a.causal, a.attn_scale, a.T = 0, n_seqs, 8, 2, 1, 0.1, 40
    a.q_stride_t, a.q_stride_h, a.k_stride_t, a.k_stride_h, a.v_stride_t, a.v_stride_h = 1024, 128, 256, 128, 256, 128
    for n in ("q", "k", "v", "cu_seqlens", "out"):
        setattr(a, n, 4096)
    for k, v in kw.items():
        setattr(a, k, v)
    return L.lib.jf_varlen_attn(C.byref(a), None)


@pytest.mark.parametrize("n", [LIMIT + 1, 10 ** 6, 2 ** 31 - 1])
def test_more_sequences_are_refused(n):
    assert _status(n) == L.JF_ERR_UNSUPPORTED


def test_as_many_are_found_well_within_a_wait():
    """Items of a level go to the blocks in turn, so a block passes at most as many levels between two of its own as there are blocks."""
    assert _status(LIMIT, T=0) == L.JF_OK
    assert MULTIPROCESSORS * (LIMIT // 32) * CHUNK_US < 0.25 * 2e6


@pytest.mark.parametrize("T", [(1 << 24) + 1, 2 ** 31, 2 ** 40])
def test_more_rows_are_refused(T):
    assert _status(2, T=T) == L.JF_ERR_UNSUPPORTED


def test_an_item_of_the_longest_sequence_ends_well_within_a_wait():
    """3500 cycles a key tile without a cap, 2.5 times as many where scores lie beyond one (one prompt of 8192 rows: 919 and 2322 us), at 1.3 GHz."""
    assert (1 << 24) // 128 * 3500 * 2322 / 919 / 1.3e9 < 0.5 * 2
