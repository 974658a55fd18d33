"""Which calls over a shared prefix go through the decode kernel, seen by the scratch that they ask for: that of the decode attention."""
import pytest

from test_block8_args import L  # noqa: F401  (the library, as a fixture)


def _by_decode(L, B, H_q, H_kv, positions):
    max_S = positions + 500
    asked = L.lib.jf_block8_shared_workspace_bytes(B, H_q, H_kv, max_S, positions // 16)
    assert asked > 0
    return asked == L.lib.jf_block8_workspace_bytes(B, H_q, H_kv, max_S)


@pytest.mark.parametrize("positions", [2048, 65536, 131072, 2 ** 20])
@pytest.mark.parametrize("H_q, H_kv", [(32, 8), (64, 8), (8, 1), (8, 8)])
@pytest.mark.parametrize("B", [1, 2, 3])
def test_so_few_sequences_have_nothing_to_share(L, B, H_q, H_kv, positions):
    assert _by_decode(L, B, H_q, H_kv, positions)


@pytest.mark.parametrize("positions", [65536, 2 ** 20])
def test_one_sequence_of_sixteen_heads(L, positions):
    assert _by_decode(L, 1, 32, 2, positions) and _by_decode(L, 1, 16, 1, positions)


@pytest.mark.parametrize("B, H_q, H_kv, positions", [(4, 32, 8, 65536), (8, 32, 8, 16384), (16, 32, 8, 4096), (64, 64, 8, 2048), (256, 64, 8, 65536),
                                                     (8, 8, 1, 65536), (4, 32, 2, 65536), (2, 40, 1, 131072), (90, 64, 8, 480), (256, 8, 1, 1024)])
def test_many_or_long(L, B, H_q, H_kv, positions):
    assert not _by_decode(L, B, H_q, H_kv, positions)


@pytest.mark.parametrize("B, H_q, H_kv, positions", [(4, 32, 8, 2048), (64, 32, 8, 512), (16, 8, 1, 16384), (100, 64, 8, 0), (4, 32, 2, 16384), (2, 40, 1, 16384), (1, 40, 1, 131072),
                                                     (256, 64, 8, 256), (256, 32, 8, 128)])
def test_short(L, B, H_q, H_kv, positions):
    assert _by_decode(L, B, H_q, H_kv, positions)
