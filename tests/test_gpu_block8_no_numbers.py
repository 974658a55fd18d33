"""Decode attention over the 8-bit cache where a score is no number and a cap is given: the cap does not make a number of it.

A row whose query is NaN, or that sees a key that is NaN, is NaN and so is its lse; the others are as ever (tolerances of
test_gpu_block8.py).  Caps far below the scores, about their size and far above take every branch of the cap's arithmetic."""
import pytest
import torch

from test_gpu_block8 import CODES, Decode

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _check(c, out, lse):
    want, want_lse = c.expected()
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    fin = ~torch.isnan(want_lse)
    vmax = (c.v.abs() * c.vs[..., None, None]).amax().item()
    tol = (2 ** -11 + 2 ** -14) * vmax + torch.finfo(c.dtype).eps / 2 * want.abs()
    assert ((out - want).abs()[fin] <= tol[fin]).all()
    assert ((lse - want_lse).abs()[fin] <= 2 ** -14 + 2 ** -22 * want_lse[fin].abs()).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("softcap", [0.0, 0.5, 4.0, 1000.0])
@pytest.mark.parametrize("lens, heads", [([40], (8, 2)), ([3000], (8, 2)), ([90, 700], (16, 1))])
def test_a_query_that_is_nan(codes, softcap, lens, heads):
    c = Decode(lens, *heads, CODES[codes], torch.bfloat16, 61, softcap=softcap)
    c.q[0, 3, 77] = NAN
    _check(c, *c.run())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("softcap", [0.0, 0.5, 4.0, 1000.0])
@pytest.mark.parametrize("options", [dict(), dict(alibi=True), dict(window=300), dict(window=60)])
def test_a_key_that_is_nan(codes, softcap, options):
    """Position 600 of 800: seen without a window and with the wider one.  (int8 codes are always numbers, so there the block's
    scale is none.)"""
    c = Decode([800, 50], 8, 2, CODES[codes], torch.float16, 62, softcap=softcap, **options)
    block, row = c.table[0, 600 // 16], 600 % 16
    if codes == "e4m3":
        c.k[1, block, row, 5] = NAN
    else:
        c.ks[1, block] = NAN
    _check(c, *c.run())
