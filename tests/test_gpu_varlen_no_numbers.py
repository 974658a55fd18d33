"""Attention of packed prompts where a score is no number or infinite and a cap is given.

A cap makes an infinite score the cap, and does not make a number of a NaN: a row whose query is NaN, or that sees a key
that is NaN, is NaN and so is its lse; the others are as ever (tolerances of test_gpu_varlen_attn.py)."""
import pytest
import torch

import block8_ref as R
from test_gpu_varlen_attn import Case

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def _check(c, out, lse):
    out, lse, eps = out.cpu().double(), lse.cpu().double(), torch.finfo(c.dtype).eps
    for lo, n in zip(c.start(), c.lens):
        q, k, v = (t[lo:lo + n].double().transpose(0, 1) for t in (c.q, c.k, c.v))
        i = torch.arange(n)
        want, want_lse = R.attend(q, k, v, i, i, c.scale, slopes=c.slopes, **c.kw)
        want, want_lse = want.transpose(0, 1), want_lse.t()
        got, got_lse = out[lo:lo + n], lse[lo:lo + n]
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isnan(got_lse), torch.isnan(want_lse))
        fin = ~torch.isnan(want_lse)
        tol = (eps / 2 + 2 ** -13) * v.abs().amax() + eps / 2 * want.abs()
        assert ((got - want).abs()[fin] <= tol[fin]).all()
        assert ((got_lse - want_lse).abs()[fin] <= 2 ** -13 + 2 ** -21 * want_lse[fin].abs()).all()


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("softcap", [0.5, 4.0, 1000.0])
@pytest.mark.parametrize("options", [dict(), dict(alibi=True), dict(window=150), dict(causal=False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_queries_under_a_cap(value, softcap, options, dtype):
    """A row in a masked tile, one that has whole tiles in front of it, one of the second head."""
    c = Case([400, 33], 2, 1, dtype, 71, softcap=softcap, **options)
    c.q[37, 0, 3] = c.q[300, 0, 9] = c.q[301, 1, 0] = c.q[405, 1, 8] = value
    _check(c, *c.run())


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("softcap", [0.5, 4.0, 1000.0])
@pytest.mark.parametrize("options", [dict(), dict(alibi=True), dict(window=150), dict(causal=False)])
def test_keys_under_a_cap(value, softcap, options):
    """Seen by the rows behind it, or by those of a window: the others are as ever."""
    c = Case([400, 33], 2, 1, torch.bfloat16, 72, softcap=softcap, **options)
    c.k[100, 0, 17] = value
    _check(c, *c.run())
