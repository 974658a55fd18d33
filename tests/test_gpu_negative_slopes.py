"""A bias that grows with distance: with negative slopes the keys far away are the heavy ones, so that what rounding takes from a large bias is
what the weights get.

Tolerances of the two operators' own tests, and the bias's: its largest, in units of log2, is |slope| n log2(e) < 2^10 here.  The prompts' kernel
adds it up in eight steps and once more to the score, nine roundings of half of 2^-14: 2^-11.8 in the exponent, so a factor of 2^-12.3
of a weight, on it and on the sum.  The decode kernel rounds it once, and twice more with log2 of the V scale and the reference: three halves
of 2^-14, 2^-13.4, a factor of 2^-13.9, on both."""
import pytest
import torch

import block8_ref as R
from test_gpu_block8 import CODES, Decode
from test_gpu_varlen_attn import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("options", [dict(), dict(causal=False), dict(window=300), dict(softcap=5.0), dict(prefix=[128], window=100)])
def test_prompts(dtype, options):
    n = 900
    c = Case([n], 4, 2, dtype, 91, **options)
    c.slopes = torch.tensor([-0.75, -0.5, -0.03, 0.2])
    out, lse = c.run()
    q, k, v = (t.double().transpose(0, 1) for t in (c.q, c.k, c.v))
    i = torch.arange(n)
    want, want_lse = R.attend(q, k, v, i, i, c.scale, slopes=c.slopes, prefix=c.prefix[0] if c.prefix else 0, **c.kw)
    want, want_lse = want.transpose(0, 1), want_lse.t()
    eps = torch.finfo(dtype).eps
    tol = (eps / 2 + 2 ** -13 + 2 * 2 ** -12.3) * v.abs().amax() + eps / 2 * want.abs()
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert ((lse.cpu().double() - want_lse).abs() <= 2 ** -13 + 2 ** -12.3 + 2 ** -21 * want_lse.abs()).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("options", [dict(), dict(window=300), dict(softcap=5.0), dict(prefix=[50], window=100)])
def test_decode(codes, options):
    c = Decode([900], 8, 2, CODES[codes], torch.float16, 92, **options)
    c.slopes = torch.tensor([-0.75, -0.5, -0.03, 0.2] * 2)
    out, lse = c.run()
    want, want_lse = c.expected()
    vmax = (c.v.abs() * c.vs[..., None, None]).amax().item()
    tol = (2 ** -11 + 2 ** -14 + 2 * 2 ** -13.9) * vmax + 2 ** -11 * want.abs()
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert ((lse.cpu().double() - want_lse).abs() <= 2 ** -14 + 2 ** -13.9 + 2 ** -22 * want_lse.abs()).all()
