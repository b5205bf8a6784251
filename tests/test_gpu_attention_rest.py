"""What rounding took from the result, and the gradients that use it, by value.

All queries are 0, so every weight is 1 before the division: exact in 16 bits, and the result before its rounding is off by the sums' roundings alone, c P |V| with
c = (keys + 32) u, u = 2^-24 (attention_reference).  The rest has a half step e of its own, e e |O| of the result, or of the smallest numbers, a.  Each test also
plants the mistake in the expected values, to show that the bound tells it apart."""
import pytest
import torch

import attention_reference as R
from test_gpu_attention_c_abi import prompt

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
U = 2.0 ** -24
ROWS, HEADS, KV_HEADS = 400, 4, 2


def _exact(k, v, window, dtype):
    """Weights [queries, keys], K and V by query head, the result and its bound, in 64 bits."""
    e, a = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    seen = R.visible(ROWS, ROWS, window, 2, "cuda").double()
    P = seen / seen.sum(1, keepdim=True)
    K, V = (x.double().transpose(0, 1).repeat_interleave(HEADS // KV_HEADS, 0) for x in (k, v))
    O = P @ V
    return P, seen, K, V, O, (ROWS + 32) * U * (P @ V.abs()) + e * e * O.abs() + a, e, a


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("window", [40, 300])
@pytest.mark.parametrize("dim", [64, 128, 20, 132])     # tensor cores, FMAs
def test_rest(dim, window, dtype):
    gen = torch.Generator(device="cuda").manual_seed(60)
    q, dout = torch.zeros(ROWS, HEADS, dim, dtype=dtype, device="cuda"), torch.ones(ROWS, HEADS, dim, dtype=dtype, device="cuda")
    k, v = (torch.randn(ROWS, KV_HEADS, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    _, _, _, _, O, bound, _, _ = _exact(k, v, window, dtype)
    got = prompt(q, k, v, dout, window, 2, 0.125)
    out, rest = (got[n].double().transpose(0, 1) for n in ("out", "rest"))
    R.check(out + rest, (O, bound), "out + rest")
    for mistake in (out, out - rest):                   # no rest, and the wrong sign
        with pytest.raises(AssertionError, match="out of bounds"):
            R.check(mistake, (O, bound))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("window", [40, 300])
@pytest.mark.parametrize("dim", [64, 128, 20, 132])
def test_gradient_of_values_that_nearly_agree(dim, window, dtype):
    """Values of a column differ by one step of the type: dP - delta is as small as the rounding of the result makes delta wrong, unless its rest
    is added.  Bounds as in attention_reference, with the bound above for the result inside delta."""
    gen = torch.Generator(device="cuda").manual_seed(61)
    scale = 0.125
    q = torch.zeros(ROWS, HEADS, dim, dtype=dtype, device="cuda")
    dout = torch.randn(ROWS, HEADS, dim, generator=gen, device="cuda").to(dtype)
    k = (torch.randn(ROWS, KV_HEADS, dim, generator=gen, device="cuda") + 1).to(dtype)
    v = 1 + torch.rand(1, KV_HEADS, dim, generator=gen, device="cuda").mul(100).floor().mul(2.0 ** -7)
    v = (v + torch.finfo(dtype).eps * (torch.rand(ROWS, KV_HEADS, dim, generator=gen, device="cuda") < 0.5)).to(dtype)
    P, seen, K, V, O, out_bound, e, a = _exact(k, v, window, dtype)
    G = dout.double().transpose(0, 1)
    x = G @ V.transpose(1, 2) - (G * O).sum(-1, keepdim=True)
    c, sums = (ROWS + 32) * U, (dim + 4) * U
    off = (G.abs() * out_bound).sum(-1, keepdim=True) + sums * (G.abs() * O).sum(-1, keepdim=True)
    dS = P * x
    dS_off = P * ((e + c + 50 * U) * x.abs() + off + sums * (G.abs() @ V.transpose(1, 2))) + a * seen * (x.abs() + 1)
    dQ = scale * (dS @ K)
    bound = a + e * dQ.abs() + scale * (dS_off @ K.abs()) + (ROWS + 32) * U * scale * (dS.abs() @ K.abs())
    got = prompt(q, k, v, dout, window, 2, scale)["dq"].transpose(0, 1)
    R.check(got, (dQ, bound), "dq")
    rounded = O.to(dtype).double()
    for wrong in (rounded, 2 * rounded - O):            # delta without the rest, and with the wrong sign
        mistake = scale * ((P * (G @ V.transpose(1, 2) - (G * wrong).sum(-1, keepdim=True))) @ K)
        with pytest.raises(AssertionError, match="out of bounds"):
            R.check(mistake, (dQ, bound))
