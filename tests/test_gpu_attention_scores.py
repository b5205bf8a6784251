"""Scores that are NaN or infinite in blocks of keys that a tile of queries sees whole."""
import pytest
import torch

import attention_reference as R
from test_gpu_attention_c_abi import prompt

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _make(rows, keys, dim, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q, dout = (torch.randn(rows, 4, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    k, v = (torch.randn(keys, 2, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    return q, k, v, dout


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("at", [1, 4, 16, 101])
def test_key_or_value_that_is_nan(at, what, dim, dtype):
    """Every query behind it has NaN, whatever the place of the key in its block."""
    q, k, v, dout = _make(600, 600, dim, dtype, 50)
    (k if what == "k" else v)[at] = float("nan")
    got = prompt(q, k, v, dout, 1000, 0, dim ** -0.5)
    assert bool(got["out"][at:].isnan().all())
    if what == "k":
        assert bool(got["lse"][:, at:].isnan().all()) and bool(got["dq"][at:].isnan().all())
        assert bool(got["dk"].isnan().all()) and bool(got["dv"].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_are_all_minus_infinity(dim, dtype):
    """No key has a weight: zeros, as for a query that sees no key."""
    q, k, v, dout = _make(300, 600, dim, dtype, 51)
    q[..., 0], k[..., 0] = 1.0, -float("inf")
    got = prompt(q, k, v, dout, 1000, 0, dim ** -0.5)
    assert not got["out"].any() and bool((got["lse"] == -float("inf")).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_some_scores_that_are_minus_infinity(dim, dtype):
    """Those keys have no weight at all, however large their values are, and no gradient."""
    q, k, v, dout = _make(300, 900, dim, dtype, 52)
    off = torch.arange(900, device="cuda") % 3 == 0
    q[..., 0] = 1.0
    keys, values = k.clone(), v.clone()
    k[off, :, 0], v[off] = -float("inf"), torch.finfo(dtype).max
    keys[off], values[off] = 0.0, 0.0
    seen = R.visible(300, 900, 2000, 0, "cuda") & ~off
    want = R.one_sequence(q, keys, values, seen, dim ** -0.5, dout)
    R.check(prompt(q, k, v, dout, 2000, 0, dim ** -0.5)["out"], want["out"])
    v[off] = values[off]
    got = prompt(q, k, v, dout, 2000, 0, dim ** -0.5)
    for name in ("out", "dk", "dv"):
        R.check(got[name], want[name], name)
    assert not got["dk"][off].any() and not got["dv"][off].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_far_below_the_largest(dtype):
    """Weights below the smallest number are 0."""
    q, k, v, dout = _make(300, 900, 64, dtype, 53)
    far = torch.arange(900, device="cuda") % 3 == 0
    q[..., 0], k[..., 0] = 1.0, 0.0
    keys, values = k.clone(), v.clone()
    k[far, :, 0], v[far] = -4000.0, torch.finfo(dtype).max      # scores of -500 and less
    keys[far], values[far] = 0.0, 0.0
    seen = R.visible(300, 900, 2000, 0, "cuda") & ~far
    R.check(prompt(q, k, v, dout, 2000, 0, 0.125)["out"], R.one_sequence(q, keys, values, seen, 0.125)["out"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 20])
def test_gradients_where_all_scores_are_minus_infinity(dim, dtype):
    """Weights of 0: no gradient of those keys and values, and none of the others is lost."""
    q, k, v, dout = _make(300, 300, dim, dtype, 54)
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[100:200, :, 0] = -float("inf")
    off = torch.zeros(300, dtype=torch.bool, device="cuda")
    off[100:200] = True
    keys = k.clone()
    keys[off] = 0.0
    seen = R.visible(300, 300, 40, 0, "cuda") & ~off            # queries 139 to 199 see keys of no weight alone
    want = R.one_sequence(q, keys, v, seen, 0.125, dout)
    got = prompt(q, k, v, dout, 40, 0, 0.125)
    assert not got["out"][139:200].any() and bool((got["lse"][:, 139:200] == -float("inf")).all())
    for name in ("out", "dk", "dv"):
        R.check(got[name], want[name], name)
    assert not got["dk"][off].any() and not got["dv"][off].any()
