"""NaN and infinities where a query sees them: they reach its result, through every kernel, part and join."""
import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAN, INF = float("nan"), float("inf")


def _normal(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _caches(batch, capacity, kv_heads, dim, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = _normal(gen, batch, 4 * kv_heads, dim, dtype=dtype)
    k, v = (_normal(gen, batch, capacity, kv_heads, dim, dtype=dtype) for _ in range(2))
    return gen, q, k, v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("capacity", [100, 5000])       # in one piece, in pieces that are joined
def test_query_that_is_nan_on_a_cache(capacity, dtype):
    from rode_b200.rode_attention import rode_window_attention_step

    _, q, k, v = _caches(3, capacity, 2, 64, dtype, 30)
    lengths = torch.tensor([capacity, capacity - 3, 17], dtype=torch.int32, device="cuda")
    clean = rode_window_attention_step(q, k, v, lengths, capacity)
    q[1] = NAN
    got = rode_window_attention_step(q, k, v, lengths, capacity)
    assert bool(got[1].isnan().all())
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


@pytest.mark.parametrize("dtype", TYPES)
def test_keys_that_are_nan_on_a_cache(dtype):
    """A stretch of keys longer than a piece."""
    from rode_b200.rode_attention import rode_window_attention_step

    _, q, k, v = _caches(2, 5000, 2, 64, dtype, 31)
    lengths = torch.tensor([5000, 5000], dtype=torch.int32, device="cuda")
    clean = rode_window_attention_step(q, k, v, lengths, 5000)
    k[0, 1000:2500] = NAN
    got = rode_window_attention_step(q, k, v, lengths, 5000)
    assert bool(got[0].isnan().all()) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,prefix,capacity", [(3, 200, 50), (3, 4000, 50), (3, 300, 3000)])
def test_query_that_is_nan_behind_a_prefix(batch, prefix, capacity, dim, dtype):
    from rode_b200.rode_attention import rode_shared_prefix_attention

    gen, q, k, v = _caches(batch, capacity, 2, dim, dtype, 32)
    pk, pv = (_normal(gen, prefix, 2, dim, dtype=dtype) for _ in range(2))
    lengths = torch.tensor([capacity, capacity // 2, 0], dtype=torch.int32, device="cuda")
    clean = rode_shared_prefix_attention(q, pk, pv, k, v, lengths)
    for bad in (1, 2):
        x = q.clone()
        x[bad] = NAN
        got = rode_shared_prefix_attention(x, pk, pv, k, v, lengths)
        assert bool(got[bad].isnan().all())
        others = [b for b in range(batch) if b != bad]
        assert torch.equal(got[others], clean[others])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_query_that_is_nan_in_a_prompt(dim, dtype):
    """Its result and the logarithm of its sum are NaN (not what says "sees no key"); the other queries do not notice."""
    from test_gpu_attention_c_abi import prompt

    gen = torch.Generator(device="cuda").manual_seed(33)
    q, dout = (_normal(gen, 300, 4, dim, dtype=dtype) for _ in range(2))
    k, v = (_normal(gen, 300, 2, dim, dtype=dtype) for _ in range(2))
    clean = prompt(q, k, v, dout, 90, 4, dim ** -0.5)
    q[200] = NAN
    got = prompt(q, k, v, dout, 90, 4, dim ** -0.5)
    others = [i for i in range(300) if i != 200]
    assert bool(got["out"][200].isnan().all()) and bool(got["lse"][:, 200].isnan().all()) and bool(got["dq"][200].isnan().all())
    for x, y in ((got["out"], clean["out"]), (got["lse"].t(), clean["lse"].t()), (got["dq"], clean["dq"])):
        assert torch.equal(x[others], y[others])
    for name in ("dk", "dv"):                           # of the keys that it sees
        assert bool(got[name][111:201].isnan().all()) and bool(got[name][:4].isnan().all())
    for keys in (slice(4, 111), slice(201, 300)):
        assert torch.equal(got["dv"][keys], clean["dv"][keys])
