"""More pieces of work than the persistent grids have thread blocks, several for each: long, short and empty ones in turn."""
import itertools

import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_given_up():
    """No kernel's warps gave up waiting for one another."""
    import ctypes

    from rode_b200 import capi

    yield
    failed = ctypes.c_int(-1)
    capi.check(capi.load().rode_attention_waits_failed(ctypes.byref(failed)))
    assert failed.value == 0


def _offsets(lens):
    return torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device="cuda")


def _normal(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _slots(q_lens, tile):
    return sum(q_lens) // tile + len(q_lens) + 2


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("heads,kv_heads,dim,window,sinks", [(8, 8, 64, 200, 3), (16, 8, 128, 90, 0), (24, 8, 64, 1000, 1), (32, 8, 128, 150, 130),
                                                             (56, 8, 96, 300, 4)])
def test_prompts(heads, kv_heads, dim, window, sinks, dtype):
    """Sequences without rows, of a part of a tile, of one tile, of two and of many, some behind a past, some with more queries than
    keys.  At least three pieces of work for each of 148 thread blocks, forward and backward."""
    from rode_b200.rode_attention import rode_window_attention

    q_lens = [0, 1, 257, 40, 700, 128, 0, 0, 65, 300, 129, 2, 0, 513, 31, 256, 7, 90, 0, 350] * 3
    past = [0, 500, 0, 130, 0, 3, 0, 50, 0, 200, -60, 0, 0, 0, 900, 0, -7, 0, 0, 128] * 3
    k_lens = [n + p for n, p in zip(q_lens, past)]
    per_tile = 128 // (heads // kv_heads)
    assert _slots(q_lens, 2 * per_tile) * kv_heads > 3 * 148
    gen = torch.Generator(device="cuda").manual_seed(40)
    q, dout = (_normal(gen, sum(q_lens), heads, dim, dtype=dtype) for _ in range(2))
    k, v = (_normal(gen, sum(k_lens), kv_heads, dim, dtype=dtype) for _ in range(2))
    want = R.packed(q, k, v, q_lens, k_lens, window, sinks, dim ** -0.5, dout)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    first = None
    for _ in range(2):
        out = rode_window_attention(*leaves, window, sinks, q_offsets=_offsets(q_lens), k_offsets=_offsets(k_lens))
        got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, dout))))
        for name, pair in want.items():
            R.check(got[name], pair, name)
        assert first is None or all(torch.equal(got[n], first[n]) for n in got)
        first = got


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("batch,heads,kv_heads,dim,prefix", [(3700, 32, 32, 64, 300), (500, 240, 15, 128, 700), (227, 512, 4, 64, 129),
                                                             (1180, 96, 32, 72, 520)])
def test_shared_prefixes(batch, heads, kv_heads, dim, prefix, dtype):
    """Requests enough for at least three pieces of work for each of 148 thread blocks, the last ones with one tile or a part of it."""
    from rode_b200.rode_attention import rode_shared_prefix_attention

    group = heads // kv_heads
    per_tile = 128 // group
    assert -(-batch // (2 * per_tile)) * kv_heads > 3 * 148
    gen = torch.Generator(device="cuda").manual_seed(41)
    capacity, scale = 24, dim ** -0.5
    q = _normal(gen, batch, heads, dim, dtype=dtype)
    pk, pv = (_normal(gen, prefix, kv_heads, dim, dtype=dtype) for _ in range(2))
    k, v = (_normal(gen, batch, capacity, kv_heads, dim, dtype=dtype) for _ in range(2))
    lengths = torch.tensor([(7 * b) % (capacity + 1) for b in range(batch)], dtype=torch.int32, device="cuda")
    got = rode_shared_prefix_attention(q, pk, pv, k, v, lengths)
    assert torch.equal(got, rode_shared_prefix_attention(q, pk, pv, k, v, lengths))
    # all requests at once, key head by key head; bounds as in attention_reference
    u, e = 2.0 ** -24, torch.finfo(dtype).eps / 2
    a = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    seen = torch.cat([torch.ones(batch, prefix, dtype=torch.bool, device="cuda"),
                      torch.arange(capacity, device="cuda")[None] < lengths[:, None]], 1)[:, None]
    for h in range(kv_heads):
        Q = q[:, h * group:(h + 1) * group].double()                                    # [batch, group, dim]
        own = k[:, :, h].double(), v[:, :, h].double()
        P, size = (torch.cat([x @ pk_.t(), x @ own_.transpose(1, 2)], 2) * scale
                   for x, pk_, own_ in ((Q, pk[:, h].double(), own[0]), (Q.abs(), pk[:, h].double().abs(), own[0].abs())))
        P = R.softmax(P, seen)
        c = 2 * (dim + 4) * u * size.masked_fill(~seen, 0.0).amax(-1, keepdim=True) + (prefix + capacity + 32) * u
        mean = lambda w, f: w[..., :prefix] @ f(pv[:, h].double()) + w[..., prefix:] @ f(own[1])
        O, size = mean(P, lambda x: x), mean(P, torch.abs)
        bound = e * O.abs() + (e + c) * size + a * mean(seen.double().expand_as(P), torch.abs) + a
        R.check(got[:, h * group:(h + 1) * group], (O, bound), h)
