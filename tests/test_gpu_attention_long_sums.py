"""Single precision over many keys: a sum's error does not grow with every key.

All scores are 0 and all weights 1, so that a result is the plain sum of n values divided by n.  The values are 1 + 2^-11 + 2^-20: from 2^13 keys
on, one addition behind the other rounds each of them up by 2^-11 - 2^-20, 2^-12 of the result and more.  Sums by tiles of 32 or 64 keys, added up behind one another, are off by
at most (64 + n / 32) u of themselves (u = 2^-24, every addition by half a step), the division and the sum of the weights by a few u."""
import pytest
import torch

pytestmark = pytest.mark.gpu

N = 16384
VALUE = 1 + 2.0 ** -11 + 2.0 ** -20
BOUND = (64 + N / 32 + 32) * 2.0 ** -24


def _check(out):
    err = float((out.double() / VALUE - 1).abs().max())
    assert err <= BOUND, (err, BOUND)


def test_single_tokens():
    from rode_b200.rode_attention import rode_window_attention_step

    batch, kv_heads, dim = 37, 8, 4                      # as many rows as thread blocks, each with all of a row's keys
    q = torch.zeros(batch, kv_heads, dim, device="cuda")
    k, v = (torch.full((batch, N, kv_heads, dim), x, device="cuda") for x in (1.0, VALUE))
    _check(rode_window_attention_step(q, k, v, torch.full((batch,), N, dtype=torch.int32, device="cuda"), N))


@pytest.mark.parametrize("dim", [4, 128, 256])
def test_shared_prefix(dim):
    from rode_b200.rode_attention import rode_shared_prefix_attention

    kv_heads = 300                                       # the prefix is not cut into parts
    q = torch.zeros(1, kv_heads, dim, device="cuda")
    k, v = (torch.full((N, 1, dim), x, device="cuda").expand(N, kv_heads, dim).contiguous() for x in (1.0, VALUE))
    empty = torch.empty(1, 0, kv_heads, dim, device="cuda")
    _check(rode_shared_prefix_attention(q, k, v, empty, empty, torch.zeros(1, dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt(dim):
    from rode_b200.rode_attention import rode_window_attention

    q = torch.zeros(3, 1, dim, device="cuda")
    k, v = (torch.full((N, 1, dim), x, device="cuda") for x in (1.0, VALUE))
    _check(rode_window_attention(q, k, v, N)[2])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_gradient_of_a_key_that_all_queries_see(dim):
    """Query i sees keys 0 and i with weights of 1/2, query 0 one key with 1."""
    from rode_b200.rode_attention import rode_window_attention

    n = 2 * N
    q, k = torch.zeros(n, 1, dim, device="cuda"), torch.ones(n, 1, dim, device="cuda")
    v = torch.ones(n, 1, dim, device="cuda").requires_grad_()
    dv, = torch.autograd.grad(rode_window_attention(q, k, v, 1, 1), v, torch.full((n, 1, dim), VALUE, device="cuda"))
    err = float((dv[0].double() / (VALUE * (1 + (n - 1) / 2)) - 1).abs().max())
    assert err <= BOUND, (err, BOUND)
