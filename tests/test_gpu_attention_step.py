"""Single tokens: window-and-sinks attention against a cache, and behind a prefix that a batch shares, against 64 bits."""
import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_given_up():
    """No kernel's warps gave up waiting for one another."""
    import ctypes

    from rode_b200 import capi

    yield
    failed = ctypes.c_int(-1)
    capi.check(capi.load().rode_attention_waits_failed(ctypes.byref(failed)))
    assert failed.value == 0


TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _normal(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _caches(gen, batch, capacity, kv_heads, dim, dtype, layout):
    res = []
    for _ in range(2):
        x = _normal(gen, batch, capacity, kv_heads, dim, dtype=dtype)
        if layout == "heads_first":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "tokens_first":
            x = x.transpose(0, 1).contiguous().transpose(0, 1)
        elif layout == "gaps":
            x = torch.cat([x, x], 3)[..., :dim]
        elif layout == "odd_rows":                      # strides that are multiples of 4 elements, not of 16 bytes
            x = torch.cat([x, x], 3)[..., :dim + 4].contiguous()[..., :dim]
        res.append(x)
    return res


def _want(q, k, v, lengths, seen_of, scale, prefix=None):
    """seen_of(n): the keys that a request with n tokens sees."""
    value, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        at = torch.tensor(seen_of(min(max(n, 0), k.shape[1])), dtype=torch.long, device="cuda")
        kk, vv = k[b][at], v[b][at]
        if prefix is not None:
            kk, vv = torch.cat([prefix[0], kk]), torch.cat([prefix[1], vv])
        one = R.one_sequence(q[b:b + 1], kk, vv, torch.ones(1, kk.shape[0], dtype=torch.bool, device="cuda"), scale)["out"]
        value[b], bound[b] = one[0][0], one[1][0]
    return value, bound


def _keys(window, sinks):
    return lambda n: [j for j in range(n) if n - 1 - j < window or j < sinks]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["rows", "heads_first", "tokens_first", "gaps", "odd_rows"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (8, 8, 128), (16, 1, 128), (12, 4, 96), (33, 3, 64), (130, 1, 64), (2, 1, 20), (4, 2, 256)])
def test_step(heads, kv_heads, dim, layout, dtype):
    gen = torch.Generator(device="cuda").manual_seed(1)
    capacity, lengths = 300, [0, 1, 2, 31, 32, 33, 100, 299, 300, 64, 7, 250]
    q = _normal(gen, len(lengths), heads, dim, dtype=dtype)
    k, v = _caches(gen, len(lengths), capacity, kv_heads, dim, dtype, layout)
    ints = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    from rode_b200.rode_attention import rode_window_attention_step

    for window, sinks in ((1, 0), (16, 4), (1000, 0), (100, 150), (33, 1)):
        want = _want(q, k, v, lengths, _keys(window, sinks), dim ** -0.5)
        at = torch.arange(capacity, device="cuda")
        back = ints[:, None] - 1 - at
        hidden = (back < 0) | ((back >= window) & (at >= sinks))    # what is not visible may hold anything
        keep = k[hidden], v[hidden]
        k[hidden], v[hidden] = float("nan"), float("inf")
        got = rode_window_attention_step(q, k, v, ints, window, sinks)
        k[hidden], v[hidden] = keep
        R.check(got, want, (window, sinks))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,heads,kv_heads,dim,capacity", [(1, 8, 2, 64, 5000), (2, 4, 4, 128, 20011), (1, 16, 1, 128, 40000), (3, 5, 1, 36, 3000)])
def test_step_over_long_caches(batch, heads, kv_heads, dim, capacity, dtype):
    """Few rows and many keys: the keys are cut into parts, some of which are empty."""
    from rode_b200.rode_attention import rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(2)
    q = _normal(gen, batch, heads, dim, dtype=dtype)
    k, v = _caches(gen, batch, capacity, kv_heads, dim, dtype, "rows")
    for lengths in ([capacity, 17, 0], [capacity // 2 + 1, capacity - 1, 1]):
        lengths = lengths[:batch]
        ints = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        for window, sinks in ((capacity, 0), (capacity // 3, 1000), (5, 5)):
            want = _want(q, k, v, lengths, _keys(window, sinks), dim ** -0.5)
            got = rode_window_attention_step(q, k, v, ints, window, sinks)
            R.check(got, want, (window, sinks))
            assert torch.equal(got, rode_window_attention_step(q, k, v, ints, window, sinks))


def test_step_far_into_a_large_cache():
    """Rows whose offsets pass 32 bits, in elements and in bytes."""
    from rode_b200.rode_attention import rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(3)
    batch, capacity, kv_heads, dim = 3, 70000, 32, 128          # 8.6e8 elements per tensor and row stride of 2^22 bytes per 1024 rows
    k = torch.zeros(batch * 3, capacity, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    k = k[::3]                                                  # sequence stride 8.6e8 elements, the last one starts behind 2^31 bytes
    assert k.stride(0) * 2 * 2 > 2**31
    v = torch.zeros_like(k)
    lengths, window = [300, 70000, 69999], 200
    for b, n in enumerate(lengths):
        k[b, max(0, n - window):n] = _normal(gen, min(n, window), kv_heads, dim, dtype=torch.bfloat16)
        v[b, max(0, n - window):n] = _normal(gen, min(n, window), kv_heads, dim, dtype=torch.bfloat16)
    q = _normal(gen, batch, kv_heads, dim, dtype=torch.bfloat16)
    want = _want(q, k, v, lengths, _keys(window, 0), dim ** -0.5)
    got = rode_window_attention_step(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"), window)
    R.check(got, want)


def test_lengths_that_lie():
    """Lengths out of range are taken as 0 and as the capacity."""
    from rode_b200.rode_attention import rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(4)
    q = _normal(gen, 4, 4, 64, dtype=torch.float16)
    k, v = _caches(gen, 4, 50, 2, 64, torch.float16, "rows")
    call = lambda x: rode_window_attention_step(q, k, v, torch.tensor(x, dtype=torch.int32, device="cuda"), 20, 2)
    assert torch.equal(call([-1, 51, 2**31 - 1, -2**31]), call([0, 50, 50, 0]))
    assert not call([0, 0, 0, 0]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,prefix,heads,kv_heads,dim", [(1, 1, 4, 2, 64), (3, 777, 8, 2, 64), (40, 300, 8, 2, 128), (5, 0, 4, 4, 64),
                                                             (130, 129, 4, 4, 96), (2, 5000, 12, 1, 128), (7, 100, 6, 2, 20), (3, 130, 2, 1, 256),
                                                             (17, 2500, 24, 3, 72), (2, 400, 130, 1, 64), (3, 1000, 128, 1, 128)])
def test_shared_prefix(batch, prefix, heads, kv_heads, dim, dtype):
    from rode_b200.rode_attention import rode_shared_prefix_attention

    gen = torch.Generator(device="cuda").manual_seed(5)
    capacity = 90
    q = _normal(gen, batch, heads, dim, dtype=dtype)
    pk, pv = (_normal(gen, prefix, kv_heads, dim, dtype=dtype) for _ in range(2))
    k, v = _caches(gen, batch, capacity, kv_heads, dim, dtype, "heads_first")
    lengths = [(37 * b) % (capacity + 1) for b in range(batch)]
    ints = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = _want(q, k, v, lengths, lambda n: list(range(n)), dim ** -0.5, (pk, pv))
    for b, n in enumerate(lengths):
        k[b, n:], v[b, n:] = float("nan"), float("nan")
    got = rode_shared_prefix_attention(q, pk, pv, k, v, ints)
    R.check(got, want)
    assert torch.equal(got, rode_shared_prefix_attention(q, pk, pv, k, v, ints))
    # the prefix as slices of a larger tensor, whose rows behind it are NaN
    big = torch.full((prefix + 200, 2 * kv_heads, dim), float("nan"), dtype=dtype, device="cuda")
    big[:prefix, :kv_heads], big[:prefix, kv_heads:] = pk, pv
    assert torch.equal(got, rode_shared_prefix_attention(q, big[:prefix, :kv_heads], big[:prefix, kv_heads:], k, v, ints))


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_then_tokens_then_samples(dtype):
    """As a server runs them: a prompt in two pieces, tokens one by one on the cache, then several samples that share the cache as
    their prefix.  Each step gives what the whole sequence at once gives."""
    from rode_b200.rode_attention import rode_shared_prefix_attention, rode_window_attention, rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(6)
    heads, kv_heads, dim, total, prompt, window, sinks = 8, 2, 64, 200, 190, 70, 4
    q = _normal(gen, total, heads, dim, dtype=dtype)
    k, v = (_normal(gen, total, kv_heads, dim, dtype=dtype) for _ in range(2))
    want = R.packed(q, k, v, [total], [total], window, sinks, dim ** -0.5)["out"]
    first = rode_window_attention(q[:100], k[:100], v[:100], window, sinks)
    second = rode_window_attention(q[100:prompt], k[:prompt], v[:prompt], window, sinks)
    k_cache, v_cache = (torch.full((1, 256, kv_heads, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    k_cache[0, :prompt], v_cache[0, :prompt] = k[:prompt], v[:prompt]
    length = torch.full((1,), prompt, dtype=torch.int32, device="cuda")
    tokens = []
    for i in range(prompt, total):
        k_cache[0, i], v_cache[0, i] = k[i], v[i]
        length += 1
        tokens.append(rode_window_attention_step(q[i:i + 1], k_cache, v_cache, length, window, sinks))
    R.check(torch.cat([first, second, *tokens]), want)
    samples = 5
    sq = _normal(gen, samples, heads, dim, dtype=dtype)
    sk, sv = _caches(gen, samples, 8, kv_heads, dim, dtype, "rows")
    lengths = [1, 2, 3, 8, 0]
    ints = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = rode_shared_prefix_attention(sq, k_cache[0, :total], v_cache[0, :total], sk, sv, ints)
    R.check(got, _want(sq, sk, sv, lengths, lambda n: list(range(n)), dim ** -0.5, (k, v)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_scales(scale, dtype):
    from rode_b200.rode_attention import rode_shared_prefix_attention, rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(9)
    lengths = [0, 5, 400]
    q = _normal(gen, 3, 4, 64, dtype=dtype)
    k, v = _caches(gen, 3, 400, 2, 64, dtype, "rows")
    pk, pv = (_normal(gen, 300, 2, 64, dtype=dtype) for _ in range(2))
    ints = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    R.check(rode_window_attention_step(q, k, v, ints, 90, 3, scale=scale), _want(q, k, v, lengths, _keys(90, 3), scale))
    R.check(rode_shared_prefix_attention(q, pk, pv, k, v, ints, scale=scale),
            _want(q, k, v, lengths, lambda n: list(range(n)), scale, (pk, pv)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,capacity", [(700, 300), (150, 3000), (129, 1000)])
def test_ragged_batches(batch, capacity, dtype):
    """Many requests, some without a token, whose blocks are dealt out in equal shares across their borders."""
    from rode_b200.rode_attention import rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(10)
    lengths = [(b * 7919) % (capacity + 1) if b % 5 else 0 for b in range(batch)]
    q = _normal(gen, batch, 6, 64, dtype=dtype)
    k, v = _caches(gen, batch, capacity, 2, 64, dtype, "rows")
    ints = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for window, sinks in ((capacity, 0), (200, 20)):
        got = rode_window_attention_step(q, k, v, ints, window, sinks)
        R.check(got, _want(q, k, v, lengths, _keys(window, sinks), 0.125), (window, sinks))
    short = torch.zeros_like(ints)
    assert not rode_window_attention_step(q, k, v, short, capacity).any()


def test_captured_replayed_and_on_two_streams():
    from rode_b200.rode_attention import rode_shared_prefix_attention, rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(7)
    q = _normal(gen, 2, 8, 128, dtype=torch.bfloat16)
    k, v = _caches(gen, 2, 4000, 2, 128, torch.bfloat16, "rows")
    pk, pv = (_normal(gen, 3000, 2, 128, dtype=torch.bfloat16) for _ in range(2))
    lengths = torch.tensor([4000, 1234], dtype=torch.int32, device="cuda")
    step = lambda: rode_window_attention_step(q, k, v, lengths, 3000, 4)
    share = lambda: rode_shared_prefix_attention(q, pk, pv, k, v, lengths)
    want = step(), share()
    graphs = []
    for f in (step, share):                 # two graphs, each with workspaces of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for new in ([4000, 1234], [17, 0]):
        lengths.copy_(torch.tensor(new, dtype=torch.int32))
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        fresh = step(), share()
        assert all(torch.equal(x[1], y) for x, y in zip(graphs, fresh))
    lengths.copy_(torch.tensor([4000, 1234], dtype=torch.int32))
    torch.cuda.synchronize()
    got = []
    for f, s in zip((step, share), streams):
        with torch.cuda.stream(s):
            got.append(f())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    from rode_b200.rode_attention import rode_shared_prefix_attention, rode_window_attention_step

    gen = torch.Generator(device="cuda").manual_seed(8)
    q = _normal(gen, 2, 4, 64, dtype=torch.float16)
    k, v = _caches(gen, 2, 10, 2, 64, torch.float16, "rows")
    n = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    for bad, error in [((q, k, v, n, 0), ValueError), ((q, k, v, n, 3, -1), ValueError), ((q, k, v[:, :9], n, 3), ValueError),
                       ((q, k, v, n[:1], 3), ValueError), ((q, k, v, n.long(), 3), TypeError), ((q, k.float(), v, n, 3), TypeError),
                       ((q, k, v, n.cpu(), 3), ValueError), ((q[:, :3], k, v, n, 3), ValueError),
                       ((q, k.transpose(2, 3).contiguous().transpose(2, 3), v, n, 3), ValueError),
                       ((q.cpu(), k.cpu(), v.cpu(), n.cpu(), 3), ValueError), ((q[0], k, v, n, 3), ValueError)]:
        with pytest.raises(error):
            rode_window_attention_step(*bad)
    p = k[0]
    for bad, error in [((q, p, p[:9], k, v, n), ValueError), ((q, p[:, :1], p[:, :1], k, v, n), ValueError),
                       ((q, p.float(), p.float(), k, v, n), TypeError), ((q, p[..., :32], p[..., :32], k, v, n), ValueError)]:
        with pytest.raises(error):
            rode_shared_prefix_attention(*bad)
    empty = rode_window_attention_step(q[:0], k[:0], v[:0], n[:0], 3)
    assert empty.shape == (0, 4, 64)
