"""Window-and-sinks attention over packed sequences, forward and backward, against the definition in 64 bits."""
import itertools

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


def _offsets(lens, start=0):
    return torch.tensor([start, *(start + x for x in itertools.accumulate(lens))], dtype=torch.int32, device="cuda")


def _normal(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _make(q_lens, k_lens, heads, kv_heads, dim, dtype, seed=0, more_q=0, more_k=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = _normal(gen, sum(q_lens) + more_q, heads, dim, dtype=dtype)
    k, v = (_normal(gen, sum(k_lens) + more_k, kv_heads, dim, dtype=dtype) for _ in range(2))
    return q, k, v, _normal(gen, *q.shape, dtype=dtype)


def _run(q, k, v, dout, window, sinks, **kw):
    from rode_b200.rode_attention import rode_window_attention

    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = rode_window_attention(*leaves, window, sinks, **kw)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        assert torch.equal(rode_window_attention(q, k, v, window, sinks, **kw), out)
    return {"out": out.detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def _check(got, want):
    for name, pair in want.items():
        R.check(got[name], pair, name)


CASES = [  # queries, keys, window, sinks
    ([1], [1], 1, 0),
    ([1], [300], 64, 4),
    ([37], [37], 16, 2),
    ([64], [64], 1000, 0),
    ([65, 1, 0, 129, 63], None, 20, 3),
    ([128, 256, 2], None, 128, 0),
    ([300], [300], 1, 5),
    ([301], [301], 127, 130),
    ([40, 7], [200, 7], 50, 10),
    ([90, 5, 4], [20, 0, 4], 12, 1),       # more queries than keys: the first ones see nothing
    ([513], [513], 200, 64),
    ([150, 410], [700, 1000], 333, 1),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", CASES)
def test_lengths_and_masks(case, dim, dtype):
    q_lens, k_lens, window, sinks = case
    k_lens = k_lens or q_lens
    q, k, v, dout = _make(q_lens, k_lens, 4, 2, dim, dtype)
    want = R.packed(q, k, v, q_lens, k_lens, window, sinks, dim ** -0.5, dout)
    kw = {} if len(q_lens) == 1 else {"q_offsets": _offsets(q_lens), "k_offsets": _offsets(k_lens) if k_lens != q_lens else None}
    got = _run(q, k, v, dout, window, sinks, **kw)
    _check(got, want)
    again = _run(q, k, v, dout, window, sinks, **kw)  # same bits whatever the order of the thread blocks
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [([5000], [5000], 100, 5), ([30, 6500], None, 700, 1), ([4200, 3], [4500, 3], 300, 128),
                                  ([2100, 2700, 0], [2100, 2600, 5], 1, 2), ([4000], [4000], 50, 129)])
@pytest.mark.parametrize("dim", [64, 120])
def test_sinks_seen_from_far(case, dim, dtype):
    """Long sequences, whose first keys get gradients from queries far behind their window."""
    q_lens, k_lens, window, sinks = case
    k_lens = k_lens or q_lens
    q, k, v, dout = _make(q_lens, k_lens, 2, 1, dim, dtype, seed=12)
    k[:3] *= 2
    want = R.packed(q, k, v, q_lens, k_lens, window, sinks, dim ** -0.5, dout)
    kw = {} if len(q_lens) == 1 else {"q_offsets": _offsets(q_lens), "k_offsets": _offsets(k_lens) if k_lens != q_lens else None}
    got = _run(q, k, v, dout, window, sinks, **kw)
    _check(got, want)
    again = _run(q, k, v, dout, window, sinks, **kw)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 4), (3, 1, 20), (6, 3, 40), (8, 1, 80), (5, 5, 96), (4, 2, 100), (2, 2, 16),
                                                (16, 2, 120), (2, 1, 132), (4, 2, 256), (128, 1, 64), (130, 1, 64), (48, 1, 128),
                                                (65, 1, 88)])
def test_head_layouts(heads, kv_heads, dim, dtype):
    q_lens = [70, 200]
    q, k, v, dout = _make(q_lens, q_lens, heads, kv_heads, dim, dtype, seed=1)
    want = R.packed(q, k, v, q_lens, q_lens, 90, 7, 0.3, dout)
    _check(_run(q, k, v, dout, 90, 7, q_offsets=_offsets(q_lens), scale=0.3), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["fused", "heads_first", "dim_first", "odd_base", "repeated_heads", "gaps"])
def test_strides(layout, dtype):
    """Slices of one projection, other orders, operands that have to be copied first."""
    rows, heads, kv_heads, dim = 200, 4, 2, 64
    q, k, v, dout = _make([rows], [rows], heads, kv_heads, dim, dtype, seed=2)
    if layout == "fused":
        fused = torch.cat([q, k, v], 1)
        q, k, v = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
    elif layout == "heads_first":
        q, k, v, dout = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, dout))
    elif layout == "dim_first":
        q, k, v, dout = (x.permute(2, 0, 1).contiguous().permute(1, 2, 0) for x in (q, k, v, dout))
    elif layout == "odd_base":
        q, k, v, dout = (torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(x.shape) for x in (q, k, v, dout))
    elif layout == "repeated_heads":
        k, v = (x[:, :1].expand(-1, kv_heads, -1) for x in (k, v))
        dout = dout[:, :1].expand(-1, heads, -1)
    else:
        q, k, v, dout = (torch.cat([x, x], 2)[..., :dim] for x in (q, k, v, dout))
    want = R.packed(q, k, v, [rows], [rows], 60, 4, dim ** -0.5, dout)
    _check(_run(q, k, v, dout, 60, 4), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_do_not_see_each_other(dim, dtype):
    """Rows in front of the first and behind the last sequence are NaN, and one sequence is: the others do not notice."""
    q_lens, k_lens = [50, 130, 70], [80, 130, 71]
    q, k, v, dout = _make(q_lens, k_lens, 4, 2, dim, dtype, seed=3, more_q=20 + 150, more_k=9 + 140)
    for x, start, lens in ((q, 20, q_lens), (dout, 20, q_lens), (k, 9, k_lens), (v, 9, k_lens)):
        x[:start] = float("nan")
        x[start + sum(lens):] = float("inf")
    clean = R.packed(q, k, v, q_lens, k_lens, 40, 5, dim ** -0.5, dout, 20, 9)
    for x, start, lens in ((k, 9, k_lens), (v, 9, k_lens), (q, 20, q_lens), (dout, 20, q_lens)):
        x[start + lens[0]:start + lens[0] + lens[1]] = float("nan")
    got = _run_nan(q, k, v, dout, 40, 5, q_offsets=_offsets(q_lens, 20), k_offsets=_offsets(k_lens, 9))
    for name, (value, bound) in clean.items():
        start, lens = (20, q_lens) if name in ("out", "dq") else (9, k_lens)
        a, b = start + lens[0], start + lens[0] + lens[1]
        assert bool(got[name][a:b].isnan().any())
        R.check(got[name][:a], (value[:a], bound[:a]), name)
        R.check(got[name][b:], (value[b:], bound[b:]), name)


def _run_nan(q, k, v, dout, window, sinks, **kw):
    from rode_b200.rode_attention import rode_window_attention

    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = rode_window_attention(*leaves, window, sinks, **kw)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, dout))))


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_far_apart(dtype):
    """Scores of many hundreds, growing and falling along the keys: the running maximum moves at every tile."""
    rows, dim = 400, 64
    q, k, v, dout = _make([rows], [rows], 2, 1, dim, dtype, seed=4)
    k = (k * torch.linspace(0.1, 12.0, rows, device="cuda")[:, None, None]).to(dtype)
    q[::2] *= 8
    for flip in (False, True):
        kk = k.flip(0).contiguous() if flip else k
        want = R.packed(q, kk, v, [rows], [rows], 1000, 0, 1.0, dout)
        _check(_run(q, kk, v, dout, 1000, 0, scale=1.0), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_operands(dtype):
    from rode_b200.rode_attention import rode_window_attention

    q, k, v, dout = _make([5], [0], 4, 2, 64, dtype)
    got = _run(q, k, v, dout, 3, 1)
    assert not got["out"].any() and not got["dq"].any() and got["dk"].shape == (0, 2, 64)
    q, k, v, dout = _make([0], [5], 4, 2, 64, dtype)
    got = _run(q, k, v, dout, 3, 1)
    assert got["out"].shape == (0, 4, 64) and not got["dk"].any() and not got["dv"].any()
    q, k, v, dout = _make([6], [6], 4, 2, 64, dtype)
    out = rode_window_attention(q, k, v, 3, 1, q_offsets=_offsets([]))      # no sequence at all
    assert not out.any()


def test_gradient_against_differences():
    """Directional derivatives of sum(out * dout) by central differences of the fp32 kernel's own results, with steps of 2^-5: their
    error is h^2 / 6 times a third derivative (taken from differences of twice the step) and the results' rounding over h."""
    q_lens, h = [70, 30], 2.0 ** -5
    q, k, v, dout = _make(q_lens, q_lens, 4, 2, 64, torch.float32, seed=5)
    offsets = _offsets(q_lens)
    got = _run(q, k, v, dout, 25, 3, q_offsets=offsets)
    from rode_b200.rode_attention import rode_window_attention as f

    gen = torch.Generator(device="cuda").manual_seed(6)
    for name, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        x = [q, k, v]
        u = _normal(gen, *x[i].shape, dtype=torch.float32)

        def value(step):
            y = list(x)
            y[i] = x[i] + step * u
            return float((f(*y, 25, 3, q_offsets=offsets).double() * dout).sum())

        want = float((got[name].double() * u).sum())
        near, far = (value(h) - value(-h)) / (2 * h), (value(2 * h) - value(-2 * h)) / (4 * h)
        rounding = 2.0 ** -22 * float((got["out"].abs() * dout.abs()).sum()) * 4 / h
        assert abs(near - want) <= abs(far - near) + rounding, (name, near, far, want, rounding)


def test_only_some_gradients():
    from rode_b200.rode_attention import rode_window_attention

    q, k, v, dout = _make([100], [100], 4, 2, 64, torch.bfloat16, seed=7)
    full = _run(q, k, v, dout, 30, 2)
    a = q.clone().requires_grad_()
    rode_window_attention(a, k, v, 30, 2).backward(dout)
    assert torch.equal(a.grad, full["dq"])
    b = v.clone().requires_grad_()
    rode_window_attention(q, k, b, 30, 2).backward(dout)
    assert torch.equal(b.grad, full["dv"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30])
def test_scales(scale, dtype):
    """Scores turned round (the smallest counts most) and all alike."""
    q_lens = [100, 30]
    q, k, v, dout = _make(q_lens, q_lens, 4, 2, 64, dtype, seed=14)
    want = R.packed(q, k, v, q_lens, q_lens, 40, 3, scale, dout)
    _check(_run(q, k, v, dout, 40, 3, q_offsets=_offsets(q_lens), scale=scale), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_no_sequence_stay_as_they_were(dtype):
    """The C entry points with clear = 0: results in front of the first and behind the last sequence keep what they held."""
    import ctypes

    from rode_b200 import capi

    lib, kind = capi.load(), {torch.float32: capi.RODE_F32, torch.float16: capi.RODE_F16, torch.bfloat16: capi.RODE_BF16}[dtype]
    q_lens, heads, kv_heads, dim = [50, 90], 4, 2, 64
    q, k, v, dout = _make(q_lens, q_lens, heads, kv_heads, dim, dtype, seed=15, more_q=37, more_k=37)
    rows = q.shape[0]
    want = R.packed(q, k, v, q_lens, q_lens, 30, 2, 0.1, dout, 20, 20)
    offsets = _offsets(q_lens, 20)
    out, dq, rest = (torch.full_like(q, 7.0) for _ in range(3))
    dk, dv = (torch.full_like(k, 7.0) for _ in range(2))
    lse = torch.empty(heads, rows, device="cuda")
    need = ctypes.c_size_t(0)
    capi.check(lib.rode_window_attention_backward_workspace_bytes(kind, 2, rows, rows, heads, kv_heads, dim, 30, 2, ctypes.byref(need)))
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    h = lambda x: ctypes.byref(capi.Heads(x.data_ptr(), 0, x.stride(0), x.stride(1)))
    stream = torch.cuda.current_stream().cuda_stream or None
    common = (kind, 2, offsets.data_ptr(), offsets.data_ptr(), rows, rows, heads, kv_heads, dim, 30, 2, 0.1, 0, h(q), h(k), h(v))
    capi.check(lib.rode_window_attention(*common, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), stream))
    capi.check(lib.rode_window_attention_backward(*common, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), h(dout), dq.data_ptr(), dk.data_ptr(),
                                                  dv.data_ptr(), ws.data_ptr(), need.value, stream))
    for name, x in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert bool((x[:20] == 7).all()) and bool((x[160:] == 7).all()), name
        R.check(x[20:160], tuple(y[20:160] for y in want[name]), name)
    assert bool((rest[:20] == 7).all()) and bool((rest[160:] == 7).all())
    if dtype != torch.float32:  # the rest: at most half a step of the result
        step = torch.finfo(dtype).eps * out[20:160].double().abs() + 2.0 ** -24
        assert bool((rest[20:160].double().abs() <= step).all()) and bool(rest[20:160].any())
    else:
        assert bool((rest == 7).all())
    capi.check(lib.rode_window_attention_backward(*common, out.data_ptr(), None, lse.data_ptr(), h(dout), dq.data_ptr(), dk.data_ptr(),
                                                  dv.data_ptr(), ws.data_ptr(), need.value, stream))
    R.check(dq[20:160], tuple(y[20:160] for y in want["dq"]), "dq without the rest")


def test_second_derivative_is_refused():
    from rode_b200.rode_attention import rode_window_attention

    q, k, v, dout = _make([50], [50], 4, 2, 64, torch.float32, seed=13)
    full = _run(q, k, v, dout, 20, 2)
    leaf = q.clone().requires_grad_()
    grad, = torch.autograd.grad(rode_window_attention(leaf, k, v, 20, 2), leaf, dout, create_graph=True)
    assert torch.equal(grad.detach(), full["dq"])
    with pytest.raises(RuntimeError, match="once"):
        grad.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_on_another_stream(dtype):
    from rode_b200.rode_attention import rode_window_attention

    q_lens = [200, 90]
    q, k, v, dout = _make(q_lens, q_lens, 4, 2, 64, dtype, seed=8)
    offsets = _offsets(q_lens)
    want = _run(q, k, v, dout, 50, 4, q_offsets=offsets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, dout, 50, 4, q_offsets=offsets)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rode_window_attention(*leaves, 50, 4, q_offsets=offsets)
        grads = torch.autograd.grad(out, leaves, dout)
    # lengths are read on the device: other ones, and other values, at every replay
    for lens, factor in (([200, 90], 1.0), ([10, 280], 0.5)):
        offsets.copy_(_offsets(lens))
        with torch.no_grad():
            for x, y in zip(leaves, (q, k, v)):
                x.copy_(y * factor)
        graph.replay()
        fresh = _run(q * factor, k * factor, v * factor, dout, 50, 4, q_offsets=offsets)
        for x, n in zip((out, *grads), ("out", "dq", "dk", "dv")):
            assert torch.equal(x, fresh[n]), n


def test_offsets_that_lie():
    """Entries out of range or out of order give some values, but nothing outside the operands is touched."""
    from rode_b200.rode_attention import rode_window_attention

    q, k, v, dout = _make([300], [300], 4, 2, 64, torch.bfloat16, seed=9)
    for bad in ([0, 400, 500], [-7, 100, 300], [200, 100, 300], [0, 2**31 - 1, -2**31], [300, 300, 0]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        for dtype in (torch.bfloat16, torch.float32):
            leaves = [x.to(dtype).requires_grad_() for x in (q, k, v)]
            out = rode_window_attention(*leaves, 30, 2, q_offsets=offsets)
            torch.autograd.grad(out, leaves, dout.to(dtype))
    torch.cuda.synchronize()


def test_refusals():
    from rode_b200.rode_attention import rode_window_attention as f

    q, k, v, _ = _make([10], [10], 4, 2, 64, torch.float32)
    ints = _offsets([10])
    for bad, error in [((q, k[:9], v, 3), ValueError), ((q, k, v[:9], 3), ValueError), ((q, k, v, 0), ValueError),
                       ((q, k, v, 3, -1), ValueError), ((q[:, :3], k, v, 3), ValueError), ((q, k[..., :32], v[..., :32], 3), ValueError),
                       ((q.double(), k.double(), v.double(), 3), TypeError), ((q, k.half(), v, 3), TypeError),
                       ((q, k, v, 3, 0, ints.long()), TypeError), ((q, k, v, 3, 0, None, ints), ValueError),
                       ((q, k, v, 3, 0, ints, _offsets([5, 5])), ValueError), ((q, k, v, 3, 0, ints.cpu()), ValueError),
                       ((q.cpu(), k.cpu(), v.cpu(), 3), ValueError), ((q[0], k, v, 3), ValueError),
                       ((q[..., :6], k[..., :6], v[..., :6], 3), ValueError), ((q, k, v, 3, 0, None, None, float("inf")), ValueError)]:
        with pytest.raises(error):
            f(*bad)
    big = torch.zeros(4, 2, 260, device="cuda")
    with pytest.raises(ValueError, match="multiple of 4, at most 256"):
        f(big, big, big, 3)


def test_from_a_thread_without_a_context():
    """A host thread whose first call of CUDA is ours (its memory comes from what the allocator holds already)."""
    import threading

    from rode_b200.rode_attention import rode_window_attention

    q, k, v, dout = _make([100], [100], 4, 2, 64, torch.bfloat16, seed=11)
    want = _run(q, k, v, dout, 30, 2)
    got = []

    def work():
        got.append(rode_window_attention(q, k, v, 30, 2))

    for _ in range(2):
        t = threading.Thread(target=work)
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert len(got) == 2 and all(torch.equal(x, want["out"]) for x in got)


def test_two_host_threads_at_once():
    """Calls from two host threads, each on a stream of its own."""
    import threading

    q_lens = [300, 200]
    sets = [_make(q_lens, q_lens, 4, 2, dim, torch.bfloat16, seed=16 + dim) for dim in (64, 128)]
    offsets = _offsets(q_lens)
    want = [_run(*x, 100, 4, q_offsets=offsets) for x in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _run(*sets[i], 100, 4, q_offsets=offsets)
                torch.cuda.current_stream().synchronize()
                bad.extend(n for n in got if not torch.equal(got[n], want[i][n]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
