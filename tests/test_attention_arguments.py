"""C entry points of the attention operators: refusals and sizes (no device), and the 64-bit reference of the GPU tests against
differences."""
import ctypes

import pytest
import torch

import attention_reference as R
from rode_b200 import capi

BAD, WS = capi.RODE_ERR_INVALID_ARGUMENT, capi.RODE_ERR_WORKSPACE


def _heads(data=256, batch=0, row=256, head=64):
    return ctypes.byref(capi.Heads(data, batch, row, head))


def _forward(lib, dtype=capi.RODE_F32, n_seq=1, qo=None, ko=None, q_rows=8, k_rows=8, heads=4, kv_heads=2, dim=64, window=4, sinks=0,
             scale=1.0, q=None, k=None, out=256, rest=None):
    return lib.rode_window_attention(dtype, n_seq, qo, ko, q_rows, k_rows, heads, kv_heads, dim, window, sinks, scale, 1, q or _heads(),
                                     k or _heads(), _heads(), out, rest, None, None)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(n_seq=2), dict(qo=256), dict(qo=256, ko=256, n_seq=-1), dict(q_rows=-1),
                                 dict(k_rows=2**30 + 1), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(dim=0), dict(dim=6),
                                 dict(dim=260), dict(window=0), dict(sinks=-1), dict(scale=float("nan")), dict(out=None), dict(out=8), dict(rest=8),
                                 dict(q=_heads(data=None)), dict(q=_heads(data=8)), dict(k=_heads(row=-4)), dict(k=_heads(head=6)),
                                 dict(heads=70000, kv_heads=1)])
def test_window_attention_refuses(built_library, bad):
    assert _forward(capi.load(), **bad) == BAD
    assert capi.load().rode_last_error()


def test_nothing_to_do_needs_no_device(built_library):
    lib = capi.load()
    assert _forward(lib, q_rows=0, out=None) == 0
    assert lib.rode_window_attention_step(0, 0, 8, 4, 2, 64, 4, 0, 1.0, None, None, None, None, None, None, 0, None) == 0
    assert lib.rode_shared_prefix_attention(0, 0, 8, 8, 4, 2, 64, 1.0, None, None, None, None, None, None, None, None, 0, None) == 0


def test_workspaces(built_library):
    lib, need = capi.load(), ctypes.c_size_t(0)
    backward = lambda n_seq, q_rows, out=ctypes.byref(need): lib.rode_window_attention_backward_workspace_bytes(
        0, n_seq, q_rows, 10, 4, 2, 64, 4, 1, out)
    assert backward(1, 10) == 0 and need.value >= 4 * 10 * 4
    assert backward(1, -1) == BAD and backward(-1, 10) == BAD and backward(1, 10, None) == BAD
    assert backward(0, 10**6) == 0
    back = lambda ws, n, dk=256, dv=256: lib.rode_window_attention_backward(
        0, 1, None, None, 8, 8, 4, 2, 64, 4, 0, 1.0, 1, _heads(), _heads(), _heads(), 256, None, 256, _heads(), 256, dk, dv, ws, n, None)
    assert back(None, 0) == WS and back(256, 8) == WS and back(264, 1 << 20) == WS
    assert back(256, 1 << 20, dk=None) == BAD and back(256, 1 << 20, dv=None) == BAD
    for batch, capacity, window, sinks in ((1, 100000, 100000, 0), (2, 5000, 3000, 4)):
        assert lib.rode_window_attention_step_workspace_bytes(0, batch, capacity, 8, 2, 64, window, sinks, ctypes.byref(need)) == 0
        assert need.value > 0
        step = lambda ws, n: lib.rode_window_attention_step(0, batch, capacity, 8, 2, 64, window, sinks, 1.0, _heads(batch=512), _heads(),
                                                            _heads(), 256, 256, ws, n, None)
        assert step(None, 0) == WS and step(256, need.value - 1) == WS and step(260, need.value) == WS
    assert lib.rode_window_attention_step_workspace_bytes(0, 1, 8, 8, 2, 64, 8, 0, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.rode_window_attention_step(0, 1, 8, 8, 2, 64, 8, 0, 1.0, _heads(), _heads(), _heads(), None, 256, None, 0, None) == BAD
    assert lib.rode_shared_prefix_attention_workspace_bytes(0, 2, 500, 8, 8, 2, 64, ctypes.byref(need)) == 0 and need.value > 0
    assert lib.rode_shared_prefix_attention(0, 2, 500, 8, 8, 2, 64, 1.0, _heads(), _heads(), _heads(), _heads(), _heads(), 256, 256, 256,
                                            need.value - 1, None) == WS
    assert lib.rode_window_attention_backward(0, 1, None, None, 0, 8, 4, 2, 64, 4, 0, 1.0, 1, None, None, None, None, None, None, None, None, 256, 256,
                                              None, 0, None) == BAD  # keys without queries still need their operands
    assert lib.rode_window_attention_step_workspace_bytes(0, 2**29, 8, 8, 2, 64, 8, 0, ctypes.byref(need)) == BAD
    assert lib.rode_shared_prefix_attention_workspace_bytes(0, 2, -1, 8, 8, 2, 64, ctypes.byref(need)) == BAD


def test_reference_gradients_are_the_differences():
    gen = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(n, h, 4, generator=gen) for n, h in ((5, 4), (7, 2), (7, 2), (5, 4)))
    seen = R.visible(5, 7, 3, 1, "cpu")
    one = R.one_sequence(q, k, v, seen, 0.7, dout)
    f = lambda *x: float((R.one_sequence(*x, seen, 0.7)["out"][0] * dout).sum())
    h = 1e-6
    for name, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        x = [q.double(), k.double(), v.double()]
        u = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + h * u, x[i] - h * u
        want = float((one[name][0] * u).sum())
        assert abs((f(*up) - f(*down)) / (2 * h) - want) < 1e-7 * max(1.0, abs(want))


def test_cpu_tensors_are_refused(built_library):
    from rode_b200.rode_attention import rode_window_attention

    x = torch.zeros(4, 2, 8)
    with pytest.raises(ValueError, match="CUDA device"):
        rode_window_attention(x, x, x, 2)
