"""The C entry points of attention with what a C caller passes and the Python module does not: windows and sinks of INT_MAX for
"no window", more queries than keys."""
import ctypes

import pytest
import torch

import attention_reference as R
from rode_b200 import capi

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
KIND = {torch.float32: capi.RODE_F32, torch.float16: capi.RODE_F16, torch.bfloat16: capi.RODE_BF16}
INT_MAX = 2**31 - 1


def heads_of(x):
    return ctypes.byref(capi.Heads(x.data_ptr(), 0, x.stride(0), x.stride(1)))


def prompt(q, k, v, dout, window, sinks, scale):
    """One sequence: the result, its rest, lse and the gradients."""
    lib, kind = capi.load(), KIND[q.dtype]
    (rows, heads, dim), (k_rows, kv_heads, _) = q.shape, k.shape
    out, dq, rest = (torch.empty_like(q) for _ in range(3))
    dk, dv = (torch.empty_like(k) for _ in range(2))
    lse = torch.empty(heads, rows, device="cuda")
    need = ctypes.c_size_t(0)
    capi.check(lib.rode_window_attention_backward_workspace_bytes(kind, 1, rows, k_rows, heads, kv_heads, dim, window, sinks, ctypes.byref(need)))
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream or None
    common = (kind, 1, None, None, rows, k_rows, heads, kv_heads, dim, window, sinks, scale, 1, heads_of(q), heads_of(k), heads_of(v))
    capi.check(lib.rode_window_attention(*common, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), stream))
    capi.check(lib.rode_window_attention_backward(*common, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), heads_of(dout), dq.data_ptr(),
                                                  dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), need.value, stream))
    torch.cuda.synchronize()
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "rest": rest, "lse": lse}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(INT_MAX, 0), (INT_MAX - 100, 3), (30, INT_MAX), (INT_MAX, INT_MAX)])
@pytest.mark.parametrize("rows,keys,dim", [(400, 400, 64), (305, 300, 64), (400, 250, 128), (130, 700, 128)])
def test_largest_window(rows, keys, dim, window, sinks, dtype):
    gen = torch.Generator(device="cuda").manual_seed(20)
    q, dout = (torch.randn(rows, 4, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    k, v = (torch.randn(keys, 2, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    want = R.one_sequence(q, k, v, R.visible(rows, keys, window, sinks, "cuda"), dim ** -0.5, dout)
    got = prompt(q, k, v, dout, window, sinks, dim ** -0.5)
    for name, pair in want.items():
        R.check(got[name], pair, name)
    # the same as with a window and sinks of all rows
    most = prompt(q, k, v, dout, min(window, 2**20), min(sinks, 2**20), dim ** -0.5)
    for name in want:
        assert torch.equal(got[name], most[name]), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(INT_MAX, 0), (20, INT_MAX), (INT_MAX, INT_MAX)])
def test_largest_window_of_single_tokens(window, sinks, dtype):
    lib, kind = capi.load(), KIND[dtype]
    gen = torch.Generator(device="cuda").manual_seed(21)
    batch, capacity, heads, kv_heads, dim = 3, 2000, 8, 2, 64
    q = torch.randn(batch, heads, dim, generator=gen, device="cuda").to(dtype)
    k, v = (torch.randn(batch, capacity, kv_heads, dim, generator=gen, device="cuda").to(dtype) for _ in range(2))
    lengths = torch.tensor([2000, 0, 777], dtype=torch.int32, device="cuda")

    def run(window, sinks):
        need, out = ctypes.c_size_t(0), torch.empty_like(q)
        capi.check(lib.rode_window_attention_step_workspace_bytes(kind, batch, capacity, heads, kv_heads, dim, window, sinks, ctypes.byref(need)))
        ws = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
        cache = lambda x: ctypes.byref(capi.Heads(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)))
        capi.check(lib.rode_window_attention_step(kind, batch, capacity, heads, kv_heads, dim, window, sinks, 0.125,
                                                  ctypes.byref(capi.Heads(q.data_ptr(), q.stride(0), 0, q.stride(1))), cache(k), cache(v),
                                                  lengths.data_ptr(), out.data_ptr(), ws.data_ptr(), need.value,
                                                  torch.cuda.current_stream().cuda_stream or None))
        torch.cuda.synchronize()
        return out

    assert torch.equal(run(window, sinks), run(min(window, capacity), min(sinks, capacity)))
