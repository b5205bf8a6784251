"""What has no derivative says so: single tokens in reverse and forward mode, prompts in forward mode.  Without a device: the check comes
before that for one."""
import pytest
import torch
import torch.autograd.forward_ad as fw


def _step(**x):
    from rode_b200.rode_attention import rode_window_attention_step

    return rode_window_attention_step(x["q"][:, 0], x["k"], x["v"], x["lengths"], 4)


def _shared(**x):
    from rode_b200.rode_attention import rode_shared_prefix_attention

    return rode_shared_prefix_attention(x["q"][:, 0], x["pk"], x["pv"], x["k"], x["v"], x["lengths"])


def _window(**x):
    from rode_b200.rode_attention import rode_window_attention

    return rode_window_attention(x["q"][:, 0], x["pk"], x["pv"], 4)


def _inputs(device):
    make = lambda *s: torch.randn(*s, device=device)
    return {"q": make(3, 1, 4, 64), "k": make(3, 8, 2, 64), "v": make(3, 8, 2, 64), "pk": make(3, 2, 64), "pv": make(3, 2, 64),
            "lengths": torch.full((3,), 8, dtype=torch.int32, device=device)}


CALLS = [(_step, n) for n in "qkv"] + [(_shared, n) for n in ("q", "k", "v", "pk", "pv")]


@pytest.mark.parametrize("call,name", CALLS)
def test_no_gradient_of_single_tokens(built_library, call, name):
    x = _inputs("cpu")
    x[name].requires_grad_()
    with pytest.raises(NotImplementedError, match="no_grad"):
        call(**x)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):       # (as far as it gets here)
        call(**x)


@pytest.mark.parametrize("call,name", CALLS + [(_window, n) for n in ("q", "pk", "pv")])
@pytest.mark.parametrize("leaf", [False, True])
def test_no_tangents(built_library, call, name, leaf):
    with fw.dual_level():
        x = _inputs("cpu")
        x[name] = fw.make_dual(x[name].requires_grad_(leaf), torch.ones_like(x[name]))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            call(**x)
        with pytest.raises(NotImplementedError):
            call(**x)


@pytest.mark.gpu
@pytest.mark.parametrize("call", [_step, _shared])
def test_without_gradients_nothing_changes(call):
    x = _inputs("cuda")
    want = call(**x)
    for name in ("q", "k", "v", "pk", "pv"):
        x[name].requires_grad_()
    with torch.no_grad():
        got = call(**x)
    with torch.inference_mode():
        again = call(**x)
    assert torch.equal(got, want) and torch.equal(again, want) and not got.requires_grad
    with pytest.raises(NotImplementedError):
        call(**x)
    call(**{n: t.detach() for n, t in x.items()})
