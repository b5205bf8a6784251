"""The question whether a kernel gave up a wait: it waits for what runs, on every stream."""
import ctypes

import pytest
import torch

from rode_b200 import capi

pytestmark = pytest.mark.gpu


def test_the_question_waits_for_all_streams():
    side = torch.cuda.Stream()
    done = torch.cuda.Event()
    failed = ctypes.c_int(-1)
    capi.check(capi.load().rode_attention_waits_failed(ctypes.byref(failed)))
    with torch.cuda.stream(side):
        torch.cuda._sleep(500_000_000)                  # a kernel of about a quarter of a second
        done.record()
    assert not done.query()
    capi.check(capi.load().rode_attention_waits_failed(ctypes.byref(failed)))
    assert done.query() and failed.value == 0


def test_the_question_from_python():
    from rode_b200.rode_attention import rode_attention_waits_failed

    side = torch.cuda.Stream()
    done = torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(500_000_000)
        done.record()
    assert rode_attention_waits_failed() is False
    assert done.query()
    assert rode_attention_waits_failed("cuda:0") is False and rode_attention_waits_failed(torch.device("cuda")) is False
    with pytest.raises(ValueError):
        rode_attention_waits_failed("cpu")
