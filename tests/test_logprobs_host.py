"""Log probabilities without a GPU: what the entry points refuse."""
import ctypes

import pytest
import torch

from nano_vllm_b200.logprobs import token_logprobs

P, P4, P2, NULL = (ctypes.c_void_p(n) for n in (4096, 4100, 4098, 0))


def test_there_is_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("change,code", [
    ({}, -6), ({"rows": 0}, 0), ({"rows": -1}, -3), ({"vocab": 0}, -3), ({"vocab": 0x7fffffff}, -3), ({"top": -1}, -3), ({"top": 65}, -3),
    ({"vocab": 5, "top": 6}, -3), ({"stride": 999}, -3), ({"logits": NULL}, -1), ({"tokens": NULL}, -1), ({"lp": NULL}, -1),
    ({"entropy": NULL}, -1), ({"ids": NULL}, -1), ({"alternatives": NULL}, -1), ({"tokens": P4}, -2), ({"ids": P4}, -2), ({"lp": P2}, -2),
    ({"t": P2}, -2), ({"logits": ctypes.c_void_p(4097)}, -2), ({"fp32": 1, "logits": P2}, -2)])
def test_token_logprobs_refuses(lib, change, code):
    a = dict(logits=P, fp32=0, stride=1000, tokens=P, t=NULL, rows=3, vocab=1000, top=5, lp=P, entropy=P, ids=P, alternatives=P)
    if not change and torch.cuda.is_available():
        pytest.skip("would launch")
    a.update(change)
    assert lib.nvllm_token_logprobs(*a.values(), None) == code
