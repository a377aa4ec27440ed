"""Log probabilities without a GPU: what the entry points refuse."""
import ctypes

import pytest
import torch

from nano_vllm_b200.logprobs import head_logprobs, token_logprobs

P, P8, P4, P2, NULL = (ctypes.c_void_p(n) for n in (4096, 4104, 4100, 4098, 0))


def test_there_is_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        head_logprobs(torch.zeros(2, 8).bfloat16(), torch.zeros(9, 8).bfloat16(), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("change,code", [
    ({}, -6), ({"rows": 0}, 0), ({"rows": -1}, -3), ({"vocab": 0}, -3), ({"vocab": 0x7fffffff}, -3), ({"top": -1}, -3), ({"top": 65}, -3),
    ({"vocab": (1 << 24) + 1}, -3),
    ({"vocab": 5, "top": 6}, -3), ({"stride": 999}, -3), ({"logits": NULL}, -1), ({"tokens": NULL}, -1), ({"lp": NULL}, -1),
    ({"entropy": NULL}, -1), ({"ids": NULL}, -1), ({"alternatives": NULL}, -1), ({"tokens": P4}, -2), ({"ids": P4}, -2), ({"lp": P2}, -2),
    ({"t": P2}, -2), ({"logits": ctypes.c_void_p(4097)}, -2), ({"fp32": 1, "logits": P2}, -2)])
def test_token_logprobs_refuses(lib, change, code):
    a = dict(logits=P, fp32=0, stride=1000, tokens=P, t=NULL, rows=3, vocab=1000, top=5, lp=P, entropy=P, ids=P, alternatives=P)
    if not change and torch.cuda.is_available():
        pytest.skip("would launch")
    a.update(change)
    assert lib.nvllm_token_logprobs(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    ({}, -6), ({"rows": 0}, 0), ({"rows": -1}, -3), ({"rows": 1 << 25}, -3), ({"hidden": 0}, -3), ({"hidden": 68}, -3), ({"hidden": 1 << 17}, -3),
    ({"vocab": 0}, -3), ({"vocab": (1 << 21) + 1}, -3), ({"x": NULL}, -1), ({"w": NULL}, -1), ({"tokens": NULL}, -1), ({"lp": NULL}, -1),
    ({"entropy": NULL}, -1), ({"x": P8}, -2), ({"w": P8}, -2), ({"x_stride": 132}, -2), ({"w_stride": 132}, -2), ({"x_stride": 120}, -3),
    ({"w_stride": 120}, -3), ({"tokens": P4}, -2), ({"lp": P2}, -2), ({"t": P2}, -2)])
def test_head_logprobs_refuses(lib, change, code):
    a = dict(x=P, x_stride=128, w=P, w_stride=128, tokens=P, t=NULL, rows=3, hidden=128, vocab=1000, lp=P, entropy=P, ws=P, bytes=1 << 30)
    if not change and torch.cuda.is_available():
        pytest.skip("would launch")
    a.update(change)
    assert lib.nvllm_head_logprobs(*a.values(), None) == code
    size = lib.nvllm_head_logprobs_workspace_bytes(a["rows"], a["hidden"], a["vocab"])
    assert size == -3 if code == -3 and not {"x_stride", "w_stride"} & set(change) else size >= 0


def test_head_logprobs_workspace_grows_with_rows_and_not_with_every_tile(lib):
    size = lib.nvllm_head_logprobs_workspace_bytes
    assert size(0, 1024, 151936) == 0
    assert 0 < size(1, 1024, 151936) < 1 << 20
    assert size(4096, 1024, 151936) < 128 << 20
    assert size(32768, 4096, 151936) < 80 << 20
    assert size(1 << 20, 4096, 151936) < 160 << 20
