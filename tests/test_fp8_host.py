"""The 8-bit cache's entry points without a GPU: what they refuse, and the oracle's own consistency."""
import ctypes

import pytest
import torch

from fp8_cases import random_planes, tables_for
from nano_vllm_b200 import _lib, attention as A
from nano_vllm_b200.step_maps import step_maps
from oracle import fp8_cache_ref as F8

P16, P8, NULL = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 8), None
F = ctypes.c_float(0.1)


def test_there_is_no_cpu_fallback():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    c, s = torch.zeros(1, 256, 2, 64).to(torch.float8_e4m3fn), torch.ones(1, 2, 16)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: A.store_kvcache_fp8(q[:, :2], q[:, :2], c, c, s, s, i),
                 lambda: A.decode_paged_fp8(q, c, c, s, s, i, i.view(2, 1), 0.1),
                 lambda: A.decode_step_fp8(q, q[:, :2], q[:, :2], c, c, s, s, i, i, i.view(2, 1), 0.1),
                 lambda: A.prefill_varlen_fp8(q, c, c, s, s, i, i, 2, 2, 0.1, i.view(2, 1)),
                 lambda: step_maps(i, i, i.view(2, 1), i, 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("change,code", [
    ({}, -6), ({"n": -1}, -3), ({"n": 0}, 0), ({"key": NULL}, -1), ({"value": NULL}, -1), ({"slots": NULL}, -1), ({"kc": NULL}, -1),
    ({"ks": NULL}, -1), ({"key": P8}, -2), ({"kc": P8}, -2), ({"vs": P8}, -2), ({"k_stride": 1028}, -2), ({"v_stride": 512}, -3),
    ({"hkv": 0}, -3), ({"d": 96}, -3), ({"blocks": 0}, -3), ({"blocks": 1 << 24}, -3)])
def test_store_refuses(lib, change, code):
    a = dict(key=P16, k_stride=1024, value=P16, v_stride=1024, kc=P16, vc=P16, ks=P16, vs=P16, slots=P16, n=4, hkv=8, d=128, blocks=10)
    if not change and torch.cuda.is_available():
        pytest.skip("would launch")
    a.update(change)
    assert lib.nvllm_store_kvcache_fp8(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    ({"q": NULL}, -1), ({"kc": NULL}, -1), ({"ks": NULL}, -1), ({"lens": NULL}, -1), ({"bt": NULL}, -1), ({"out": NULL}, -1),
    ({"q": P8}, -2), ({"out_stride": 2052}, -2), ({"q_stride": 1024}, -3), ({"bt_stride": 8}, -3), ({"vs": P8}, -2), ({"d": 96}, -3),
    ({"hq": 12}, -3), ({"hq": 128}, -3), ({"blocks": 0}, -3), ({"ws": NULL}, -4), ({"ws_bytes": 100}, -4), ({"ws": P8}, -2),
    ({"batch": 4096}, -3), ({"batch": 0}, 0), ({"scale": ctypes.c_float(-0.1)}, -3)])
def test_decode_refuses(lib, change, code):
    a = dict(q=P16, q_stride=2048, kc=P16, vc=P16, ks=P16, vs=P16, lens=P16, bt=P16, bt_stride=16, width=16, out=P16, out_stride=2048,
             batch=2, hq=16, hkv=8, d=128, scale=F, blocks=100, ws=P16, ws_bytes=1 << 30)
    a.update(change)
    assert lib.nvllm_decode_paged_fp8(*a.values(), None) == code
    step = dict(q=P16, q_stride=2048, key=P16, k_stride=1024, value=P16, v_stride=1024, slots=P16)
    step.update({k: a.pop(k) for k in ("q", "q_stride")})
    assert lib.nvllm_decode_step_fp8(*step.values(), *a.values(), None) == code


@pytest.mark.parametrize("change,code", [({"key": NULL}, -1), ({"slots": NULL}, -1), ({"k_stride": 1028}, -2), ({"v_stride": 8}, -3),
                                         ({"value": P8}, -2)])
def test_step_refuses(lib, change, code):
    a = dict(q=P16, q_stride=2048, key=P16, k_stride=1024, value=P16, v_stride=1024, slots=P16, kc=P16, vc=P16, ks=P16, vs=P16, lens=P16,
             bt=P16, bt_stride=16, width=16, out=P16, out_stride=2048, batch=2, hq=16, hkv=8, d=128, scale=F, blocks=100, ws=P16,
             ws_bytes=1 << 30)
    a.update(change)
    assert lib.nvllm_decode_step_fp8(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    ({"q": NULL}, -1), ({"vc": NULL}, -1), ({"ks": NULL}, -1), ({"bt": NULL}, -1), ({"cu_k": NULL}, -1), ({"out": NULL}, -1), ({"q": P8}, -2),
    ({"ks": P8}, -2), ({"q_stride": 2052}, -2), ({"out_stride": 8}, -3), ({"bt_stride": 1}, -3), ({"width": 0}, -3), ({"batch": 1025}, -3),
    ({"batch": -1}, -3), ({"hq": 15}, -3), ({"d": 32}, -3), ({"blocks": 0}, -3), ({"scale": ctypes.c_float(-1)}, -3),
    ({"scale": ctypes.c_float(float("nan"))}, -3), ({"ws": P8}, -2), ({"ws_bytes": 1000}, -4), ({"batch": 0}, 0), ({"total": 0}, 0), ({"max_q": 0}, 0)])
def test_prefill_refuses(lib, change, code):
    a = dict(q=P16, q_stride=2048, kc=P16, vc=P16, ks=P16, vs=P16, bt=P16, bt_stride=4, width=4, out=P16, out_stride=2048, cu_q=P16, cu_k=P16,
             total=100, batch=2, max_q=60, max_k=600, hq=16, hkv=8, d=128, scale=F, blocks=10, ws=P16, ws_bytes=1 << 30)
    a.update(change)
    assert lib.nvllm_prefill_varlen_fp8(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [
    ({"lens": NULL}, -1), ({"cached": NULL}, -1), ({"bt": NULL}, -1), ({"free": NULL}, -1), ({"cu_q": NULL}, -1), ({"slots": NULL}, -1),
    ({"taken": NULL}, -1), ({"batch": 0}, -3), ({"batch": 4097}, -3), ({"width": 0}, -3), ({"bt_stride": 3}, -3), ({"n_free": -1}, -3),
    ({"rows": -1}, -3), ({"rows": 1 << 31}, -3), ({"width": 1 << 23, "bt_stride": 1 << 23}, -3)])
def test_step_maps_refuses(lib, change, code):
    a = dict(lens=P16, cached=P16, batch=2, bt=P16, bt_stride=4, width=4, free=P16, n_free=3, cu_q=P16, cu_k=P16, slots=P16, pos=P16,
             rows=10, taken=P16)
    a.update(change)
    assert lib.nvllm_step_maps(*a.values(), None) == code and _lib.last_error().startswith("step_maps")


def test_oracle_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    v = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(v.nan_to_num(7e9), F8.VALUES.nan_to_num(7e9))
    x = torch.cat([v[v.isfinite()], torch.randn(20000, dtype=torch.float64) * torch.exp(3 * torch.randn(20000, dtype=torch.float64))])
    x = torch.cat([x, (x[:-1] + x[1:]) / 2]).clamp(-448, 448).float()
    assert torch.equal(F8.encode(x.double()), x.to(torch.float8_e4m3fn).view(torch.uint8))


def test_a_quantised_plane_is_within_half_a_step():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(2, 256, 3, 64, generator=g) * torch.exp(2 * torch.randn(2, 256, 3, 1, generator=g))).bfloat16()
    codes, scales = F8.quantize(x)
    table = torch.arange(2, dtype=torch.int32)
    back = F8.gather(codes, scales, table, 512).view(x.shape)
    step = scales.double().transpose(1, 2).repeat_interleave(16, 1)[..., None] * 2.0 ** -10  # half of a subnormal's
    assert ((back - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + step).all()
    # and rows stored one by one, as a sequence grows, are what the plane is within another rounding of small values
    k, ks = torch.zeros_like(codes), torch.zeros_like(scales)
    for i in range(40):
        F8.store_plane(x.view(512, 3, 64)[i:i + 1], k, ks, torch.tensor([i], dtype=torch.int32))
    grown = F8.gather(k, ks, table, 32)
    assert torch.equal(ks[0, :, :2], scales[0, :, :2])
    assert ((grown - x.double().view(512, 3, 64)[:32]).abs() <= 2.0 ** -4 * x.double().view(512, 3, 64)[:32].abs() + 2 * step.view(512, 3, 1)[:32]).all()


def test_oracle_attention_is_a_softmax():
    g = torch.Generator().manual_seed(2)
    k, v, ks, vs = random_planes(g, 3, 2, 64)
    table = tables_for(g, [300], 3)
    q = torch.randn(1, 4, 64, generator=g).bfloat16()
    out, _ = F8.decode_fp8_ref(q, k, v, ks, vs, torch.tensor([300]), table, 0.125)
    kk, vv = F8.gather(k, ks, table[0], 300), F8.gather(v, vs, table[0], 300)
    for h in range(4):
        want = torch.softmax(kk[:, h // 2] @ q[0, h].double() * 0.125, 0) @ vv[:, h // 2]
        assert torch.allclose(out[0, h], want, rtol=1e-12)
    pre, _ = F8.prefill_fp8_ref(q, k, v, ks, vs, torch.tensor([0, 1]), torch.tensor([0, 300]), 0.125, table)
    assert torch.allclose(pre, out, rtol=1e-12)


def test_oracle_maps_are_the_runners():
    """Two prompts, one behind a cached block: slots and positions as the model runner lists them."""
    table, cu_q, cu_k, slots, pos, taken = F8.step_maps_ref(
        torch.tensor([3, 258]), torch.tensor([0, 256]), torch.tensor([[9, 9], [5, 9]]), torch.tensor([7, 4]), 7)
    assert table == [[7, -1], [5, 4]] and cu_q == [0, 3, 5] and cu_k == [0, 3, 261] and taken == 2
    assert slots == [7 * 256, 7 * 256 + 1, 7 * 256 + 2, 4 * 256, 4 * 256 + 1, -1, -1] and pos == [0, 1, 2, 256, 257, 0, 0]
