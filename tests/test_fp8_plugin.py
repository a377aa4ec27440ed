"""The engine's cache in 8 bits: how ``plugin.fp8_kv_cache`` lays it out, and what the fused attention block then asks for, against
stand-ins of the engine's modules."""
import sys
import types

import pytest
import torch

from nano_vllm_b200 import attention as A, context as C, plugin


def module(monkeypatch, name, **names):
    m = types.ModuleType(name)
    for k, v in names.items():
        setattr(m, k, v)
    monkeypatch.setitem(sys.modules, name, m)
    return m


def runner_class(layers, blocks, block_size, heads, head_dim, layer=A.Attention):
    class ModelRunner:
        def __init__(self):
            self.config = types.SimpleNamespace(num_kvcache_blocks=-1)
            self.model = torch.nn.ModuleList([torch.nn.ModuleList([torch.nn.Identity(), layer(4, head_dim, 0.1, heads)]) for _ in range(layers)])
            self.allocate_kv_cache()

        def allocate_kv_cache(self):
            self.config.num_kvcache_blocks = blocks
            self.kv_cache = torch.empty(2, layers, blocks, block_size, heads, head_dim, dtype=torch.bfloat16)
            at = 0
            for m in self.model.modules():
                if hasattr(m, "k_cache") and hasattr(m, "v_cache"):
                    m.k_cache, m.v_cache = self.kv_cache[0, at], self.kv_cache[1, at]
                    at += 1

    return ModelRunner


@pytest.mark.parametrize("layers,blocks,heads,head_dim", [(3, 10, 2, 128), (2, 7, 1, 64), (1, 1, 8, 128)])
def test_the_cache_is_laid_out_in_the_same_memory(monkeypatch, layers, blocks, heads, head_dim):
    for name in ("nanovllm", "nanovllm.engine"):
        module(monkeypatch, name)
    module(monkeypatch, "nanovllm.engine.model_runner", ModelRunner=runner_class(layers, blocks, 256, heads, head_dim))
    plugin.fp8_kv_cache()
    r = sys.modules["nanovllm.engine.model_runner"].ModelRunner()
    n = r.config.num_kvcache_blocks
    had, has = 2 * layers * blocks * 256 * heads * head_dim * 2, r.kv_cache.nbytes + r.kv_scale.nbytes
    assert has <= had < has + 2 * layers * heads * (256 * head_dim + 64) and n >= 2 * blocks - 1 - blocks // 64
    attn = [m for m in r.model.modules() if isinstance(m, A.Attention)]
    for i, m in enumerate(attn):
        for plane, cache, scale in ((0, m.k_cache, m.k_scale), (1, m.v_cache, m.v_scale)):
            assert cache.dtype == torch.float8_e4m3fn and cache.shape == (n, 256, heads, head_dim) and cache.is_contiguous()
            assert cache.data_ptr() == r.kv_cache[plane, i].data_ptr()
            assert scale.dtype == torch.float32 and scale.shape == (n, heads, 256 // A.SCALE_GROUP) and (scale == 1).all()
            assert scale.is_contiguous() and scale.data_ptr() == r.kv_scale[plane, i].data_ptr()


def test_refusals(monkeypatch):
    class Other(torch.nn.Module):
        def __init__(self, *_):
            super().__init__()
            self.k_cache = self.v_cache = torch.tensor([])

    for name in ("nanovllm", "nanovllm.engine"):
        module(monkeypatch, name)
    for cls in (runner_class(1, 2, 128, 2, 128), runner_class(1, 2, 256, 2, 96), runner_class(1, 2, 256, 2, 64, Other)):
        module(monkeypatch, "nanovllm.engine.model_runner", ModelRunner=cls)
        plugin.fp8_kv_cache()
        with pytest.raises(RuntimeError):
            cls()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_the_fused_block_leaves_the_store_to_the_layer(monkeypatch, dtype):
    calls = []
    monkeypatch.setattr(plugin._attention, "qk_norm_rope_store", lambda *a: calls.append(a[6]))
    slots = torch.zeros(3, dtype=torch.int32)
    monkeypatch.setattr(plugin._attention, "_get_context", lambda: C.Context(False, slot_mapping=slots))

    class Layer:
        k_cache = v_cache = torch.zeros(2, 256, 1, 64).to(dtype)

        def __call__(self, q, k, v, kv_stored=False):
            calls.append(kv_stored)
            return q

    weight = types.SimpleNamespace(weight=None, eps=0.0)
    block = types.SimpleNamespace(qkv_proj=lambda x: x, attn=Layer(), q_norm=weight, k_norm=weight, q_size=128, kv_size=64, num_heads=2,
                                  num_kv_heads=1, head_dim=64, o_proj=lambda x: x, rotary_emb=types.SimpleNamespace(cos_sin_cache=None))
    out = plugin._fused_attention_forward(True)(block, None, torch.zeros(3, 256))
    assert out.shape == (3, 128)
    assert (calls[0] is None, calls[1]) == ((True, False) if dtype == torch.float8_e4m3fn else (False, True))
