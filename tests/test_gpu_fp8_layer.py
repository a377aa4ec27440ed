"""The attention layer over a cache held in 8 bits, with the maps of its steps built on the GPU: prompts, prompts behind cached
blocks, decode steps, as a runner would issue them."""
import pytest
import torch

from fp8_cases import assert_within, prefill_reference, to_codes
from nano_vllm_b200 import _lib, attention as A, context as C
from nano_vllm_b200.step_maps import step_maps
from oracle import fp8_cache_ref as F8

pytestmark = pytest.mark.gpu


class Runner:
    """Lengths and tables of a batch of sequences on the GPU, and the same on the CPU for the oracle."""

    def __init__(self, cuda, batch, width, blocks, hq, hkv, d):
        self.cuda, self.hq, self.hkv, self.d, self.scale = cuda, hq, hkv, d, d ** -0.5
        self.layer = A.Attention(hq, d, self.scale, hkv)
        for name in ("k_cache", "v_cache"):
            setattr(self.layer, name, torch.zeros(blocks, 256, hkv, d, device=cuda).to(torch.float8_e4m3fn))
        for name in ("k_scale", "v_scale"):
            setattr(self.layer, name, torch.zeros(blocks, hkv, 16, device=cuda))
        self.lens = torch.zeros(batch, dtype=torch.int32)
        self.tables = torch.full((batch, width), -1, dtype=torch.int32, device=cuda)
        self.free = torch.arange(blocks, dtype=torch.int32).flip(0)
        self.ref = [torch.zeros(blocks, 256, hkv, d, dtype=torch.uint8) for _ in range(2)] + [torch.zeros(blocks, hkv, 16) for _ in range(2)]

    def maps(self, new):
        cached, seq = self.lens.to(self.cuda), (self.lens + new).to(self.cuda)
        n = int(new.sum())
        want = F8.step_maps_ref(self.lens + new, self.lens, self.tables.cpu(), self.free, n)
        m = step_maps(seq, cached, self.tables, self.free.to(self.cuda), n)
        assert self.tables.tolist() == want[0] and m.slot_mapping.tolist() == want[3] and m.positions.tolist() == want[4]
        self.free = self.free[int(m.blocks_taken):]
        self.lens = self.lens + new
        return m, n

    def rows(self, gen, n):
        qkv = torch.randn(n, (self.hq + 2 * self.hkv) * self.d, generator=gen)
        qkv = (qkv * torch.exp(torch.randn(n, 1, generator=gen))).bfloat16()
        return qkv, qkv.split([self.hq * self.d, self.hkv * self.d, self.hkv * self.d], dim=-1)

    def forward(self, gen, n):
        qkv, (q, k, v) = self.rows(gen, n)
        parts = qkv.to(self.cuda).split([self.hq * self.d, self.hkv * self.d, self.hkv * self.d], dim=-1)
        out = self.layer(*parts).view(n, self.hq, self.d)
        return out, q.view(n, self.hq, self.d), k.view(n, self.hkv, self.d), v.view(n, self.hkv, self.d)

    def same_cache(self):
        layer = self.layer
        for got, want in zip((to_codes(layer.k_cache), to_codes(layer.v_cache), layer.k_scale.cpu(), layer.v_scale.cpu()), self.ref):
            assert torch.equal(got, want)


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (14, 2, 64)])
def test_a_conversation(cuda, hq, hkv, d):
    g = torch.Generator().manual_seed(hq)
    run = Runner(cuda, 4, 4, 16, hq, hkv, d)
    # prompts without a cached prefix: attention over this step's own rows, which are stored as well
    m, n = run.maps(torch.tensor([300, 17, 255, 64], dtype=torch.int32))
    C.set_context(True, m.cu_seqlens_q, m.cu_seqlens_k, 300, 300, m.slot_mapping, None, None)
    out, q, k, v = run.forward(g, n)
    F8.store_kvcache_fp8_ref(k, v, *run.ref, m.slot_mapping.cpu())
    run.same_cache()
    cu = m.cu_seqlens_q.tolist()
    for a, b in zip(cu, cu[1:]):
        seen = torch.ones(b - a, b - a).tril().bool()
        ref, bound = F8.attend(q[a:b], k[a:b], v[a:b], run.scale, seen)
        # the bf16 prefill rounds P to bf16, 2^-8 A where the bound has 1.5 * 2^-11 A: less than 5.4 times that
        assert_within(out[a:b], ref, 6 * bound, "prompts")
    # decode steps, over group and block borders
    for step in range(3):
        m, n = run.maps(torch.ones(4, dtype=torch.int32))
        lens = run.lens.to(cuda)
        C.set_context(False, slot_mapping=m.slot_mapping, context_lens=lens, block_tables=run.tables)
        out, q, k, v = run.forward(g, n)
        F8.store_kvcache_fp8_ref(k, v, *run.ref, m.slot_mapping.cpu())
        run.same_cache()
        assert_within(out, *F8.decode_fp8_ref(q, *run.ref, run.lens, run.tables.cpu(), run.scale), f"decode {step}")
    # the next question: prompts behind what is cached, starting inside groups
    m, n = run.maps(torch.tensor([40, 300, 1, 200], dtype=torch.int32))
    C.set_context(True, m.cu_seqlens_q, m.cu_seqlens_k, 300, int(run.lens.max()), m.slot_mapping, None, run.tables)
    out, q, k, v = run.forward(g, n)
    F8.store_kvcache_fp8_ref(k, v, *run.ref, m.slot_mapping.cpu())
    run.same_cache()
    ref = prefill_reference(q, run.ref, m.cu_seqlens_q.cpu(), m.cu_seqlens_k.cpu(), run.tables.cpu(), run.scale)
    assert_within(out, *ref, "prefill behind cached")
    # rows stored by the caller: decode alone
    m, n = run.maps(torch.ones(4, dtype=torch.int32))
    C.set_context(False, slot_mapping=m.slot_mapping, context_lens=run.lens.to(cuda), block_tables=run.tables)
    qkv, (q, k, v) = run.rows(g, n)
    kv = [t.view(n, hkv, d) for t in (k, v)]
    A.store_kvcache_fp8(kv[0].to(cuda), kv[1].to(cuda), run.layer.k_cache, run.layer.v_cache, run.layer.k_scale, run.layer.v_scale, m.slot_mapping)
    out = run.layer(q.to(cuda), k.to(cuda), v.to(cuda), kv_stored=True).view(n, hq, d)
    C.reset_context()
    F8.store_kvcache_fp8_ref(*kv, *run.ref, m.slot_mapping.cpu())
    run.same_cache()
    assert_within(out, *F8.decode_fp8_ref(q.view(n, hq, d), *run.ref, run.lens, run.tables.cpu(), run.scale))
    assert _lib.read_status() == 0


def test_layers_scales_have_to_fit(cuda):
    run = Runner(cuda, 2, 1, 3, 4, 2, 64)
    i32 = dict(dtype=torch.int32, device=cuda)
    qkv = [torch.zeros(2, n * 64, dtype=torch.bfloat16, device=cuda) for n in (4, 2, 2)]
    C.set_context(False, slot_mapping=torch.tensor([0, 256], **i32), context_lens=torch.ones(2, **i32),
                  block_tables=torch.tensor([[0], [1]], **i32))
    run.layer(*qkv)
    run.layer.k_scale = torch.tensor([])
    with pytest.raises((RuntimeError, AssertionError)):
        run.layer(*qkv)
    run.layer.k_scale = torch.zeros(3, 1, 16, device=cuda)
    with pytest.raises((RuntimeError, AssertionError)):
        run.layer(*qkv)
    C.reset_context()
    assert _lib.read_status() == 0
