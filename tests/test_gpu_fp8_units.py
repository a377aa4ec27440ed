"""Attention over the 8-bit cache where the scales of V differ from sequence to sequence and head to head, and where weights are
small: what the kernels hold their sums in must not show in the results."""
import pytest
import torch

from fp8_cases import assert_within, planes_on, prefill_reference, random_planes, tables_for
from nano_vllm_b200 import _lib, attention as A

pytestmark = pytest.mark.gpu


def by_head(planes, h):
    """The planes of one KV head: a bound then takes this head's values for its largest."""
    k, v, ks, vs = planes
    return k[:, :, h:h + 1], v[:, :, h:h + 1], ks[:, h:h + 1], vs[:, h:h + 1]


def scaled_apart(gen, planes, tables, lens):
    """V's scales of every sequence and head times 2^-10, 1 or 2^10."""
    hkv = planes[3].shape[1]
    for b, n in enumerate(lens):
        by = torch.exp2(10.0 * torch.randint(-1, 2, (hkv, 1), generator=gen))
        planes[3][tables[b, :-(-n // 256)].long()] *= by


# items of 128 query rows: 768, 928 and 736 of them, which two blocks to each of 148 SMs take more than two at a time
@pytest.mark.parametrize("hq,hkv,d,batch,cached,new", [(16, 8, 128, 12, 200, 512), (16, 2, 64, 29, 180, 250), (14, 2, 64, 16, 256, 400)])
def test_items_whose_scales_differ(cuda, hq, hkv, d, batch, cached, new):
    """Several items of four key tiles or more to a block, their V's scales up to 2^20 apart, on two streams, over and over."""
    g = torch.Generator().manual_seed(hq + d)
    lens = [cached + new + 7 * b for b in range(batch)]
    blocks = sum(-(-n // 256) for n in lens)
    planes, tables = random_planes(g, blocks, hkv, d), tables_for(g, lens, blocks)
    scaled_apart(g, planes, tables, lens)
    cu_q = torch.arange(batch + 1, dtype=torch.int32) * new
    cu_k = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    q = torch.randn(batch * new, hq, d, generator=g).bfloat16()
    args = (q.to(cuda), *planes_on(cuda, *planes), cu_q.to(cuda), cu_k.to(cuda), new, max(lens), d ** -0.5, tables.to(cuda))
    first = A.prefill_varlen_fp8(*args)
    torch.cuda.synchronize()
    streams, wrong = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(100):
        for s in streams:
            with torch.cuda.stream(s):
                wrong.append((A.prefill_varlen_fp8(*args) != first).sum())
    torch.cuda.synchronize()
    assert torch.stack(wrong).sum() == 0
    group = hq // hkv
    for h in range(hkv):
        heads = slice(h * group, (h + 1) * group)
        ref, bound = prefill_reference(q[:, heads], by_head(planes, h), cu_q, cu_k, tables, d ** -0.5)
        assert_within(first[:, heads], ref, bound, f"KV head {h}")
    assert _lib.read_status() == 0
