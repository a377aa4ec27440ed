"""Decode attention over the 8-bit cache on the GPU, against the definition in 64 bits."""
import pytest
import torch

from fp8_cases import HEADS, assert_within, planes_on, random_planes, spoil_behind, tables_for, to_codes
from nano_vllm_b200 import _lib, attention as A
from oracle import fp8_cache_ref as F8

pytestmark = pytest.mark.gpu

LENS = {
    "one": [1], "short": [317], "borders": [1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 512, 513],
    "empty rows": [0, 0, 40, 0, 300, 0], "all empty": [0, 0, 0], "cut": [3000, 1, 1500], "many": [(37 * i) % 400 for i in range(200)],
    "one to a thread": [(13 * i) % 90 for i in range(300)],
}


def case(gen, lens, hq, hkv, d, spread=1.0, spoil=True):
    blocks = sum(-(-n // 256) for n in lens) + 2
    planes = random_planes(gen, blocks, hkv, d, spread)
    tables = tables_for(gen, lens, blocks)
    if spoil:
        spoil_behind(planes, tables, lens)
    q = torch.randn(len(lens), hq, d, generator=gen).bfloat16()
    return q, planes, torch.tensor(lens, dtype=torch.int32), tables


def run(cuda, q, planes, lens, tables, scale, **kw):
    return A.decode_paged_fp8(q.to(cuda), *planes_on(cuda, *planes), lens.to(cuda), tables.to(cuda), scale, **kw)


@pytest.mark.parametrize("lens", LENS.values(), ids=LENS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode(cuda, hq, hkv, d, lens):
    g = torch.Generator().manual_seed(hq * 7 + len(lens))
    q, planes, ctx, tables = case(g, lens, hq, hkv, d)
    out = run(cuda, q, planes, ctx, tables, d ** -0.5)
    assert_within(out, *F8.decode_fp8_ref(q, *planes, ctx, tables, d ** -0.5))
    assert (out[ctx == 0] == 0).all()
    assert _lib.read_status() == 0


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (8, 1, 64)])
def test_a_long_cache(cuda, hq, hkv, d):
    g = torch.Generator().manual_seed(5)
    q, planes, ctx, tables = case(g, [20000], hq, hkv, d)
    assert_within(run(cuda, q, planes, ctx, tables, d ** -0.5), *F8.decode_fp8_ref(q, *planes, ctx, tables, d ** -0.5))


@pytest.mark.parametrize("d", [64, 128])
def test_scales_of_every_size(cuda, d):
    """Groups' scales far apart, no powers of two, and queries of every size (scores stay below 100)."""
    g = torch.Generator().manual_seed(6)
    lens = [70, 700, 40]
    q, planes, ctx, tables = case(g, lens, 8, 2, d, spread=0.3)
    planes[3].mul_(torch.exp2(torch.randint(-30, 31, planes[3].shape, generator=g)))
    planes[3].mul_(1 + torch.rand(planes[3].shape, generator=g))
    planes[2].mul_(2.0 ** 20 * (1 + torch.rand(planes[2].shape, generator=g)))
    q = (q.float() * 2.0 ** -20 * torch.exp2(torch.randint(-8, 1, q.shape, generator=g))).bfloat16()
    ref, bound = F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1)
    assert_within(run(cuda, q, planes, ctx, tables, 0.1), ref, bound)
    q = (q.float() * 1e-30).bfloat16()  # all keys alike
    assert_within(run(cuda, q, planes, ctx, tables, 0.1), *F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1))
    q.zero_()
    assert_within(run(cuda, q, planes, ctx, tables, 0.1), *F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1))


def test_a_group_of_tiny_values_behind_large_ones(cuda):
    """V's scales fall from 2^100 to 2^-60 and rise again: O stays finite and right."""
    g = torch.Generator().manual_seed(7)
    d = 128
    q, planes, ctx, tables = case(g, [200], 4, 1, d, spread=0.1)
    q.zero_()
    k, v, ks, vs = planes
    blk = int(tables[0, 0])
    vs[blk, 0, :13] = torch.tensor([2.0 ** e for e in (100, 90, 20, 0, -20, -60, -60, -30, 0, 0, 50, -10, 1)])
    out = run(cuda, q, planes, ctx, tables, 0.1)
    assert_within(out, *F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1))
    ctx[0] = 17 * 4  # from small to large only
    vs[blk, 0, :5] = torch.tensor([2.0 ** e for e in (-60, -60, -30, 0, 100)])
    assert_within(run(cuda, q, planes, ctx, tables, 0.1), *F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1))


def test_nan_and_infinities_that_are_seen(cuda):
    g = torch.Generator().manual_seed(8)
    q, planes, ctx, tables = case(g, [100, 100, 300, 100], 4, 2, 64)
    k, v, ks, vs = planes
    k[int(tables[0, 0]), 50, 1, 3] = 0x7F
    v[int(tables[2, 0]), 7, 0, 5] = 0xFF
    q[3, 0, 4] = float("nan")
    out = run(cuda, q, planes, ctx, tables, 0.1).float().cpu()
    ref, _ = F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1)
    assert torch.equal(out.isnan(), ref.isnan())
    assert out[0, 2:].isnan().all() and not out[0, :2].isnan().any() and not out[1].isnan().any() and out[3, 0].isnan().all()


def test_bad_blocks_and_strides(cuda):
    g = torch.Generator().manual_seed(9)
    hq, hkv, d = 4, 2, 64
    q, planes, ctx, tables = case(g, [300, 300, 40], hq, hkv, d)
    wide = torch.full((3, 5), 7000, dtype=torch.int32)
    wide[:, :2] = tables
    rows = torch.randn(3, hq * d + 64, generator=g).bfloat16().to(cuda)
    qd = rows[:, :hq * d].view(3, hq, d).copy_(q)
    out = torch.zeros(3, hq * d + 8, dtype=torch.bfloat16, device=cuda)[:, :hq * d].view(3, hq, d)
    got = A.decode_paged_fp8(qd, *planes_on(cuda, *planes), ctx.to(cuda), wide.to(cuda)[:, :2], 0.1, out=out)
    assert got.data_ptr() == out.data_ptr()
    ref, bound = F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1)
    assert_within(out, ref, bound)
    _lib.read_status()
    tables[1, 1] = planes[0].shape[0]
    got = run(cuda, q, planes, ctx, tables, 0.1)
    assert _lib.read_status() == 2
    keep = torch.tensor([0, 2])
    assert_within(got[keep], ref[keep], bound[keep])


def test_refusals(cuda):
    bf = dict(dtype=torch.bfloat16, device=cuda)
    q, c = torch.zeros(2, 4, 64, **bf), torch.zeros(3, 256, 2, 64, device=cuda).to(torch.float8_e4m3fn)
    s, i = torch.ones(3, 2, 16, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    t = torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    key = torch.zeros(2, 2, 64, **bf)
    A.decode_paged_fp8(q, c, c, s, s, i, t, 0.1)
    for bad in ((q.float(), c, c, s, s, i, t), (q, c.view(torch.uint8), c, s, s, i, t), (q, c, c[:2], s, s, i, t), (q, c, c, s[:2], s, i, t),
                (q, c, c, s, s.half(), i, t), (q, c, c, s, s, i.long(), t), (q, c, c, s, s, i[:1], t), (q, c, c, s, s, i, t[:1]),
                (q[..., :32], c, c, s, s, i, t), (q, c, c, s, s.cpu(), i, t), (q, c, c, s, s, i.cpu(), t), (q, c.transpose(0, 1), c, s, s, i, t),
                (torch.zeros(2, 3, 64, **bf), c, c, s, s, i, t)):
        with pytest.raises((RuntimeError, AssertionError)):
            A.decode_paged_fp8(*bad, 0.1)
    with pytest.raises((RuntimeError, AssertionError)):
        A.decode_paged_fp8(q, c, c, s, s, i, t, 0.1, out=torch.zeros(2, 4, 64, device=cuda))
    with pytest.raises((RuntimeError, AssertionError)):
        A.decode_paged_fp8(q, c, c, s, s, i, t, 0.1, out=torch.zeros(1, 4, 64, **bf))
    for k, v, sl in ((key[:1], key, i), (key, key[:, :1], i), (key, key, i[:1]), (key.cpu(), key, i), (key, key, i.long())):
        with pytest.raises((RuntimeError, AssertionError)):
            A.store_kvcache_fp8(k, v, c, c, s, s, sl)
        with pytest.raises((RuntimeError, AssertionError)):
            A.decode_step_fp8(q, k, v, c, c, s, s, sl, i, t, 0.1)
    torch.cuda.synchronize()
    assert _lib.read_status() == 0


# ---- the step: store and decode in one launch -------------------------------------------------------

def new_rows(gen, n, hkv, d):
    size = torch.exp(2 * torch.randn(n, hkv, 1, generator=gen))
    return (torch.randn(n, hkv, d, generator=gen) * size).bfloat16()


def slots_of(tables, lens):
    return torch.tensor([int(tables[b, (n - 1) // 256]) * 256 + (n - 1) % 256 if n else -1 for b, n in enumerate(lens)], dtype=torch.int32)


@pytest.mark.parametrize("lens", LENS.values(), ids=LENS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_step_is_store_and_decode(cuda, hq, hkv, d, lens):
    g = torch.Generator().manual_seed(hq * 11 + len(lens))
    q, planes, ctx, tables = case(g, lens, hq, hkv, d, spoil=False)
    spoil_behind(planes, tables, [max(n - 1, 0) for n in lens])
    key, value, slots = new_rows(g, len(lens), hkv, d), new_rows(g, len(lens), hkv, d), slots_of(tables, lens)
    dev = planes_on(cuda, *planes)
    out = A.decode_step_fp8(q.to(cuda), key.to(cuda), value.to(cuda), *dev, slots.to(cuda), ctx.to(cuda), tables.to(cuda), 0.1)
    F8.store_kvcache_fp8_ref(key, value, *planes, slots)
    for got, want in zip((to_codes(dev[0]), to_codes(dev[1]), dev[2].cpu(), dev[3].cpu()), planes):
        assert ((got == want) | (got.isnan() & want.isnan())).all()
    assert_within(out, *F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1))
    two = A.decode_paged_fp8(q.to(cuda), *dev, ctx.to(cuda), tables.to(cuda), 0.1)
    assert torch.equal(out, two)
    assert _lib.read_status() == 0


def test_step_rules_for_slots(cuda):
    """A negative slot stores nothing, a slot that is not the newest position's is flagged, an empty row stores nothing."""
    g = torch.Generator().manual_seed(13)
    hq, hkv, d = 4, 2, 128
    lens = [30, 300, 0, 33]
    q, planes, ctx, tables = case(g, lens, hq, hkv, d)
    key, value = new_rows(g, 4, hkv, d), new_rows(g, 4, hkv, d)
    slots = slots_of(tables, lens)
    slots[0], slots[2] = -1, 5
    slots[1] -= 1
    dev = planes_on(cuda, *planes)
    _lib.read_status()
    out = A.decode_step_fp8(q.to(cuda), key.to(cuda), value.to(cuda), *dev, slots.to(cuda), ctx.to(cuda), tables.to(cuda), 0.1)
    assert _lib.read_status() == 1
    slots[:3] = -1
    F8.store_kvcache_fp8_ref(key, value, *planes, slots)
    for got, want in zip((to_codes(dev[0]), to_codes(dev[1]), dev[2].cpu(), dev[3].cpu()), planes):
        assert ((got == want) | (got.isnan() & want.isnan())).all()
    assert_within(out, *F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1))


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (14, 2, 64)])
def test_a_captured_step_follows_its_sequences(cuda, hq, hkv, d):
    """Forty tokens, one replay each, over group and block borders; rows of the batch end and others begin."""
    g = torch.Generator().manual_seed(14)
    B, blocks = 5, 12
    zero = torch.zeros(blocks, 256, hkv, d, dtype=torch.uint8)
    planes = [zero, zero.clone(), torch.zeros(blocks, hkv, 16), torch.zeros(blocks, hkv, 16)]
    lens = [0, 240, 13, 255, 0]
    tables = torch.arange(10, dtype=torch.int32).view(B, 2)
    for b, n in enumerate(lens):
        if n:
            slots = torch.tensor([int(tables[b, p // 256]) * 256 + p % 256 for p in range(n)], dtype=torch.int32)
            F8.store_kvcache_fp8_ref(new_rows(g, n, hkv, d), new_rows(g, n, hkv, d), *planes, slots)
    dev = planes_on(cuda, *planes)
    static = [torch.zeros(B, n, d, dtype=torch.bfloat16, device=cuda) for n in (hq, hkv, hkv)]
    slots_d, lens_d = (torch.zeros(B, dtype=torch.int32, device=cuda) for _ in range(2))
    tables_d = tables.to(cuda)
    run = lambda: A.decode_step_fp8(*static, *dev, slots_d, lens_d, tables_d, 0.1)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for step in range(40):
        live = [1, 1, 1, step < 20, step >= 10]
        lens = [n + 1 if on else n for n, on in zip(lens, live)]
        ctx = torch.tensor([n if on else 0 for n, on in zip(lens, live)], dtype=torch.int32)
        slots = slots_of(tables, ctx.tolist())
        rows = [torch.randn(B, hq, d, generator=g).bfloat16(), new_rows(g, B, hkv, d), new_rows(g, B, hkv, d)]
        for to, t in zip((*static, slots_d, lens_d), (*rows, slots, ctx)):
            to.copy_(t)
        graph.replay()
        F8.store_kvcache_fp8_ref(*rows[1:], *planes, slots)
        assert_within(out, *F8.decode_fp8_ref(rows[0], *planes, ctx, tables, 0.1), f"step {step}")
    for got, want in zip((to_codes(dev[0]), to_codes(dev[1]), dev[2].cpu(), dev[3].cpu()), planes):
        assert torch.equal(got, want)
    assert _lib.read_status() == 0


def test_two_captured_graphs_and_the_bf16_decode_share_the_scratch(cuda):
    """Launches that cut their sequences, one after the other on one stream, leave the scratch as the next needs it."""
    from nano_vllm_b200 import workloads as W
    g = torch.Generator().manual_seed(15)
    cases = [case(g, lens, 16, 8, 128) for lens in ([3000, 20, 900], [1, 4000])]
    args = [(q.to(cuda), *planes_on(cuda, *p), ctx.to(cuda), t.to(cuda), 0.1) for q, p, ctx, t in cases]
    bf = W.make_decode_case(3, 6, 500, 3000, 16, 8, 128).to(cuda)
    other = lambda: A.decode_paged(bf.q, bf.k_cache, bf.v_cache, bf.context_lens, bf.block_tables, bf.scale)  # noqa: E731
    want = [A.decode_paged_fp8(*a) for a in args] + [other()]
    graphs = []
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = A.decode_paged_fp8(*a)
        graphs.append((graph, out))
    for k in range(6):
        graph, out = graphs[k % 2]
        graph.replay()
        assert torch.equal(other(), want[2])
        assert torch.equal(out, want[k % 2])
    assert _lib.read_status() == 0
