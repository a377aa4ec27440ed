"""Prefill attention over the 8-bit cache on the GPU, against the definition in 64 bits."""
import pytest
import torch

from fp8_cases import HEADS, assert_within, planes_on, prefill_reference, random_planes, spoil_behind, tables_for
from nano_vllm_b200 import _lib, attention as A

pytestmark = pytest.mark.gpu


def case(gen, lens, hq, hkv, d, spread=1.0, spoil=True):
    """lens: (cached, new) of every sequence."""
    total = [c + n for c, n in lens]
    blocks = sum(-(-n // 256) for n in total) + 2
    planes = random_planes(gen, blocks, hkv, d, spread)
    tables = tables_for(gen, total, blocks)
    if spoil:
        spoil_behind(planes, tables, total)
    cu_q = torch.tensor([0] + [n for _, n in lens]).cumsum(0).to(torch.int32)
    cu_k = torch.tensor([0] + total).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu_q[-1]), hq, d, generator=gen).bfloat16()
    return q, planes, cu_q, cu_k, tables


def run(cuda, q, planes, cu_q, cu_k, tables, scale, **kw):
    lq, lk = int(cu_q.diff().max()), int(cu_k.diff().max())
    return A.prefill_varlen_fp8(q.to(cuda), *planes_on(cuda, *planes), cu_q.to(cuda), cu_k.to(cuda), lq, lk, scale, tables.to(cuda), **kw)


SHAPES = {
    "one token": [(0, 1)], "one token behind": [(300, 1)], "a tile": [(0, 64)], "borders": [(0, 63), (0, 65), (0, 127), (0, 129), (1, 128)],
    "behind cached": [(256, 20), (512, 100), (255, 2), (17, 48)], "empty rows": [(0, 0), (30, 0), (5, 7), (0, 0), (0, 200), (64, 0)],
    "long": [(0, 1500)], "long behind long": [(2000, 700)], "many": [((37 * i) % 300, (11 * i) % 50) for i in range(90)],
}


@pytest.mark.parametrize("lens", SHAPES.values(), ids=SHAPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_prefill(cuda, hq, hkv, d, lens):
    g = torch.Generator().manual_seed(hq * 7 + len(lens))
    args = case(g, lens, hq, hkv, d)
    assert_within(run(cuda, *args, d ** -0.5), *prefill_reference(*args, d ** -0.5))
    assert _lib.read_status() == 0


def test_rows_that_see_no_key(cuda):
    """Fewer keys than queries: the first rows of a sequence are zeros, whole tiles of them too."""
    g = torch.Generator().manual_seed(3)
    for hq, hkv, d in HEADS:
        q, planes, _, _, _ = case(g, [(0, 400)], hq, hkv, d)
        cu_q = torch.tensor([0, 150, 300, 301, 400], dtype=torch.int32)
        cu_k = torch.tensor([0, 3, 103, 103, 203], dtype=torch.int32)
        tables = torch.arange(4, dtype=torch.int32).view(4, 1) % planes[0].shape[0]
        out = torch.full_like(q, 7.0).to(cuda)
        run(cuda, q, planes_without_nan(planes), cu_q, cu_k, tables, 0.1, out=out)
        ref, bound = prefill_reference(q, planes_without_nan(planes), cu_q, cu_k, tables, 0.1)
        assert (ref[:147] == 0).all() and (ref[300] == 0).all()
        assert_within(out, ref, bound)
    assert _lib.read_status() == 0


def planes_without_nan(planes):
    k, v, ks, vs = planes
    return (torch.where(k & 0x7F == 0x7F, 0, k), torch.where(v & 0x7F == 0x7F, 0, v), ks.nan_to_num(1.0), vs.nan_to_num(1.0))


@pytest.mark.parametrize("d", [64, 128])
def test_scales_of_every_size(cuda, d):
    """Groups' scales far apart, no powers of two, queries of every size and none (scores stay below 100)."""
    g = torch.Generator().manual_seed(6)
    q, planes, *rest = case(g, [(0, 70), (300, 200), (0, 40)], 8, 2, d, spread=0.3)
    planes[3].mul_(torch.exp2(torch.randint(-30, 31, planes[3].shape, generator=g)))
    planes[3].mul_(1 + torch.rand(planes[3].shape, generator=g))
    planes[2].mul_(2.0 ** 20 * (1 + torch.rand(planes[2].shape, generator=g)))
    q = (q.float() * 2.0 ** -20 * torch.exp2(torch.randint(-8, 1, q.shape, generator=g))).bfloat16()
    for f in (1.0, 1e-30, 0.0):
        x = (q.float() * f).bfloat16()
        ref, bound = prefill_reference(x, planes, *rest, 0.1)
        # scales that are no powers of two: V times scale over unit is rounded to f16 twice, 2^-10 A more, where the bound
        # holds 1.5 * 2^-11 A: 4 / 3 of it
        assert_within(run(cuda, x, planes, *rest, 0.1), ref, bound * (1 + 4 / 3), f"queries times {f}")


def test_a_group_of_tiny_values_behind_large_ones(cuda):
    g = torch.Generator().manual_seed(7)
    q, planes, cu_q, cu_k, tables = case(g, [(0, 600)], 4, 1, 128, spread=0.1)
    q.zero_()
    exps = [100, 90, 20, 0, -20, -60, -60, -30, 0, 0, 50, -10, 1, -60, -60, -64] + [-64] * 10 + [0, 100, 3, -5, -7, 4] + [-40] * 6
    for i, e in enumerate(exps):
        planes[3][int(tables[0, i // 16]), 0, i % 16] = 2.0 ** e
    assert_within(run(cuda, q, planes, cu_q, cu_k, tables, 0.1), *prefill_reference(q, planes, cu_q, cu_k, tables, 0.1))


def test_nan_and_infinities_that_are_seen(cuda):
    g = torch.Generator().manual_seed(8)
    q, planes, cu_q, cu_k, tables = case(g, [(0, 100), (0, 130), (20, 10)], 4, 2, 64)
    k, v, ks, vs = planes
    k[int(tables[0, 0]), 50, 1, 3] = 0x7F   # seen by queries 50 .. of heads 2 and 3
    v[int(tables[1, 0]), 7, 0, 5] = 0xFF    # column 5 of queries 7 .. of heads 0 and 1
    q[235, 3, 4], q[236, 0, 7] = float("nan"), float("inf")
    out = run(cuda, q, planes, cu_q, cu_k, tables, 0.1).float().cpu()
    want = torch.zeros_like(out, dtype=torch.bool)
    want[50:100, 2:] = True
    want[235, 3] = want[236, 0] = True
    got = out.isnan()
    assert got[want].all()
    # V's: rows of the query's tile that do not see the key have weight zero for it, and zero times NaN is NaN in their column
    column = torch.zeros_like(want)
    column[100:230, :2, 5] = True
    assert got[107:230, :2, 5].all() and not (got & ~want & ~column).any()


def test_bad_blocks_strides_and_streams(cuda):
    g = torch.Generator().manual_seed(9)
    hq, hkv, d = 4, 2, 64
    q, planes, cu_q, cu_k, tables = case(g, [(100, 200), (0, 300), (0, 40)], hq, hkv, d)
    wide = torch.full((3, 5), 7000, dtype=torch.int32)
    wide[:, :2] = tables
    n = q.shape[0]
    ref, bound = prefill_reference(q, planes, cu_q, cu_k, tables, 0.1)
    qd = torch.randn(n, hq * d + 64, generator=g).bfloat16().to(cuda)[:, :hq * d].view(n, hq, d).copy_(q)
    out = torch.full((n + 9, hq * d + 8), 5.0, dtype=torch.bfloat16, device=cuda)
    dev = planes_on(cuda, *planes)
    lens = [t.to(cuda) for t in (cu_q, cu_k, wide)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = A.prefill_varlen_fp8(qd, *dev, *lens[:2], 300, 300, 0.1, lens[2][:, :2], out=out[:n, :hq * d].view(n, hq, d))
    stream.synchronize()
    assert_within(got, ref, bound)
    assert (out[n:] == 5).all() and (out[:, hq * d:] == 5).all()
    _lib.read_status()
    tables[1, 1] = planes[0].shape[0]
    got = run(cuda, q, planes, cu_q, cu_k, tables, 0.1)
    assert _lib.read_status() == 2
    keep = torch.cat([torch.arange(200), torch.arange(500, 540)])
    assert_within(got[keep], ref[keep], bound[keep])


def test_captured_and_replayed_with_other_lengths(cuda):
    """Two graphs of one launch each, replayed in turn with other lengths and tables, as a chunked prefill would."""
    g = torch.Generator().manual_seed(10)
    hq, hkv, d = 8, 2, 128
    q, planes, _, _, _ = case(g, [(0, 500), (0, 500)], hq, hkv, d, spoil=False)
    dev, qd = planes_on(cuda, *planes), q.to(cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    static = [(torch.zeros(3, **i32), torch.zeros(3, **i32), torch.zeros(2, 2, **i32)) for _ in range(2)]
    graphs = []
    for cq, ck, bt in static:
        call = lambda: A.prefill_varlen_fp8(qd, *dev, cq, ck, 1000, 512, 0.1, bt)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for step, (a, b, ka, kb) in enumerate([(300, 700, 400, 512), (0, 1000, 1, 512), (17, 3, 17, 5), (1, 1, 512, 512)]):
        cu_q = torch.tensor([0, a, a + b], dtype=torch.int32)
        cu_k = torch.tensor([0, ka, ka + kb], dtype=torch.int32)
        tables = torch.tensor([[0, 3], [2, 1]], dtype=torch.int32).roll(step, 1)
        for to, t in zip(static[step % 2], (cu_q, cu_k, tables)):
            to.copy_(t)
        graph, out = graphs[step % 2]
        graph.replay()
        ref, bound = prefill_reference(q[:a + b], planes, cu_q, cu_k, tables, 0.1)
        assert_within(out[:a + b], ref, bound, f"step {step}")
    assert _lib.read_status() == 0


FEW = {
    "one token": [(5000, 1)], "a block in part": [(2817, 3)], "two lengths": [(3, 2), (4000, 30)], "one more than blocks": [(2047, 2)],
    "tiles of all": [(1000, 130)], "shorter than parts": [(7000, 4), (0, 1), (0, 0), (100, 3)], "no key in some": [(-40, 60), (3000, 9)],
}


@pytest.mark.parametrize("lens", FEW.values(), ids=FEW)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_few_tokens_behind_long_prefixes(cuda, hq, hkv, d, lens):
    """An item's keys in parts, and the same without a workspace; a workspace that is as it was (counters at zero) behind each."""
    g = torch.Generator().manual_seed(hq + 31 * len(lens))
    q, planes, cu_q, cu_k, tables = case(g, lens, hq, hkv, d)
    ref, bound = prefill_reference(q, planes, cu_q, cu_k, tables, d ** -0.5)
    dev, qd = planes_on(cuda, *planes), q.to(cuda)
    cq, ck, bt = cu_q.to(cuda), cu_k.to(cuda), tables.to(cuda)
    lib, lq, lk = _lib.load(), int(cu_q.diff().max()), int(cu_k.diff().max())
    need = lib.nvllm_prefill_fp8_workspace_bytes(len(lens), lq, lk, hq, hkv, d)
    ws = torch.zeros(max(need, 1), dtype=torch.uint8, device=cuda)
    for w, size in ((ws.data_ptr(), need), (ws.data_ptr(), need), (0, 0)):
        out = torch.full_like(qd, 9.0)
        k, v, ks, vs = (t.data_ptr() for t in dev)
        rc = lib.nvllm_prefill_varlen_fp8(qd.data_ptr(), hq * d, k, v, ks, vs, bt.data_ptr(), bt.stride(0), bt.shape[1], out.data_ptr(),
                                          hq * d, cq.data_ptr(), ck.data_ptr(), q.shape[0], len(lens), lq, lk, hq, hkv, d,
                                          d ** -0.5, dev[0].shape[0], w, size, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert_within(out, ref, bound, f"workspace of {size}")
    assert (ws[:65536] == 0).all()
    assert _lib.read_status() == 0


def test_split_in_graphs(cuda):
    """Graphs of a prefill behind a long prefix, of a decode over the same cache and of both, replayed in turn."""
    g = torch.Generator().manual_seed(12)
    hq, hkv, d = 8, 2, 128
    q, planes, cu_q, cu_k, tables = case(g, [(3000, 20)], hq, hkv, d)
    dev, qd, ctx = planes_on(cuda, *planes), q.to(cuda), torch.tensor([3020], dtype=torch.int32, device=cuda)
    cq, ck, bt = cu_q.to(cuda), cu_k.to(cuda), tables.to(cuda)
    pre = lambda: A.prefill_varlen_fp8(qd, *dev, cq, ck, 20, 3020, 0.1, bt)  # noqa: E731
    dec = lambda: A.decode_paged_fp8(qd[19:], *dev, ctx, bt, 0.1)  # noqa: E731
    want = [pre().clone(), dec().clone()]
    ref, bound = prefill_reference(q, planes, cu_q, cu_k, tables, 0.1)
    assert_within(want[0], ref, bound)
    torch.cuda.synchronize()
    graphs = []
    for calls in ((pre,), (dec,), (pre, dec, dec, pre, pre)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [c() for c in calls]
        graphs.append((graph, calls, outs))
    for n in (0, 1, 2, 1, 0, 2):
        graph, calls, outs = graphs[n]
        for o in outs:
            o.zero_()
        graph.replay()
        pre()
        for c, o in zip(calls, outs):
            assert torch.equal(o, want[0 if c is pre else 1])
    assert _lib.read_status() == 0


def test_split_on_two_streams_at_once(cuda):
    """Every call has a scratch of its own: calls that overlap do not meet."""
    g = torch.Generator().manual_seed(13)
    jobs = []
    for lens in ([(6000, 30)], [(4000, 9), (2500, 64)]):
        q, planes, cu_q, cu_k, tables = case(g, lens, 14, 2, 64)
        args = (q.to(cuda), *planes_on(cuda, *planes), cu_q.to(cuda), cu_k.to(cuda), int(cu_q.diff().max()), int(cu_k.diff().max()), 0.1, tables.to(cuda))
        jobs.append((torch.cuda.Stream(), args, prefill_reference(q, planes, cu_q, cu_k, tables, 0.1)))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for o, (stream, args, _) in zip(outs, jobs):
            with torch.cuda.stream(stream):
                o.append(A.prefill_varlen_fp8(*args))
    torch.cuda.synchronize()
    for o, (_, _, (ref, bound)) in zip(outs, jobs):
        assert_within(o[0], ref, bound)
        assert all(torch.equal(x, o[0]) for x in o)
    assert _lib.read_status() == 0


def test_refusals(cuda):
    bf = dict(dtype=torch.bfloat16, device=cuda)
    q, c = torch.zeros(4, 4, 64, **bf), torch.zeros(3, 256, 2, 64, device=cuda).to(torch.float8_e4m3fn)
    s, cu = torch.ones(3, 2, 16, device=cuda), torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    t = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    good = (q, c, c, s, s, cu, cu, 4, 4, 0.1, t)
    A.prefill_varlen_fp8(*good)
    assert A.prefill_varlen_fp8(q[:0], *good[1:]).shape == (0, 4, 64)
    for at, bad in ((0, q.float()), (0, q[..., :32]), (0, q[:, :3]), (1, c.view(torch.uint8)), (2, c[:2]), (3, s[:, :1]), (4, s.double()),
                    (4, s.cpu()), (5, cu.long()), (6, cu[:1]), (5, cu.cpu()), (9, -0.1), (9, float("nan")), (10, t.long()),
                    (10, t.expand(2, 1)), (10, t.cpu())):
        args = list(good)
        args[at] = bad
        with pytest.raises((RuntimeError, AssertionError)):
            A.prefill_varlen_fp8(*args)
    with pytest.raises((RuntimeError, AssertionError)):
        A.prefill_varlen_fp8(*good, out=torch.zeros(5, 4, 64, **bf))
    torch.cuda.synchronize()
    assert _lib.read_status() == 0
