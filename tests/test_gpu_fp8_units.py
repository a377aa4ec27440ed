"""Attention over the 8-bit cache where the scales of V differ from sequence to sequence and head to head, and where weights are
small: what the kernels hold their sums in must not show in the results."""
import pytest
import torch

from fp8_cases import assert_within, planes_on, prefill_reference, random_planes, tables_for
from nano_vllm_b200 import _lib, attention as A
from oracle import fp8_cache_ref as F8

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


def sink(gen, hkv, d, n, nats, apart, bits=35):
    """Planes of one sequence of ``n`` tokens whose first key is ``nats`` above all others, with V = 0, in a group whose scale is
    2^``apart`` of the others'; and the output of a query of ones in column 0.  V is an e4m3 number in every column."""
    blocks = -(-n // 256)
    k = torch.zeros(blocks, 256, hkv, d, dtype=torch.uint8)
    v = torch.randint(0x30, 0x38, (1, 1, hkv, d), generator=gen, dtype=torch.uint8).repeat(blocks, 256, 1, 1)  # 0.5 to 0.94
    ks, vs = torch.ones(blocks, hkv, 16), torch.ones(blocks, hkv, 16)
    k[0, 0, :, 0], v[0, 0] = {14: 0x56, 16: 0x58, 18: 0x59}[nats], 0
    vs[0, :, 0] = 2.0 ** apart
    values = v[0, 1].view(torch.float8_e4m3fn).double()  # [hkv, d]
    p = torch.exp(torch.tensor(-float(nats), dtype=torch.float64))
    total = 1 + (n - 1) * p
    own = min(15, n - 1)  # of the first key's group
    out = p * (own * 2.0 ** apart + (n - 1 - own)) / total * values
    # half a step of the result's rounding to bf16, of every weight's to f16, as much again for half of it for sums and
    # exponentials in 32 bits; and for weights below f16's normal range n 2^-bits max |v| / total: 2^-25 of the unit, which is 4
    # times a tile's largest scale at most, over a largest weight of 2^12 (decode, 35), or 2^-25 over one of 2^8 (prefill, 33)
    bound = (2.0 ** -8 + 1.5 * 2.0 ** -11) * out + 2.0 ** -bits * n * values.amax() * 2.0 ** max(apart, 0) / total
    return (k, v, ks, vs), out, bound


SINKS = [(16384, 14), (32768, 16), (32768, 18), (131072, 18)]


@pytest.mark.parametrize("apart", [-4, -1, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("n,nats", SINKS)
@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 64), (4, 1, 128)])
def test_decode_of_small_weights_in_great_number(cuda, hq, hkv, d, n, nats, apart):
    """One such sequence, cut into parts with maxima of their own, and 300 of them (the same blocks), a range to each or so."""
    planes, out, bound = sink(torch.Generator().manual_seed(n + nats), hkv, d, n, nats, apart)
    dev = planes_on(cuda, *planes)
    for batch in (1, 300):
        q = torch.zeros(batch, hq, d, dtype=torch.bfloat16, device=cuda)
        q[:, :, 0] = 1
        table = torch.arange(n // 256, dtype=torch.int32, device=cuda).expand(batch, -1).contiguous()
        got = A.decode_paged_fp8(q, *dev, torch.full((batch,), n, dtype=torch.int32, device=cuda), table, 1.0)
        assert_within(got, out.expand(batch, hq, d), bound.expand(batch, hq, d), f"{batch} sequences")
    assert _lib.read_status() == 0


@pytest.mark.parametrize("apart", [-4, 0, 3, 7])
@pytest.mark.parametrize("n,nats", SINKS)
@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 64), (4, 1, 128)])
def test_prefill_of_small_weights_in_great_number(cuda, hq, hkv, d, n, nats, apart):
    """One query token behind such a sequence, its keys in parts, and 300 of them, whole."""
    planes, out, bound = sink(torch.Generator().manual_seed(n + nats), hkv, d, n, nats, apart, 33)
    dev = planes_on(cuda, *planes)
    for batch in (1, 300):
        q = torch.zeros(batch, hq, d, dtype=torch.bfloat16, device=cuda)
        q[:, :, 0] = 1
        table = torch.arange(n // 256, dtype=torch.int32, device=cuda).expand(batch, -1).contiguous()
        cu = torch.arange(batch + 1, dtype=torch.int32, device=cuda)
        got = A.prefill_varlen_fp8(q, *dev, cu, cu * n, 1, n, 1.0, table)
        assert_within(got, out.expand(batch, hq, d), bound.expand(batch, hq, d), f"{batch} sequences")
    assert _lib.read_status() == 0


@pytest.mark.parametrize("n", [300, 500, 1500])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (4, 2, 64)])
def test_nan_in_cut_sequences(cuda, hq, hkv, d, n):
    """Sequences whose keys several blocks share, in parts of few and of many: a query of NaN, a head whose every key is NaN in one
    part alone, and in all of them."""
    g = torch.Generator().manual_seed(n + d)
    lens = [n] * 4
    blocks = 4 * -(-n // 256)
    planes, tables = random_planes(g, blocks, hkv, d), tables_for(g, lens, blocks)
    q = torch.randn(4, hq, d, generator=g).bfloat16()
    q[0, 1] = float("nan")
    planes[0][int(tables[1, 0]), 128:256, 0, 5] = 0x7F
    planes[0][tables[2].long(), :, 1, 7] = 0xFF
    ctx = torch.tensor(lens, dtype=torch.int32)
    got = A.decode_paged_fp8(q.to(cuda), *planes_on(cuda, *planes), ctx.to(cuda), tables.to(cuda), 0.1).cpu()
    ref, bound = F8.decode_fp8_ref(q, *planes, ctx, tables, 0.1)
    assert ref[0, 1].isnan().all() and ref[1, :2].isnan().all() and ref[2, 2:].isnan().all() and ref.isnan().sum() == 5 * d
    assert torch.equal(got.isnan(), ref.isnan())
    whole = ~ref.isnan()
    assert_within(got[whole], ref[whole], bound.nan_to_num(float("inf"))[whole])
    assert _lib.read_status() == 0


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (14, 2, 64)])
def test_nan_in_keys_in_parts(cuda, hq, hkv, d):
    """Few queries behind a long prefix, whose keys go to several blocks: NaN queries, a head whose every key is NaN, and one whose
    keys are NaN in a stretch that makes up whole parts."""
    g = torch.Generator().manual_seed(d)
    n, new = 4000, 5
    planes, tables = random_planes(g, 16, hkv, d), tables_for(g, [n], 16)
    cu_q, cu_k = torch.tensor([0, new], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32)
    assert _lib.load().nvllm_prefill_fp8_workspace_bytes(1, new, n, hq, hkv, d) > 0  # in parts
    for stretch in (0, 12):
        k = planes[0].clone()
        if stretch:
            k[tables[0, 1:1 + stretch].long(), :, 1, 7] = 0xFF
        q = torch.randn(new, hq, d, generator=g).bfloat16()
        q[1, 0], q[3, hq - 1, 0] = float("nan"), float("inf")
        args = (q, (k, *planes[1:]), cu_q, cu_k, tables, 0.1)
        got = A.prefill_varlen_fp8(q.to(cuda), *planes_on(cuda, *args[1]), cu_q.to(cuda), cu_k.to(cuda), new, n, 0.1, tables.to(cuda)).cpu()
        want = torch.zeros(got.shape, dtype=torch.bool)
        want[1, 0] = want[3, hq - 1] = True
        if stretch:
            want[:, hq // 2:] = True
        assert torch.equal(got.isnan(), want)
        group = hq // hkv
        for h in range(1 if stretch else hkv):
            heads = slice(h * group, (h + 1) * group)
            finite = torch.where(q[:, heads].isfinite(), q[:, heads], 0)
            ref, bound = prefill_reference(finite, by_head(args[1], h), cu_q, cu_k, tables, 0.1)
            whole = ~want[:, heads]
            assert_within(got[:, heads][whole], ref[whole], bound[whole], f"KV head {h}")
    assert _lib.read_status() == 0


@pytest.mark.parametrize("n", [70, 900, 4000])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (14, 2, 64)])
def test_scales_from_the_smallest_to_the_largest(cuda, hq, hkv, d, n):
    """V's scales anywhere in fp32's range, subnormal ones too, in decode and in prefill with keys whole and in parts; results that
    are normal numbers are as right as any."""
    g = torch.Generator().manual_seed(n)
    blocks = 2 * -(-n // 256)
    planes, tables = random_planes(g, blocks, hkv, d, spread=0.3), tables_for(g, [n, n], blocks)
    k, v, ks, vs = planes
    vs = vs.double() / vs.max()
    q = torch.randn(2, hq, d, generator=g).bfloat16()
    ctx, cu_q = torch.tensor([n, n], dtype=torch.int32), torch.arange(3, dtype=torch.int32)
    few = (v & 0x87)  # the smallest codes, for the largest scales
    for exponent, codes in [(e, v) for e in (0, -64, -100, -118, -126, -130, -140, 64, 100, 110)] + [(127, few)]:
        now = (k, codes, ks, (vs * 2.0 ** exponent).float())
        ref, bound = prefill_reference(q, now, cu_q, cu_q * n, tables, 0.1)
        # a few terms and the result may be flushed to zero, 2^-126 each; V over a unit with a scale that is no power of two
        # is rounded twice
        bound = bound * (1 + 4 / 3) + 2.0 ** -123
        dev = planes_on(cuda, *now)
        outs = [A.decode_paged_fp8(q.to(cuda), *dev, ctx.to(cuda), tables.to(cuda), 0.1)]
        for batch in (1, 150):  # 150 of them, of the same two sequences: keys whole
            rows = torch.arange(2).repeat(batch)
            many = torch.arange(2 * batch + 1, dtype=torch.int32)
            outs.append(A.prefill_varlen_fp8(q[rows].to(cuda), *dev, many.to(cuda), (many * n).to(cuda), 1, n, 0.1, tables[rows].to(cuda))[-2:])
        for out in outs:
            assert_within(out.double().cpu() * 2.0 ** -exponent, ref * 2.0 ** -exponent, bound * 2.0 ** -exponent, f"2^{exponent}")
    assert _lib.read_status() == 0


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (14, 2, 64)])
def test_scores_of_millions(cuda, hq, hkv, d):
    """Scores so large that their own rounding is a good part of a binade of a weight, and more: results stay within the values attended,
    and are the value of a key that is clearly above all others."""
    g = torch.Generator().manual_seed(hq)
    n, rows, group = 1700, 40, hq // hkv
    planes, tables = random_planes(g, 7, hkv, d), tables_for(g, [n], 7)
    dev, table = planes_on(cuda, *planes), tables.to(cuda)
    keys, values = (F8.gather(planes[i], planes[2 + i], tables[0], n).repeat_interleave(group, 1) for i in (0, 1))
    low, high = values.amin(0), values.amax(0)  # [hq, d]
    slack = 2.0 ** -7 * torch.maximum(low.abs(), high.abs())  # weights and the result are rounded, sums too
    ctx = torch.full((rows,), n, dtype=torch.int32, device=cuda)
    seen = torch.arange(n) <= torch.arange(rows)[:, None] + n - rows
    for exponent in range(8, 19):
        q = (torch.randn(rows, hq, d, generator=g) * 2.0 ** exponent).bfloat16()  # scores up to 2^(exponent + 10)
        outs = [(torch.ones(rows, n, dtype=torch.bool), A.decode_paged_fp8(q.to(cuda), *dev, ctx, table.expand(rows, -1).contiguous(), 1.0))]
        for batch in (1, 20):  # keys in parts; keys whole
            cu = torch.arange(batch + 1, dtype=torch.int32, device=cuda)
            out = A.prefill_varlen_fp8(q.repeat(batch, 1, 1).to(cuda), *dev, cu * rows, cu * n, rows, n, 1.0, table.expand(batch, -1).contiguous())
            outs += [(seen, part) for part in out.view(batch, rows, hq, d)]
        scores = torch.einsum("qhd,khd->qhk", q.double(), keys)
        # 32-bit sums and products: 2^-20 of the terms' magnitudes; the prefill's query in two parts: 2^-17 of its largest value
        error = 2.0 ** -20 * torch.einsum("qhd,khd->qhk", q.double().abs(), keys.abs()).amax(-1)
        error += 2.0 ** -17 * q.double().abs().amax(-1) * keys.abs().sum(-1).amax(0)
        for mask, out in outs:
            out = out.double().cpu()
            assert ((out >= low - slack) & (out <= high + slack)).all(), f"2^{exponent}"
            two = scores.masked_fill(~mask[:, None], -torch.inf).topk(2)
            clear = two.values[..., 0] - two.values[..., 1] > 2 * error + 30
            clear &= two.values.abs().amax(-1) < 2.0 ** 26
            assert clear.sum() > rows or exponent > 16
            want = values.permute(1, 0, 2)[torch.arange(hq), two.indices[..., 0]]
            assert ((out - want).abs() <= 2.0 ** -7 * want.abs())[clear].all(), f"2^{exponent}"
    assert _lib.read_status() == 0
