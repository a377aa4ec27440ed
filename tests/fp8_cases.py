"""Inputs shared by the tests of the 8-bit cache."""
import torch

from oracle import fp8_cache_ref as F8

HEADS = [(16, 8, 128), (14, 2, 64), (4, 1, 128), (7, 1, 64), (3, 3, 128), (16, 2, 64)]


def to_codes(t):
    return t.cpu().view(torch.uint8)


def planes_on(device, *planes):
    """k codes, v codes, k scales, v scales on the device, as the entry points take them."""
    k, v, ks, vs = (t.to(device) for t in planes)
    return k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs


def random_planes(gen, blocks, hkv, d, spread=1.0):
    """A filled cache whose groups differ in size by about ``spread`` in the logarithm."""
    out = []
    for _ in range(2):
        x = torch.randn(blocks, 256, hkv, d, generator=gen)
        x *= torch.exp(spread * torch.randn(blocks, 256, hkv, 1, generator=gen))
        out.append(F8.quantize(x.bfloat16()))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def spoil_behind(planes, tables, lens):
    """NaN codes and scales in everything that no sequence of ``lens`` holds."""
    k, v, ks, vs = planes
    rows = torch.ones(k.shape[0], 256, dtype=torch.bool)
    groups = torch.ones(k.shape[0], 16, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t0 in range(0, n, 256):
            blk, m = int(tables[b, t0 // 256]), min(256, n - t0)
            rows[blk, :m] = False
            groups[blk, :(m + 15) // 16] = False
    for c in (k, v):
        c[rows] = 0x7F
    for s in (ks, vs):
        s.transpose(1, 2)[groups] = float("nan")


def tables_for(gen, lens, blocks, width=None):
    """Disjoint random blocks for every sequence, -1 behind."""
    need = [-(-n // 256) for n in lens]
    assert sum(need) <= blocks
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.full((len(lens), width or max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def assert_within(out, ref, bound, what=""):
    out = out.double().cpu()
    assert not out.isnan().any(), f"{what}: NaN in output"
    over = (out - ref).abs() / bound.clamp(min=1e-30)
    over[(out == ref)] = 0
    assert over.max() <= 1, f"{what}: {over.max():.3g} times the bound at {tuple((over == over.max()).nonzero()[0].tolist())}"


def prefill_reference(q, planes, cu_q, cu_k, tables, scale):
    """The definition, and the bound with what the query's two e4m3 parts may add: values below 2^-10 of a row's largest are
    off by 2^-17 of it at most, so a score by scale * 2^-17 * max|q| * sum |k|, and a weight by as much of itself."""
    out, bound = F8.prefill_fp8_ref(q, *planes, cu_q, cu_k, scale, tables)
    k, v, ks, vs = planes
    most = 0.0
    for b in range(len(cu_q) - 1):
        n = int(cu_k[b + 1] - cu_k[b])
        if n and cu_q[b + 1] > cu_q[b]:
            most = max(most, float(F8.gather(k, ks, tables[b], n).abs().sum(-1).max()) * float(q[cu_q[b]:cu_q[b + 1]].abs().max()))
    extra = 2 * scale * 2.0 ** -17 * most
    return out, bound * (1 + extra / (1.5 * 2.0 ** -11))
