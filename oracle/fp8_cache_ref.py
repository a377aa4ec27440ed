"""CPU restatement, in 64 bits, of the operators around a K/V cache held in 8 bits — TEST INFRASTRUCTURE, not product code.

Written from the definitions alone, slot by slot and sequence by sequence: codes are ``uint8`` e4m3 (sign, four bits of exponent
with bias 7, three of mantissa, 0x7f / 0xff NaN, no infinities), scales are fp32 ``[num_blocks, Hkv, 16]``.
"""
from __future__ import annotations

import math

import torch

BLOCK_SIZE, GROUP = 256, 16


def _values() -> torch.Tensor:
    out = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = math.nan if c & 127 == 127 else math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


VALUES = _values()  # of the 256 codes
_GRID = VALUES[:127].clone()  # of the codes without a sign, rising


def encode(y: torch.Tensor) -> torch.Tensor:
    """Nearest codes, ties to the even one, of values within +-448; NaN and infinities to 0x7f."""
    a = y.abs().clamp(max=448.0).nan_to_num(0.0)
    hi = torch.searchsorted(_GRID, a.contiguous()).clamp(max=126)  # first code whose value is >= a
    lo = (hi - 1).clamp(min=0)
    to_lo, to_hi = a - _GRID[lo], _GRID[hi] - a
    up = (to_hi < to_lo) | ((to_hi == to_lo) & (hi % 2 == 0))
    code = torch.where(up, hi, lo) + torch.where(torch.signbit(y), 128, 0)
    return torch.where(y.isfinite(), code, 0x7F).to(torch.uint8)


def smallest_scale(a: float) -> float:
    """The smallest power of two from 2^-64 on with a <= 448 * scale."""
    e = -64
    while a > math.ldexp(448.0, e):
        e += 1
    return math.ldexp(1.0, e)


def _power_above(scale: float) -> float:
    if not scale > 0:
        return math.ldexp(1.0, -64)
    m, e = math.frexp(scale)
    return math.ldexp(1.0, min(120, max(-64, e - 1 if m == 0.5 else e)))


def store_plane(rows, codes, scales, slots):
    """In place on one plane (``codes`` uint8 [blocks, 256, Hkv, D]); a group's rows are taken in the order of the list."""
    flat, hkv = codes.view(-1, *codes.shape[2:]), codes.shape[2]
    groups: dict[int, list[int]] = {}
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < flat.shape[0]:
            groups.setdefault(s // GROUP, []).append(i)
    for g, members in groups.items():
        x = rows[members].double()  # [n, Hkv, D]
        to = [int(slots[i]) for i in members]
        first = min(to) % GROUP
        for h in range(hkv):
            finite = x[:, h][x[:, h].isfinite()]
            need = smallest_scale(float(finite.abs().max()) if finite.numel() else 0.0)
            old = float(scales[g // GROUP, h, g % GROUP])
            now = need if first == 0 else max(need, _power_above(old))
            if first > 0 and now != old:
                below = flat[g * GROUP:g * GROUP + first, h]
                flat[g * GROUP:g * GROUP + first, h] = torch.where(
                    VALUES[below.int()].isnan(), 0x7F, encode((VALUES[below.int()].float() * torch.tensor(old / now).float()).double()))
            for k, s in enumerate(to):
                flat[s, h] = encode(x[k, h] / now)
            scales[g // GROUP, h, g % GROUP] = now


def store_kvcache_fp8_ref(key, value, k_codes, v_codes, k_scale, v_scale, slot_mapping):
    store_plane(key, k_codes, k_scale, slot_mapping)
    store_plane(value, v_codes, v_scale, slot_mapping)


def quantize(plane):
    """Codes and scales of a bf16 plane [blocks, 256, Hkv, D], every group filled."""
    blocks, _, hkv, d = plane.shape
    x = plane.double().view(blocks, GROUP, GROUP, hkv, d)
    most = x.abs().amax((2, 4))  # [blocks, groups, heads]
    scale = torch.tensor([[[smallest_scale(float(a)) for a in g] for g in b] for b in most], dtype=torch.float64)
    codes = encode(x / scale[:, :, None, :, None]).view(plane.shape)
    return codes, scale.transpose(1, 2).float().contiguous()


def gather(codes, scales, table_row, length):
    """[length, Hkv, D] values in 64 bits of a sequence's tokens."""
    n = (length + BLOCK_SIZE - 1) // BLOCK_SIZE
    ids = table_row[:n].long()
    x = VALUES[codes[ids].int()]  # [n, 256, Hkv, D]
    s = scales[ids].double().transpose(1, 2).repeat_interleave(GROUP, 1)[..., None]
    return (x * s).reshape(n * BLOCK_SIZE, *x.shape[2:])[:length]


def attend(q, k, v, scale, seen):
    """q [lq, Hq, D], k and v [lk, Hkv, D], seen [lq, lk]; rows that see nothing give zeros.  Returns the output, and how far a
    kernel may be from it that rounds P to f16 and the output to bf16:
      2^-8 |out|            the output's rounding, half a step
      (2^-11 + 2^-12) A     A = sum p |v| / sum p: every weight's rounding to f16 (half a step, 2^-11), and as much again
                            for half of it: scores and exponentials in 32 bits (their errors are some 2^-18 at |s| < 100)
      2^-33 n max|v| / L    L = sum p / max p: weights below f16's normal range are off by 2^-25.  Prefill: of a largest weight of
                            2^8 at least; decode: of one of 2^12, in a unit at most 4 times the largest scale of a tile,
                            which is 2 times what max|v| calls for at most: 2^-34
      2^-24 max|v|          prefill: a group's scale over the unit is rounded to f16, off by 2^-25 where it is far smaller, times
                            a code of 448 at most; the unit is a tile's largest scale, max|v| / 224 at most
    """
    lq, hq, d = q.shape
    lk, hkv, _ = k.shape
    q, k, v = q.double(), k.double().repeat_interleave(hq // hkv, 1), v.double().repeat_interleave(hq // hkv, 1)
    s = torch.einsum("qhd,khd->hqk", q, k) * scale
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top.isinf(), 0.0, top)), 0.0)
    total = p.sum(-1)
    div = torch.where(total > 0, total, 1.0)
    out = torch.einsum("hqk,khd->qhd", p, v) / div.T[..., None]
    a = torch.einsum("hqk,khd->qhd", p, v.abs()) / div.T[..., None]
    bound = 2.0 ** -8 * out.abs() + 1.5 * 2.0 ** -11 * a + (2.0 ** -33 * lk / div.T[..., None] + 2.0 ** -24) * v.abs().amax()
    return out, bound


def decode_fp8_ref(q, k_codes, v_codes, k_scale, v_scale, context_lens, block_tables, scale):
    """(out, bound) [B, Hq, D] in 64 bits."""
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(context_lens.tolist()):
        if n > 0:
            k, v = gather(k_codes, k_scale, block_tables[b], n), gather(v_codes, v_scale, block_tables[b], n)
            o, e = attend(q[b:b + 1], k, v, scale, torch.ones(1, n, dtype=torch.bool))
            out[b], bound[b] = o[0], e[0]
    return out, bound


def prefill_fp8_ref(q, k_codes, v_codes, k_scale, v_scale, cu_q, cu_k, scale, block_tables):
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(cu_q.numel() - 1):
        q0, q1 = int(cu_q[b]), int(cu_q[b + 1])
        lq, lk = q1 - q0, int(cu_k[b + 1]) - int(cu_k[b])
        if lq == 0 or lk == 0:
            continue
        k, v = gather(k_codes, k_scale, block_tables[b], lk), gather(v_codes, v_scale, block_tables[b], lk)
        seen = torch.arange(lk) <= torch.arange(lq)[:, None] + (lk - lq)
        out[q0:q1], bound[q0:q1] = attend(q[q0:q1], k, v, scale, seen)
    return out, bound


def step_maps_ref(seq_lens, cached_lens, block_tables, free_blocks, num_tokens):
    """(block_tables, cu_q, cu_k, slot_mapping, positions, taken) as lists of the packed step."""
    table = [list(r) for r in block_tables.tolist()]
    free, taken = free_blocks.tolist(), 0
    cu_q, cu_k, slots, positions = [0], [0], [], []
    for b, (n, c) in enumerate(zip(seq_lens.tolist(), cached_lens.tolist())):
        held, need = -(-c // BLOCK_SIZE), -(-n // BLOCK_SIZE)
        for col in range(held, len(table[b])):
            table[b][col] = -1
            if col < need:
                table[b][col] = free[taken] if taken < len(free) else -1
                taken += 1
        for pos in range(c, n):
            block = table[b][pos // BLOCK_SIZE]
            slots.append(block * BLOCK_SIZE + pos % BLOCK_SIZE if block >= 0 else -1)
            positions.append(pos)
        cu_q.append(cu_q[-1] + max(n - c, 0))
        cu_k.append(cu_k[-1] + n)
    pad = num_tokens - len(slots)
    return table, cu_q, cu_k, slots + [-1] * pad, positions + [0] * pad, taken
