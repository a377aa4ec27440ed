"""The operators around a paged K/V cache held in 8 bits, as cases that can be timed and compared.

  store    ``store_kvcache_fp8``: new K/V rows to e4m3 codes, one power-of-two scale for every 16 slots and head
  decode   ``decode_paged_fp8``: one query token per sequence over the cache
  step     ``decode_step_fp8``: store of the new token and decode attention in one call
  prefill  ``prefill_varlen_fp8``: packed prompts, causal, over the cache through the block table
  maps     ``step_maps``: block tables, slot map, positions and offsets of a step from the requests' lengths

With ``own`` false a case is computed in plain torch operations in 32 bits.  Lengths belong to a case (they follow from
its own numbers); all values, block placements and queries follow from the seed of ``prepare``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 256   # slots of a cache block
GROUP = 16    # slots that share a scale
LARGEST = 448.0  # of e4m3
SMALLEST_SCALE = 2.0 ** -64

# (query heads, KV heads, head_dim): whole models and one rank's shard of them
SMALL, LARGE, NARROW = (16, 8, 128), (32, 8, 128), (14, 2, 64)


def _case(name, op, heads, batch, cached, new, lengths, padded=0, width=0):
    """``batch`` sequences with cached[0]..cached[1] tokens before the step and new[0]..new[1] of the step; ``padded`` rows
    behind them that stand for no sequence, as in the batch of a captured graph; tables ``width`` blocks wide (0: the widest)."""
    return {"name": name, "op": op, "hq": heads[0], "hkv": heads[1], "d": heads[2], "batch": batch, "cached_lo": cached[0],
            "cached_hi": cached[1], "new_lo": new[0], "new_hi": new[1], "lengths": lengths, "padded": padded, "width": width}


def listed():
    return [
        # one user's chat: a single row of a step, and the smallest call
        _case("store_1", "store", SMALL, 1, (317, 317), (1, 1), 1),
        # a decode step of a full batch, padded to the size of its graph
        _case("store_decode_250", "store", SMALL, 250, (100, 4000), (1, 1), 2, padded=6),
        # a prefill chunk as the scheduler packs it: 16 K tokens of short prompts
        _case("store_prompts_29", "store", SMALL, 29, (0, 0), (100, 1024), 3),
        # a large batch of a model with four query heads to a KV head: bandwidth alone
        _case("decode_128_of_1024-8192", "decode", LARGE, 128, (1023, 8191), (1, 1), 4),
        # two long documents, two KV heads of 64: little work to spread over the GPU
        _case("decode_2_of_100000", "decode", NARROW, 2, (99999, 131071), (1, 1), 5),
        # one user's chat
        _case("step_1_of_317", "step", SMALL, 1, (316, 316), (1, 1), 6),
        # a batch in the middle of its answers, padded to the size of its graph
        _case("step_60_of_100-1024", "step", SMALL, 60, (99, 1023), (1, 1), 7, padded=4),
        # a follow-up question behind a cached conversation
        _case("prefill_25_behind_600", "prefill", SMALL, 1, (600, 600), (25, 25), 8),
        # long prompts, read back through the table
        _case("prefill_4_of_4096", "prefill", SMALL, 4, (0, 0), (4096, 4096), 9),
        # ragged prompts behind shared documents
        _case("prefill_12_behind_cached", "prefill", NARROW, 12, (256, 4096), (100, 2000), 10),
        # the maps of a decode step, tables as wide as the longest sequence allowed
        _case("maps_decode_256", "maps", SMALL, 256, (100, 4000), (1, 1), 11, width=16),
        # the maps of prompts with and without a cached part
        _case("maps_prompts_512", "maps", SMALL, 512, (0, 1500), (1, 512), 12, padded=100, width=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    op = rng.choice(["store", "decode", "step", "prefill", "maps"])
    heads = hq, hkv, d = rng.choice([SMALL, LARGE, NARROW, (4, 1, 128), (7, 1, 64), (16, 16, 64), (64, 8, 128)])
    seed = rng.randrange(1 << 20)
    if op == "maps":
        batch = _log(rng, 1, 512)
        top = _log(rng, 1, 4096)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(4096, 131072 // batch)))
        width = _blocks(top + new) + rng.randrange(4)
        return _unnamed(_case("", op, heads, batch, (0, top), (1, new), seed, rng.randrange(50), width))
    row = hkv * d
    if op == "store":
        batch = _log(rng, 1, 300)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(4096, 16384 * 1024 // (row * batch))))
        cached = _log(rng, 1, 2000)
        return _unnamed(_case("", op, heads, batch, (0, cached), (1, new), seed, rng.randrange(5)))
    if op == "prefill":
        batch = _log(rng, 1, 24)
        new = _log(rng, 2, max(2, min(4096, int(math.sqrt(1.0e9 / (hq * batch))))))
        cached = rng.choice([0, _log(rng, 1, 4096)])
        cached = min(cached, int(1.0e9 / (hq * batch * new)))
        return _unnamed(_case("", op, heads, batch, (cached // 4, cached), (max(1, new // 3), new), seed))
    batch = _log(rng, 1, 200)
    most = (0.25e9 if op == "step" else 0.5e9) / (row * batch)
    ctx = _log(rng, 1, max(2, min(131072, int(most))))
    return _unnamed(_case("", op, heads, batch, (ctx // 4, ctx), (1, 1), seed, rng.choice([0, 0, 3])))


def _lengths(case):
    """(tokens cached before the step, tokens of the step) of every sequence."""
    r = random.Random(case["lengths"])
    return [(r.randint(case["cached_lo"], case["cached_hi"]), r.randint(case["new_lo"], case["new_hi"])) for _ in range(case["batch"])]


def _blocks(tokens):
    return (tokens + BLOCK - 1) // BLOCK


# ---- inputs ---------------------------------------------------------------------------------

def _power_of_two(a):
    """Smallest power of two s, no less than SMALLEST_SCALE, with a <= 448 s."""
    m, e = torch.frexp(a / LARGEST)
    return torch.ldexp(torch.ones_like(a), torch.where(m == 0.5, e - 1, e)).clamp_(min=SMALLEST_SCALE)


def _filled(gen, num_blocks, hkv, d, live):
    """A cache plane with data in the slots that ``live`` marks, and what an earlier owner left in the others."""
    x = torch.randn(num_blocks, BLOCK // GROUP, GROUP, hkv, d, device=DEVICE, generator=gen)
    x *= torch.exp(0.5 * torch.randn(num_blocks, BLOCK // GROUP, GROUP, 1, 1, device=DEVICE, generator=gen))  # tokens differ in size
    x *= 1 + 5 * (torch.rand(hkv, d, device=DEVICE, generator=gen) < 0.04)  # and a few channels stand out
    x = x.bfloat16().float()
    a = (x.abs().amax(-1) * live.view(num_blocks, BLOCK // GROUP, GROUP, 1)).amax(2)  # [blocks, groups, heads]
    scale = torch.where(a > 0, _power_of_two(a), torch.ones_like(a))
    codes = (x / scale[:, :, None, :, None]).clamp_(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    return codes.view(num_blocks, BLOCK, hkv, d), scale.transpose(1, 2).contiguous()


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    hq, hkv, d, padded = case["hq"], case["hkv"], case["d"], case["padded"]
    lens = _lengths(case)
    batch = len(lens)
    cached = torch.tensor([c for c, _ in lens], dtype=torch.int32)
    new = torch.tensor([n for _, n in lens], dtype=torch.int32)
    total = cached + new
    need = [_blocks(c + n) for c, n in lens]
    used = sum(need)
    num_blocks = used + 3
    order = torch.randperm(num_blocks, device=DEVICE, generator=gen).to(torch.int32)
    width = case["width"] or max(need)
    at = torch.tensor([0] + need).cumsum(0)
    col = torch.arange(width).expand(batch, width)
    mine = col < torch.tensor(need)[:, None]
    table = torch.where(mine.to(DEVICE), order[(at[:-1, None] + col).clamp(max=used - 1).to(DEVICE)], -1)
    s = {"case": dict(case), "scale": d ** -0.5}
    if case["op"] == "maps":
        held = (cached + BLOCK - 1) // BLOCK
        s["block_tables"] = torch.where((col < held[:, None]).to(DEVICE), table, -1)
        s["free_blocks"] = torch.randperm(used + 40, device=DEVICE, generator=gen).to(torch.int32) + num_blocks
        s["seq_lens"], s["cached_lens"] = total.to(DEVICE), cached.to(DEVICE)
        s["num_tokens"] = int(new.sum()) + padded
        i32 = dict(dtype=torch.int32, device=DEVICE)
        s["out"] = (torch.empty(batch + 1, **i32), torch.empty(batch + 1, **i32), torch.empty(s["num_tokens"], **i32),
                    torch.empty(s["num_tokens"], dtype=torch.int64, device=DEVICE), torch.empty(1, **i32))
        return s

    bf16 = dict(dtype=torch.bfloat16, device=DEVICE, generator=gen)
    storing = case["op"] in ("store", "step")
    in_cache = cached if storing else total  # tokens of each sequence that the cache holds before the call
    pos = torch.arange(width * BLOCK).expand(batch, -1)
    there = (pos < in_cache[:, None]).view(batch, width, BLOCK).to(DEVICE)
    live = torch.zeros(num_blocks + 1, BLOCK, dtype=torch.bool, device=DEVICE)
    live[torch.where(table < 0, num_blocks, table).long().view(-1)] = there.reshape(-1, BLOCK)
    s["k_cache"], s["k_scale"] = _filled(gen, num_blocks, hkv, d, live[:-1])
    s["v_cache"], s["v_scale"] = _filled(gen, num_blocks, hkv, d, live[:-1])
    if storing:
        n = int(new.sum())
        qkv = torch.randn(n + padded, (hq + 2 * hkv) * d, **bf16) * torch.exp(0.5 * torch.randn(n + padded, 1, **bf16))
        q, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=-1)
        s["key"], s["value"] = k.unflatten(-1, (hkv, d)), v.unflatten(-1, (hkv, d))  # strided views, as a model hands them over
        seq = torch.repeat_interleave(torch.arange(batch), new.long())
        starts = torch.cat([torch.zeros(1, dtype=torch.long), new.long().cumsum(0)])
        p = cached.long()[seq] + torch.arange(n) - starts[seq]
        slots = table[seq.to(DEVICE), (p // BLOCK).to(DEVICE)] * BLOCK + (p % BLOCK).to(DEVICE)
        s["slot_mapping"] = torch.cat([slots.to(torch.int32), torch.full((padded,), -1, dtype=torch.int32, device=DEVICE)])
    if case["op"] in ("decode", "step"):
        s["q"] = q.unflatten(-1, (hq, d)) if storing else torch.randn(batch + padded, hq, d, **bf16)
        s["context_lens"] = torch.cat([total, torch.zeros(padded, dtype=torch.int32)]).to(DEVICE)
        s["block_tables"] = torch.cat([table, torch.full((padded, width), -1, dtype=torch.int32, device=DEVICE)])
    if case["op"] == "prefill":
        s["q"] = torch.randn(int(new.sum()), hq, d, **bf16)
        zero = torch.zeros(1, dtype=torch.int32)
        s["cu_seqlens_q"] = torch.cat([zero, new.cumsum(0).to(torch.int32)]).to(DEVICE)
        s["cu_seqlens_k"] = torch.cat([zero, total.cumsum(0).to(torch.int32)]).to(DEVICE)
        s["max_seqlen_q"], s["max_seqlen_k"] = int(new.max()), int(total.max())
        s["block_tables"] = table
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _store_plain(x, cache, scale, slots):
    """Codes and scales of one plane after the rows ``x`` have gone to ``slots``."""
    num_blocks, _, hkv, d = cache.shape
    groups, n_slots = num_blocks * (BLOCK // GROUP), num_blocks * BLOCK
    ok = slots >= 0
    at = torch.where(ok, slots.long(), n_slots)
    group = torch.where(ok, slots.long() // GROUP, groups)
    x = x.float()
    most = torch.zeros(groups + 1, hkv, device=x.device).scatter_reduce(0, group[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")[:-1]
    first = torch.full((groups + 1,), GROUP, device=x.device).scatter_reduce(0, group, at % GROUP, "amin")[:-1]
    old = scale.transpose(1, 2).reshape(groups, hkv)
    need = _power_of_two(most)
    now = torch.where((first == 0)[:, None], need, torch.maximum(need, old))
    now = torch.where((first < GROUP)[:, None], now, old)
    row = torch.full((n_slots + 1,), -1, device=x.device).scatter(0, at, torch.arange(len(slots), device=x.device))[:-1]
    coded = (x / now[group.clamp(max=groups - 1)][:, :, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn).view(torch.uint8)
    before = cache.view(groups, GROUP, hkv, d)
    kept = (before.float() * (old / now)[:, None, :, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn).view(torch.uint8)
    below = torch.arange(GROUP, device=x.device) < first[:, None]
    codes = torch.where((below & (first < GROUP)[:, None])[:, :, None, None], kept, before.view(torch.uint8)).view(n_slots, hkv, d)
    codes = torch.where((row >= 0)[:, None, None], coded[row.clamp(min=0)], codes)
    return codes.view(cache.shape).view(torch.float8_e4m3fn), now.view(num_blocks, -1, hkv).transpose(1, 2).contiguous()


def _gather_plain(cache, scale, block_tables):
    """[batch, KV heads, tokens, D] in 32 bits of all blocks of the tables."""
    at = block_tables.clamp(min=0).long()
    batch, width = at.shape
    _, _, hkv, d = cache.shape
    x = cache.view(torch.uint8)[at].view(torch.float8_e4m3fn).float().view(batch, width, BLOCK // GROUP, GROUP, hkv, d)
    x *= scale[at].transpose(2, 3)[:, :, :, None, :, None]
    return x.view(batch, width * BLOCK, hkv, d).transpose(1, 2)


def _attend_plain(s, visible, v):
    """Softmax of the scores [..., rows, keys] over the visible keys, times v; rows that see none give zeros."""
    s = s.masked_fill(~visible, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    return p @ v / torch.where(total > 0, total, 1)


def _decode_plain(q, k_cache, v_cache, k_scale, v_scale, context_lens, block_tables, scale):
    batch, hq, d = q.shape
    hkv = k_cache.shape[2]
    k = _gather_plain(k_cache, k_scale, block_tables)
    scores = q.float().view(batch, hkv, hq // hkv, d) @ k.transpose(-1, -2) * scale
    visible = torch.arange(k.shape[2], device=q.device) < context_lens[:, None, None, None]
    out = _attend_plain(scores, visible, _gather_plain(v_cache, v_scale, block_tables))
    return out.reshape(batch, hq, d).bfloat16()


def _prefill_plain(s):
    q, cu_q, cu_k, most = s["q"], s["cu_seqlens_q"].long(), s["cu_seqlens_k"].long(), s["max_seqlen_q"]
    n, hq, d = q.shape
    hkv = s["k_cache"].shape[2]
    batch, lq, lk = len(cu_q) - 1, cu_q.diff(), cu_k.diff()
    i = torch.arange(most, device=q.device)
    rows = q.float()[(cu_q[:-1, None] + i).clamp(max=n - 1)]  # [batch, most, hq, d]
    rows = rows.view(batch, most, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    k = _gather_plain(s["k_cache"], s["k_scale"], s["block_tables"])[:, :, None]
    v = _gather_plain(s["v_cache"], s["v_scale"], s["block_tables"])[:, :, None]
    j = torch.arange(k.shape[3], device=q.device)
    visible = (j <= i[:, None] + (lk - lq)[:, None, None]) & (j < lk[:, None, None])
    out = _attend_plain(rows @ k.transpose(-1, -2) * s["scale"], visible[:, None, None], v)  # [batch, hkv, g, most, d]
    token = torch.arange(n, device=q.device)
    seq = torch.searchsorted(cu_q[1:].contiguous(), token, right=True)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, d)[seq, token - cu_q[seq]].bfloat16()


def _maps_plain(s):
    seq_lens, cached, table, free = s["seq_lens"].long(), s["cached_lens"].long(), s["block_tables"], s["free_blocks"]
    batch, width = table.shape
    zero = torch.zeros(1, dtype=torch.long, device=table.device)
    cu_q = torch.cat([zero, (seq_lens - cached).clamp(min=0).cumsum(0)])
    cu_k = torch.cat([zero, seq_lens.cumsum(0)])
    held, need = (cached + BLOCK - 1) // BLOCK, (seq_lens + BLOCK - 1) // BLOCK
    taken = torch.cat([zero, (need - held).clamp(min=0).cumsum(0)])
    col = torch.arange(width, device=table.device)
    k = taken[:-1, None] + col - held[:, None]
    fresh = torch.where(k < len(free), free[k.clamp(0, len(free) - 1)], -1)
    table = torch.where(col < held[:, None], table, torch.where(col < need[:, None], fresh, -1))
    token = torch.arange(s["num_tokens"], device=table.device)
    seq = torch.searchsorted(cu_q[1:].contiguous(), token, right=True)
    live, seq = seq < batch, seq.clamp(max=batch - 1)
    pos = torch.where(live, cached[seq] + token - cu_q[seq], 0)
    block = table[seq, (pos // BLOCK).clamp(max=width - 1)].long()
    slot = torch.where(live & (block >= 0), block * BLOCK + pos % BLOCK, -1)
    i32 = torch.int32
    return {"block_tables": table, "cu_seqlens_q": cu_q.to(i32), "cu_seqlens_k": cu_k.to(i32), "slot_mapping": slot.to(i32),
            "positions": pos, "blocks_taken": taken[-1:].to(i32)}


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from nano_vllm_b200 import attention as A
        from nano_vllm_b200.step_maps import step_maps
        if op == "maps":
            m = step_maps(s["seq_lens"], s["cached_lens"], s["block_tables"], s["free_blocks"], s["num_tokens"], out=s["out"])
            return {"block_tables": s["block_tables"], **m._asdict()}
        planes = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
        if op == "prefill":
            return {"out": A.prefill_varlen_fp8(s["q"], *planes, s["cu_seqlens_q"], s["cu_seqlens_k"], s["max_seqlen_q"],
                                                s["max_seqlen_k"], s["scale"], s["block_tables"])}
        if op == "decode":
            return {"out": A.decode_paged_fp8(s["q"], *planes, s["context_lens"], s["block_tables"], s["scale"])}
        after = dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), planes))
        if op == "store":
            A.store_kvcache_fp8(s["key"], s["value"], *planes, s["slot_mapping"])
            return after
        return {"out": A.decode_step_fp8(s["q"], s["key"], s["value"], *planes, s["slot_mapping"], s["context_lens"],
                                         s["block_tables"], s["scale"]), **after}
    if op == "maps":
        return _maps_plain(s)
    if op == "prefill":
        return {"out": _prefill_plain(s)}
    planes = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if op == "decode":
        return {"out": _decode_plain(s["q"], *planes, s["context_lens"], s["block_tables"], s["scale"])}
    k_cache, k_scale = _store_plain(s["key"], s["k_cache"], s["k_scale"], s["slot_mapping"])
    v_cache, v_scale = _store_plain(s["value"], s["v_cache"], s["v_scale"], s["slot_mapping"])
    after = {"k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale}
    if op == "store":
        return after
    return {"out": _decode_plain(s["q"], k_cache, v_cache, k_scale, v_scale, s["context_lens"], s["block_tables"], s["scale"]), **after}


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    lens = _lengths(case)
    new = sum(n for _, n in lens)
    if case["op"] == "maps":
        rows = new + case["padded"]
        taken = sum(_blocks(c + n) - _blocks(c) for c, n in lens)
        return {"bytes": 8 * len(lens) + 4 * taken + 8 * len(lens) * case["width"] + 8 * (len(lens) + 1) + 12 * rows + 4, "flops": 0}
    token = 2 * hkv * (d + 4 / GROUP)  # K and V codes and scales of a cached token
    stored = new * (2 * hkv * d * 2 + token + 4)
    if case["op"] == "store":
        return {"bytes": stored, "flops": 0}
    keys = sum(c + n for c, n in lens)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in lens)
    entries = 4 * sum(_blocks(c + n) for c, n in lens) + 8 * len(lens)
    return {"bytes": keys * token + 2 * 2 * (new + case["padded"]) * hq * d + entries + (stored if case["op"] == "step" else 0),
            "flops": 4 * pairs * hq * d}


# ---- the definition, in 64 bits -------------------------------------------------------------------

def _code_values():
    """The value of each of the 256 codes: sign, four bits of exponent (bias 7), three of mantissa; no infinities."""
    values = []
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = math.nan if c & 127 == 127 else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        values.append(-v if c & 128 else v)
    return torch.tensor(values, dtype=torch.float64, device=DEVICE)


def _nearest_code_value(y):
    """y rounded to the values of e4m3, ties to even."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _exact_store(s, what, values):
    """Code values and scales of a plane, group by group of the slots that rows go to."""
    plane, scales, rows = s[what + "_cache"], s[what + "_scale"].double().clone(), s["key" if what == "k" else "value"].double()
    x = values[plane.view(torch.uint8).int()].view(-1, *plane.shape[2:])
    slots = s["slot_mapping"].long()
    rows, slots = rows[slots >= 0], slots[slots >= 0]
    ids, which = torch.unique(slots // GROUP, return_inverse=True)
    slot_of = torch.full((len(ids), GROUP), -1, device=DEVICE)
    slot_of[which, slots % GROUP] = torch.arange(len(slots), device=DEVICE)
    new = slot_of >= 0
    in_group = torch.where(new[:, :, None, None], rows[slot_of.clamp(min=0)], 0)
    m, e = torch.frexp(in_group.abs().amax((1, 3)))  # 448 = 0.875 * 2^9
    need = torch.ldexp(torch.ones_like(m), torch.where(m > 0.875, e - 8, e - 9).clamp(min=-64))
    first = torch.argmax(new.int(), 1)
    b, g = ids // (BLOCK // GROUP), ids % (BLOCK // GROUP)
    old = scales[b, :, g]
    now = torch.where((first == 0)[:, None], need, torch.maximum(need, old))
    places = ids[:, None] * GROUP + torch.arange(GROUP, device=DEVICE)
    have = x[places]
    kept = _nearest_code_value(have * (old / now)[:, None, :, None])
    have = torch.where((torch.arange(GROUP, device=DEVICE) < first[:, None])[:, :, None, None], kept, have)
    x[places] = torch.where(new[:, :, None, None], _nearest_code_value(in_group / now[:, None, :, None]), have)
    scales[b, :, g] = now
    return x.view(plane.shape), scales


def _exact_attention(q, k, v, scale, lq):
    """q [lq, hq, d], k and v [lk, hkv, d] in 64 bits; the last query sees all keys."""
    hq, hkv, lk = q.shape[1], k.shape[1], len(k)
    seen = torch.arange(lk, device=DEVICE) <= torch.arange(lq, device=DEVICE)[:, None] + (lk - lq)
    out = torch.zeros_like(q)
    for h in range(hq):
        p = torch.softmax((q[:, h] @ k[:, h * hkv // hq].T * scale).masked_fill(~seen, -math.inf), -1)
        out[:, h] = p @ v[:, h * hkv // hq]
    return out


def exact(case, seed):
    if case["op"] == "maps":
        return None  # whole numbers
    s = prepare(case, seed)
    values = _code_values()
    if case["op"] in ("store", "step"):
        (k, ks), (v, vs) = _exact_store(s, "k", values), _exact_store(s, "v", values)
        after = {"k_cache": k, "v_cache": v, "k_scale": ks, "v_scale": vs}
        if case["op"] == "store":
            return after
    else:
        after, ks, vs = {}, s["k_scale"].double(), s["v_scale"].double()
        k, v = s["k_cache"].view(torch.uint8), s["v_cache"].view(torch.uint8)

    def sequence(plane, scales, b, n):
        at = s["block_tables"][b, :_blocks(n)].long()
        x = plane[at] if plane.is_floating_point() else values[plane[at].int()]
        x = x * scales[at].transpose(1, 2).repeat_interleave(GROUP, 1)[..., None]
        return x.reshape(-1, *x.shape[2:])[:n]

    q = s["q"].double()
    out, row = torch.zeros_like(q), 0
    for b, (cached, new) in enumerate(_lengths(case)):
        n = cached + new
        out[row:row + new] = _exact_attention(q[row:row + new], sequence(k, ks, b, n), sequence(v, vs, b, n), s["scale"], new)
        row += new
    return {"out": out, **after}
