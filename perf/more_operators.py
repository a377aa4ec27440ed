"""The operators of answers that are scored and branched, as cases that can be timed and compared.

  logprobs  ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives from rows of logits
  head      ``head_logprobs``: log probabilities and entropy from hidden states and the LM head's weight, without logits
  fork      ``fork_sequences``: sequences go on from given ones; whole cache blocks are shared, the begun one is copied
  copy      ``copy_blocks``: blocks of a K/V cache, or their first slots, to other blocks
  compact   ``compact_blocks``: live blocks to the lowest ids
  free      ``free_list``: how often every block is referred to, and which are free

With ``own`` false a case is computed in plain torch operations in 32 bits.  Lengths, parents and the placement of blocks
belong to a case (they follow from its own numbers); all values follow from the seed of ``prepare``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 256  # slots of a cache block
GROUP = 16   # slots that share a scale in a cache held in 8 bits

# (KV heads, head_dim, layers) of the caches
WIDE, NARROW = (8, 128, 28), (2, 64, 24)


def _rows(name, rows, vocab, dtype, top, padded=0, masked=0.0, tempered=False):
    """``padded`` of the rows stand for no sequence; a share ``masked`` of them has most of its logits masked."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "padded": padded,
            "masked": masked, "tempered": tempered}


def _head(name, rows, hidden, vocab, tempered=False):
    return {"name": name, "op": "head", "rows": rows, "hidden": hidden, "vocab": vocab, "tempered": tempered}


def _pages(name, op, cache, eight, batch, lens, lengths, new=0, spare=8, shared=0, width=0):
    """``batch`` sequences of lens[0]..lens[1] tokens, groups of ``shared`` of them behind a common prefix, ``new`` sequences
    or copies, ``spare`` blocks of the cache that no sequence has."""
    return {"name": name, "op": op, "hkv": cache[0], "d": cache[1], "layers": cache[2], "eight": eight, "batch": batch,
            "lo": lens[0], "hi": lens[1], "new": new, "spare": spare, "shared": shared, "width": width, "lengths": lengths}


def listed():
    return [
        # one user's chat that asks for alternatives: a row of a step
        _rows("logprobs_1", 1, 151936, "bfloat16", 20),
        # a decode step of a full batch, rows that start off a 16-byte boundary, padded to the size of its graph
        _rows("logprobs_250", 250, 151643, "bfloat16", 5, padded=6, masked=0.1, tempered=True),
        # beams: 32 bits, two alternatives for each beam and more
        _rows("logprobs_beams_64", 64, 151936, "float32", 32),
        # scores of the tokens of long prompts
        _rows("logprobs_prompts_4096", 4096, 151936, "bfloat16", 1),
        # a step of one user, scored from the hidden state
        _head("head_1", 1, 1024, 151936),
        # a ragged batch of short answers, an odd vocabulary
        _head("head_77", 77, 896, 151643, tempered=True),
        # a prompt of a larger model
        _head("head_1000_wide", 1000, 4096, 151936),
        # four prompts of 1024 tokens
        _head("head_4096", 4096, 1024, 151936),
        # beam search of one prompt: four beams go on from some of them
        _pages("fork_4", "fork", WIDE, False, 4, (1100, 1100), 1, new=4, shared=4),
        # twelve prompts, four answers each: the prompts' begun blocks are copied
        _pages("fork_12_to_48_8bit", "fork", WIDE, True, 12, (300, 2000), 2, new=48, spare=44),
        # a cache after half of its sequences have ended: what is left goes to the front
        _pages("compact_100", "compact", NARROW, False, 100, (100, 4000), 3, spare=700, shared=4),
        # which blocks are free, for the next steps of a full batch
        _pages("free_256", "free", NARROW, False, 256, (100, 4000), 4, spare=2500, shared=4, width=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "head", "head", "fork", "copy", "compact", "free"])
    if op == "logprobs":
        vocab = rng.choice([151936, 151643, 50257, 32000, _log(rng, 100, 160000)])
        dtype = rng.choice(["bfloat16", "float32"])
        rows = _log(rng, 1, max(2, min(5000, int((6.0e8 if dtype == "bfloat16" else 3.0e8) / vocab))))
        case = _rows("", rows, vocab, dtype, min(vocab, rng.choice([0, 1, 5, 20, 64])), min(rows - 1, rng.choice([0, 0, 3])),
                     rng.choice([0.0, 0.3]), rng.random() < 0.3)
    elif op == "head":
        vocab = rng.choice([151936, 151643, 50257, 32000, _log(rng, 100, 160000)])
        hidden = rng.choice([896, 1024, 2048, 4096, 8 * _log(rng, 8, 640)])
        rows = _log(rng, 1, max(2, min(8192, int(6.3e11 / (vocab * hidden)))))
        case = _head("", rows, hidden, vocab, rng.random() < 0.3)
    else:
        eight = rng.random() < 0.4
        hkv, d, layers = cache = rng.choice([WIDE, NARROW, (8, 128, 1), (1, 64, 7), (4, 128, 36), (16, 64, 3)])
        if op == "free":
            batch = _log(rng, 1, 1024)
            hi = _log(rng, 1, max(2, min(131072, 8000000 // batch)))
            case = _pages("", op, cache, eight, batch, (hi // 4, hi), rng.randrange(1 << 20), spare=_log(rng, 1, 20000),
                          shared=rng.choice([0, 3]), width=_blocks(hi) + rng.randrange(20))
        else:
            most = int(2.5e9 / (2 * layers * hkv * BLOCK * d * (1 if eight else 2)))  # blocks
            batch = _log(rng, 1, max(2, min(200, most // 4)))
            hi = _log(rng, 1, max(2, min(8192, most // (2 * batch) * BLOCK)))
            new = _log(rng, 1, max(2, min(256, most // 4)))
            spare = rng.randrange(3, 20) if op == "compact" else new
            if op == "compact" and rng.random() < 0.5:
                spare = max(3, most // 3)
            case = _pages("", op, cache, eight, batch, (hi // 3, hi), rng.randrange(1 << 20), new=new, spare=spare,
                          shared=rng.choice([0, 2, 4]))
    return {k: v for k, v in case.items() if k != "name"}


def _blocks(tokens):
    return (tokens + BLOCK - 1) // BLOCK


# ---- inputs ---------------------------------------------------------------------------------

def _layout(case):
    """Lengths, tables (lists of block ids), ids that no sequence has, blocks of the cache, blocks held for other reasons."""
    r = random.Random(case["lengths"])
    batch, shared = case["batch"], case["shared"]
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(batch)]
    common = [0] * batch  # whole blocks that a sequence has from the first one of its group
    if shared:
        for b in range(batch):
            first = b - b % shared
            common[b] = 0 if b == first else r.randint(0, min(lens[b], lens[first]) // BLOCK)
    need = [_blocks(n) - c for n, c in zip(lens, common)]
    num_blocks = sum(need) + case["spare"]
    order = list(range(num_blocks))
    r.shuffle(order)
    tables, at = [], 0
    for b in range(batch):
        tables.append((tables[b - b % shared][:common[b]] if common[b] else []) + order[at:at + need[b]])
        at += need[b]
    free = order[at:]
    held = free[:len(free) // 10] if case["op"] in ("compact", "free") else []
    return lens, tables, free, num_blocks, held, r


def _forks(case):
    """(parent of every new sequence, (parent, new sequence) of those that need a copy of a begun block)."""
    lens, _, _, _, _, r = _layout(case)
    parents = [b % case["batch"] for b in range(case["new"])]
    if case["new"] <= case["batch"]:  # beams: the best ones go on, some of them twice
        parents = [r.randrange(case["batch"]) for _ in range(case["new"])]
    seen, copies = set(), []
    for i, p in enumerate(parents):
        if lens[p] % BLOCK and p in seen:
            copies.append((p, i))
        seen.add(p)
    return parents, copies


def _copies(case):
    """(source blocks, destination blocks, slots) of a copy."""
    lens, tables, free, _, _, r = _layout(case)
    live = sorted({b for t in tables for b in t})
    n = case["new"]
    src = [r.choice(live) for _ in range(n)] if live else [-1] * n
    slots = [r.choice([BLOCK, r.randint(1, BLOCK)]) for _ in range(n)]
    return src, free[:n], slots


def _moves(case):
    """How many blocks a compaction moves."""
    _, tables, _, _, held, _ = _layout(case)
    live = {b for t in tables for b in t} | set(held)
    return sum(b >= len(live) for b in live)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def _logits(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    dtype = getattr(torch, case["dtype"])
    x = torch.randn(rows, vocab, dtype=dtype, device=DEVICE, generator=gen)
    x *= 1.5 + 1.5 * torch.rand(rows, 1, device=DEVICE, generator=gen).to(dtype)
    tokens = torch.randint(vocab, (rows,), device=DEVICE, generator=gen)
    sure = 12 * torch.rand(rows, device=DEVICE, generator=gen).to(dtype)  # what the model thinks of the token that follows
    x[torch.arange(rows, device=DEVICE), tokens] += sure
    if case["masked"]:  # a grammar that allows a few tokens, or a mask of the type's lowest value
        some = torch.rand(rows, device=DEVICE, generator=gen) < case["masked"]
        share = torch.rand(rows, 1, device=DEVICE, generator=gen) ** 4
        kept = torch.rand(rows, vocab, device=DEVICE, generator=gen) < share
        kept[torch.arange(rows, device=DEVICE), tokens] = True
        low = torch.where(torch.rand(rows, 1, device=DEVICE, generator=gen) < 0.5, -math.inf, torch.finfo(dtype).min).to(dtype)
        x = torch.where(some[:, None] & ~kept, low, x)
    if case["padded"]:
        tokens[rows - case["padded"]:] = -1
    return x, tokens


def _cache(case, num_blocks, gen):
    shape = 2, case["layers"], num_blocks, BLOCK, case["hkv"], case["d"]
    x = torch.randn(shape, dtype=torch.bfloat16, device=DEVICE, generator=gen)
    if not case["eight"]:
        return (x,)
    scale = torch.exp2(torch.randint(-9, -2, (2, case["layers"], num_blocks, case["hkv"], BLOCK // GROUP), device=DEVICE, generator=gen).float())
    return (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)
    s = {"case": dict(case)}
    if case["op"] in ("logprobs", "head"):
        rows = case["rows"]
        if case["op"] == "logprobs":
            s["logits"], s["tokens"] = _logits(case, gen)
        else:
            hidden, vocab = case["hidden"], case["vocab"]
            s["weight"] = torch.randn(vocab, hidden, dtype=torch.bfloat16, device=DEVICE, generator=gen) * (2.5 / math.sqrt(hidden))
            s["tokens"] = torch.randint(vocab, (rows,), device=DEVICE, generator=gen)
            toward = torch.rand(rows, 1, device=DEVICE, generator=gen) * 2.0
            x = torch.randn(rows, hidden, device=DEVICE, generator=gen)
            s["hidden"] = (x + toward * s["weight"][s["tokens"]].float()).bfloat16()
        s["temperatures"] = None
        if case["tempered"]:
            t = 0.3 + 1.2 * torch.rand(rows, device=DEVICE, generator=gen)
            s["temperatures"] = torch.where(torch.rand(rows, device=DEVICE, generator=gen) < 0.2, 0.0, t)  # some rows greedy
        return s
    lens, tables, free, num_blocks, held, _ = _layout(case)
    width = case["width"] or max(1, max(map(len, tables)))
    s["block_tables"] = _i32([t + [-1] * (width - len(t)) for t in tables])
    if case["op"] == "free":  # other blocks of the same cache
        named = torch.randperm(num_blocks, device=DEVICE, generator=gen).to(torch.int32)
        s["block_tables"] = torch.where(s["block_tables"] < 0, -1, named[s["block_tables"].clamp(min=0).long()])
    s["seq_lens"] = _i32(lens)
    s["num_blocks"] = num_blocks
    if case["op"] != "free":
        s["caches"] = _cache(case, num_blocks, gen)
    if case["op"] == "fork":
        s["parents"], s["free_blocks"] = _i32(_forks(case)[0]), _i32(free)
    elif case["op"] == "copy":
        src, dst, slots = _copies(case)
        s["src"], s["dst"], s["slots"] = _i32(src), _i32(dst), _i32(slots)
    else:
        counts = torch.zeros(num_blocks, dtype=torch.int32)
        counts[held] = 1
        s["held"] = counts.to(DEVICE)
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _distribution_plain(logits, tokens, temperatures):
    """(log probabilities of the tokens, entropy, log probability of a logit) in 32 bits."""
    t = torch.ones(len(logits), device=logits.device) if temperatures is None else torch.where(temperatures > 0, temperatures, 1.0)
    most = logits.amax(-1, keepdim=True)

    def scaled(x):
        return (x - most) / t[:, None]

    y = scaled(logits)
    e = torch.exp(y)
    total = e.sum(-1, keepdim=True)
    entropy = torch.log(total) - torch.where(e == 0, 0.0, e * y).sum(-1, keepdim=True) / total

    def log_prob(x):
        return scaled(x) - torch.log(total)

    given = log_prob(logits.gather(1, tokens.clamp(min=0)[:, None]))[:, 0]
    return torch.where(tokens < 0, 0.0, given), entropy[:, 0], log_prob


def _logprobs_plain(s):
    x = s["logits"].float()
    logprobs, entropy, log_prob = _distribution_plain(x, s["tokens"], s["temperatures"])
    ranked = torch.where(torch.isnan(x), -math.inf, x) + 0.0  # one zero
    bits = ranked.view(torch.int32)
    bits = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
    key = (bits << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
    top = 0xFFFFFFFF - (torch.topk(key, s["case"]["top"], dim=-1).values & 0xFFFFFFFF)
    return {"logprobs": logprobs, "entropy": entropy, "top_tokens": top, "top_logprobs": log_prob(x.gather(1, top))}


def _free_plain(block_tables, seq_lens, num_blocks, held):
    col = torch.arange(block_tables.shape[1], device=block_tables.device)
    mine = col < ((seq_lens + BLOCK - 1) // BLOCK)[:, None]
    at = torch.where(mine, block_tables, num_blocks).long().view(-1)
    counts = torch.zeros(num_blocks + 1, dtype=torch.int32, device=at.device).scatter_add(0, at, torch.ones_like(at, dtype=torch.int32))
    counts = counts[:-1] + held
    place = torch.where(counts == 0, (counts == 0).cumsum(0) - 1, num_blocks)
    ids = torch.arange(num_blocks, dtype=torch.int32, device=at.device)
    free = torch.full((num_blocks + 1,), -1, dtype=torch.int32, device=at.device).scatter(0, place, ids)
    free[-1] = -1
    return counts, free[:-1], (counts == 0).sum(dtype=torch.int32)[None], mine


def _copy_plain(caches, src, dst, slots):
    """In place; pairs with a negative block are left out."""
    ok = (src >= 0) & (dst >= 0)
    src, dst, slots = src[ok].long(), dst[ok].long(), slots[ok]
    for c in caches:
        c = c.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c
        if c.dtype == torch.float32:
            kept = torch.arange(BLOCK // GROUP, device=c.device) < ((slots + GROUP - 1) // GROUP)[:, None, None]
        else:
            kept = (torch.arange(BLOCK, device=c.device) < slots[:, None])[:, :, None, None]
        c[:, :, dst] = torch.where(kept, c[:, :, src], c[:, :, dst])


def _fork_plain(s):
    table, lens, parents, free = s["block_tables"], s["seq_lens"], s["parents"].long(), s["free_blocks"]
    new, width = len(parents), table.shape[1]
    ok = (parents >= 0) & (parents < len(lens))
    at = parents.clamp(0, len(lens) - 1)
    now_lens = torch.where(ok, lens[at], 0)
    row = torch.arange(new, device=table.device)
    first = torch.full((len(lens) + 1,), new, device=table.device).scatter_reduce(0, torch.where(ok, at, len(lens)), row, "amin")
    begun = now_lens % BLOCK
    copied = ok & (begun > 0) & (first[at] < row)
    taken = copied.cumsum(0)
    fresh = torch.where(taken <= len(free), free[(taken - 1).clamp(0, len(free) - 1)], -1)
    last = (now_lens + BLOCK - 1) // BLOCK - 1
    col = torch.arange(width, device=table.device)
    now = torch.where(ok[:, None] & (col <= last[:, None]), table[at], -1)
    src = torch.where(copied, now.gather(1, last.clamp(min=0)[:, None].long())[:, 0], -1)
    now = torch.where(copied[:, None] & (col == last[:, None]), fresh[:, None], now)
    _copy_plain(s["caches"], src, torch.where(copied, fresh, -1), begun)
    return {"block_tables": now, "seq_lens": now_lens, "blocks_taken": taken[-1:].to(torch.int32)}


def _compact_plain(s):
    table, num_blocks = s["block_tables"], s["num_blocks"]
    counts, _, _, mine = _free_plain(table, s["seq_lens"], num_blocks, s["held"])
    live = counts > 0
    n = live.sum()
    ids = torch.arange(num_blocks, device=table.device)
    src = ids[live & (ids >= n)]
    dst = ids[~live & (ids < n)]
    moved = torch.where(live, ids, -1)
    moved[src] = dst
    _copy_plain(s["caches"], src, dst, torch.full_like(src, BLOCK))
    now = torch.where(mine, moved[table.clamp(min=0).long()], -1)
    return {"block_tables": now.to(torch.int32), "moved_to": moved.to(torch.int32), "num_live": n.to(torch.int32)[None]}


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from nano_vllm_b200 import logprobs as L
        from nano_vllm_b200 import pages as P
        if op == "logprobs":
            return L.token_logprobs(s["logits"], s["tokens"], s["case"]["top"], s["temperatures"])._asdict()
        if op == "head":
            return L.head_logprobs(s["hidden"], s["weight"], s["tokens"], s["temperatures"])._asdict()
        if op == "free":
            return P.free_list(s["block_tables"], s["seq_lens"], s["num_blocks"], s["held"])._asdict()
        caches = s["caches"]
        if op == "copy":
            P.copy_blocks(caches, s["src"], s["dst"], s["slots"])
            return {"caches": caches}
        if op == "fork":
            return {**P.fork_sequences(caches, s["block_tables"], s["seq_lens"], s["parents"], s["free_blocks"])._asdict(), "caches": caches}
        return {**P.compact_blocks(caches, s["block_tables"], s["seq_lens"], s["held"])._asdict(), "caches": caches}
    if op == "logprobs":
        return _logprobs_plain(s)
    if op == "head":
        logits = s["hidden"].float() @ s["weight"].float().T
        logprobs, entropy, _ = _distribution_plain(logits, s["tokens"], s["temperatures"])
        return {"logprobs": logprobs, "entropy": entropy}
    if op == "free":
        counts, free, n, _ = _free_plain(s["block_tables"], s["seq_lens"], s["num_blocks"], s["held"])
        return {"ref_counts": counts, "free_blocks": free, "num_free": n}
    if op == "copy":
        _copy_plain(s["caches"], s["src"], s["dst"], s["slots"])
        return {"caches": s["caches"]}
    return {**(_fork_plain(s) if op == "fork" else _compact_plain(s)), "caches": s["caches"]}


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("logprobs", "head"):
        rows, vocab = case["rows"], case["vocab"]
        about = 8 * rows + 8 * rows + (4 * rows if case["tempered"] else 0)  # tokens, results, temperatures
        if op == "head":
            return {"bytes": 2 * case["hidden"] * (rows + vocab) + about, "flops": 2 * rows * vocab * case["hidden"]}
        return {"bytes": rows * vocab * (2 if case["dtype"] == "bfloat16" else 4) + about + 12 * rows * case["top"], "flops": 0}
    lens, tables, _, num_blocks, _, _ = _layout(case)
    width = case["width"] or max(1, max(map(len, tables)))
    entries = sum(map(len, tables)) + len(lens)  # of the tables, and the lengths
    slot = 2 * case["layers"] * case["hkv"] * case["d"] * (1 if case["eight"] else 2)
    scales = 2 * case["layers"] * case["hkv"] * 4 if case["eight"] else 0  # of a group of slots

    def moved(slots):  # read and written
        return 2 * sum(n * slot + (n + GROUP - 1) // GROUP * scales for n in slots)

    if op == "free":
        return {"bytes": 4 * entries + 12 * num_blocks + 4, "flops": 0}
    if op == "copy":
        _, _, slots = _copies(case)
        return {"bytes": moved(slots) + 12 * len(slots), "flops": 0}
    if op == "fork":
        parents, copies = _forks(case)
        kept = sum(len(tables[p]) + 1 for p in set(parents))
        return {"bytes": moved([lens[p] % BLOCK for p, _ in copies]) + 4 * (kept + len(parents) * (width + 2) + len(copies) + 1), "flops": 0}
    return {"bytes": moved([BLOCK] * _moves(case)) + 4 * (entries + 2 * num_blocks + len(lens) * width + 1), "flops": 0}


# ---- the definition, in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op not in ("logprobs", "head"):
        return None  # whole numbers and copies
    s = prepare(case, seed)
    tokens, t = s["tokens"], s["temperatures"]
    results = []
    step = max(1, 2**28 // case["vocab"])  # rows at a time
    weight = s["weight"].double() if op == "head" else None
    for i in range(0, case["rows"], step):
        z = s["hidden"][i:i + step].double() @ weight.T if op == "head" else s["logits"][i:i + step].double()
        top = z
        if t is not None:
            z = z / torch.where(t[i:i + step] > 0, t[i:i + step], 1).double()[:, None]
        log_p = z - torch.logsumexp(z, -1, keepdim=True)
        p = torch.exp(log_p)
        k = tokens[i:i + step]
        given = torch.where(k < 0, 0, log_p.gather(1, k.clamp(min=0)[:, None])[:, 0])
        one = [given, -(p * log_p.clamp(min=-1e300)).sum(-1)]
        if op == "logprobs":
            best = torch.sort(torch.topk(top, case["top"], dim=-1).values, -1, descending=True).values
            if t is not None:
                best = best / torch.where(t[i:i + step] > 0, t[i:i + step], 1).double()[:, None]
            one.append(best - torch.logsumexp(z, -1, keepdim=True))
        results.append(one)
    parts = [torch.cat(x) for x in zip(*results)]
    if op == "head":
        return {"logprobs": parts[0], "entropy": parts[1]}
    return {"logprobs": parts[0], "entropy": parts[1], "top_tokens": None, "top_logprobs": parts[2]}
