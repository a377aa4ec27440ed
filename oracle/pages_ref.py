"""Blocks of a cache, entry by entry: what pages.py does, on lists and CPU tensors."""
import torch

BLOCK, GROUP = 256, 16


def blocks_of(tokens):
    return -(-tokens // BLOCK)


def in_use(table, lens):
    """(row, column, id) of the entries below each sequence's last block."""
    width = len(table[0]) if table else 0
    return [(b, c, table[b][c]) for b, n in enumerate(lens) for c in range(blocks_of(max(0, min(n, width * BLOCK))))]


def free_list_ref(table, lens, num_blocks, held=None):
    counts = [max(h, 0) for h in held] if held is not None else [0] * num_blocks
    for _, _, i in in_use(table, lens):
        if 0 <= i < num_blocks:
            counts[i] += 1
    free = [i for i, n in enumerate(counts) if n == 0]
    return counts, free + [-1] * (num_blocks - len(free)), len(free)


def copy_ref(caches, pairs):
    """In place: (src, dst, slots) of every pair that names blocks of the cache."""
    for src, dst, slots in pairs:
        num_blocks = caches[0].shape[-4]
        if not (0 <= src < num_blocks and 0 <= dst < num_blocks):
            continue
        slots = max(0, min(slots, BLOCK))
        for c in caches:
            if c.dtype == torch.float32:
                groups = -(-slots // GROUP)
                c[..., dst, :, :groups] = c[..., src, :, :groups]
            else:
                c = c.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c
                c[..., dst, :slots, :, :] = c[..., src, :slots, :, :]


def fork_ref(table, lens, parents, free):
    """(new table, new lens, blocks taken, copies)."""
    width = len(table[0])
    rows, now, copies, seen, taken = [], [], [], set(), 0
    for p in parents:
        if not 0 <= p < len(lens):
            rows.append([-1] * width)
            now.append(0)
            continue
        n = max(0, min(lens[p], width * BLOCK))
        row = table[p][:blocks_of(n)] + [-1] * (width - blocks_of(n))
        if n % BLOCK and p in seen:
            to = free[taken] if taken < len(free) else -1
            copies.append((row[blocks_of(n) - 1], to, n % BLOCK))
            row[blocks_of(n) - 1] = to
            taken += 1
        seen.add(p)
        rows.append(row)
        now.append(n)
    return rows, now, taken, copies


def compact_ref(table, lens, num_blocks, held=None):
    """(new table, moved_to, live, moves)."""
    counts, _, free = free_list_ref(table, lens, num_blocks, held)
    live = num_blocks - free
    moves = list(zip([i for i in range(live, num_blocks) if counts[i]], [i for i in range(live) if not counts[i]]))
    moved = [i if counts[i] else -1 for i in range(num_blocks)]
    for src, dst in moves:
        moved[src] = dst
    now = [[-1] * len(row) for row in table]
    for b, c, i in in_use(table, lens):
        now[b][c] = moved[i] if 0 <= i < num_blocks else -1
    return now, moved, live, moves
