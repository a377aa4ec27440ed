"""Answers that branch, end to end: beams over a paged cache, each step scored by ``token_logprobs``, forked by ``fork_sequences``,
given blocks by ``free_list`` and ``step_maps``, attended by the decode kernels, compacted on the way; and scored again at the end
by ``head_logprobs``.  What every beam reads back must be the tokens that it has, whatever happened to its blocks."""
import pytest
import torch

from nano_vllm_b200 import _lib, attention as A, pages
from nano_vllm_b200.logprobs import head_logprobs, token_logprobs
from nano_vllm_b200.step_maps import step_maps
from oracle.logprobs_ref import assert_same, head_logprobs_ref

pytestmark = pytest.mark.gpu
HQ, HKV, D, LAYERS, HIDDEN, VOCAB, BLOCKS = 16, 8, 128, 2, 256, 3001, 40
SCALE = D ** -0.5


class Model:
    """Rows of q, k and v by token, a projection of the attention's output, an LM head."""

    def __init__(self, cuda):
        g = torch.Generator("cuda").manual_seed(7)
        r = lambda *s: torch.randn(*s, device=cuda, generator=g).bfloat16()  # noqa: E731
        self.q, self.k, self.v = r(LAYERS, VOCAB, HQ, D), r(LAYERS, VOCAB, HKV, D), r(LAYERS, VOCAB, HKV, D)
        self.out, self.head = r(HQ * D, HIDDEN) / 16, r(VOCAB, HIDDEN) / 4

    def hidden(self, tokens, kv, lens, tables):
        """Of one new token a sequence, whose rows are in the cache."""
        h = 0
        for layer in range(LAYERS):
            o = A.decode_paged(self.q[layer][tokens], kv[0, layer], kv[1, layer], lens, tables, SCALE)
            h = h + o.view(len(tokens), -1) @ self.out
        return h


def store(model, kv, tokens, slots):
    for layer in range(LAYERS):
        A.store_kvcache(model.k[layer][tokens], model.v[layer][tokens], kv[0, layer], kv[1, layer], slots)


def reads_back(model, kv, tables, lens, history):
    for row, n, had in zip(tables.tolist(), lens.tolist(), history):
        assert n == len(had)
        at = torch.tensor([row[t // 256] * 256 + t % 256 for t in range(n)], device=kv.device)
        for i, rows in enumerate((model.k, model.v)):
            for layer in range(LAYERS):
                assert torch.equal(kv[i, layer].view(-1, HKV, D)[at], rows[layer][had])


def test_beams(cuda):
    model, beams = Model(cuda), 5
    kv = torch.zeros(2, LAYERS, BLOCKS, 256, HKV, D, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator().manual_seed(1)
    _lib.read_status()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    # the prompt, of which the last token is the first step's
    prompt = torch.randint(VOCAB, (508,), generator=g).to(cuda)
    tables, lens = torch.full((1, 6), -1, dtype=torch.int32, device=cuda), i32([0])
    free = pages.free_list(tables, lens, BLOCKS)
    m = step_maps(i32([507]), lens, tables, free.free_blocks, 507)
    store(model, kv, prompt[:-1], m.slot_mapping)
    lens, tokens, scores, history = i32([507]), prompt[-1:], torch.zeros(1, device=cuda), [prompt[:-1]]
    states = [[]]  # of every beam, its steps' hidden states and the tokens that followed
    for step in range(14):
        free = pages.free_list(tables, lens, BLOCKS)
        assert free.num_free.item() == BLOCKS - len({b for row, n in zip(tables.tolist(), lens.tolist()) for b in row[:-(-n // 256)]})
        m = step_maps(lens + 1, lens, tables, free.free_blocks, len(tokens))
        store(model, kv, tokens, m.slot_mapping)
        lens = lens + 1
        history = [torch.cat([h, t[None]]) for h, t in zip(history, tokens)]
        reads_back(model, kv, tables, lens, history)
        hidden = model.hidden(tokens, kv, lens, tables)
        logits = hidden @ model.head.T
        best = token_logprobs(logits, tokens, 2 * beams)
        # the same sequences in blocks of their own, in order
        own = torch.arange(len(tokens) * 6, dtype=torch.int32, device=cuda).view(-1, 6)
        plain = torch.zeros(2, LAYERS, len(tokens) * 6, 256, HKV, D, dtype=torch.bfloat16, device=cuda)
        for b, h in enumerate(history):
            store(model, plain, h, torch.arange(len(h), dtype=torch.int32, device=cuda) + b * 6 * 256)
        assert torch.equal(model.hidden(tokens, plain, lens, own), hidden)
        total = (scores[:, None] + best.top_logprobs).flatten()
        scores, which = torch.topk(total, beams)
        parents = which // (2 * beams)
        tokens = best.top_tokens.flatten()[which]
        states = [states[p] + [(hidden[p], t, best.top_logprobs.flatten()[w])] for p, t, w in zip(parents.tolist(), tokens, which.tolist())]
        history = [history[p] for p in parents.tolist()]
        free = pages.free_list(tables, lens, BLOCKS)
        f = pages.fork_sequences((kv,), tables, lens, parents.to(torch.int32), free.free_blocks)
        tables, lens = f.block_tables, f.seq_lens
        reads_back(model, kv, tables, lens, history)
        if step % 5 == 3:
            c = pages.compact_blocks((kv,), tables, lens)
            tables = c.block_tables
            kv[:, :, c.num_live.item():] = torch.nan  # nothing of it is read again
            reads_back(model, kv, tables, lens, history)
    assert len({tuple(h.tolist()) for h in history}) >= 1 and lens.tolist() == [521] * beams
    assert len({row[2] for row in tables.tolist()}) == beams  # the begun block is each beam's own
    # the beams' tokens scored from their hidden states
    for path, score in zip(states, scores.tolist()):
        x = torch.stack([h for h, _, _ in path])
        t = torch.stack([t for _, t, _ in path])
        got = head_logprobs(x, model.head, t)
        given, entropy, bounds = head_logprobs_ref(x.cpu(), model.head.cpu(), t.cpu())
        assert_same(got.logprobs, given, bounds[0], "logprobs")
        # its steps' own scores went by logits rounded to bf16: each half a step of 2^-8 of the largest
        largest = (x.float() @ model.head.float().T).abs().amax(-1).cpu()
        steps = torch.stack([s for _, _, s in path]).cpu()
        assert bool(((steps - given).abs() <= 2 * largest * 2.0 ** -8 + bounds[0]).all())
        assert abs(steps.double().sum().item() - score) <= 2.0 ** -20 * abs(score) * len(path)
    assert _lib.read_status() == 0


@pytest.mark.parametrize("prompts,each", [(3, 4), (1, 16)])
def test_answers_of_prompts_over_a_cache_in_8_bits(cuda, prompts, each):
    """Forked answers over e4m3 planes and scales: they go on with steps of their own, and read what a cache of their own would hold."""
    g = torch.Generator("cuda").manual_seed(prompts)
    rows = prompts * each
    blocks = prompts * 3 + 3 * rows
    lens = torch.randint(200, 600, (prompts,), generator=torch.Generator().manual_seed(2)).tolist()
    lens[0] = 512  # whole blocks only: nothing to copy
    planes = tuple(torch.zeros(1, blocks, 256, HKV, D, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn) for _ in range(2))
    scales = tuple(torch.ones(1, blocks, HKV, 16, device=cuda) for _ in range(2))
    caches = (*planes, *scales)
    r = lambda *s: torch.randn(*s, device=cuda, generator=g).bfloat16()  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    tables = torch.full((prompts, 4), -1, dtype=torch.int32, device=cuda)
    free = pages.free_list(tables, i32([0] * prompts), blocks)
    m = step_maps(i32(lens), i32([0] * prompts), tables, free.free_blocks, sum(lens))
    k, v = r(sum(lens), HKV, D), r(sum(lens), HKV, D)
    A.store_kvcache_fp8(k, v, *(c[0] for c in caches), m.slot_mapping)
    parents = i32([p for p in range(prompts) for _ in range(each)])
    free = pages.free_list(tables, i32(lens), blocks)
    f = pages.fork_sequences(caches, tables, i32(lens), parents, free.free_blocks)
    assert f.blocks_taken.item() == (each - 1) * sum(n % 256 > 0 for n in lens)
    tables, now = f.block_tables, f.seq_lens
    # every answer in a cache of its own
    apart = (*(torch.zeros(rows * 4, 256, HKV, D, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn) for _ in range(2)),
             *(torch.ones(rows * 4, HKV, 16, device=cuda) for _ in range(2)))
    own = torch.arange(rows * 4, dtype=torch.int32, device=cuda).view(rows, 4)
    starts = [sum(lens[:p]) for p in range(prompts + 1)]
    for row, p in enumerate(parents.tolist()):
        A.store_kvcache_fp8(k[starts[p]:starts[p + 1]], v[starts[p]:starts[p + 1]], *apart, torch.arange(lens[p], dtype=torch.int32, device=cuda) + row * 1024)
    for step in range(20):
        free = pages.free_list(tables, now, blocks)
        m = step_maps(now + 1, now, tables, free.free_blocks, rows)
        q, nk, nv = r(rows, HQ, D), r(rows, HKV, D) * (1 + step % 3), r(rows, HKV, D)
        now = now + 1
        out = A.decode_step_fp8(q, nk, nv, *(c[0] for c in caches), m.slot_mapping, now, tables, SCALE)
        slots = (torch.arange(rows, device=cuda) * 1024 + now - 1).to(torch.int32)
        want = A.decode_step_fp8(q, nk, nv, *apart, slots, now, own, SCALE)
        assert torch.equal(out, want)
        if step == 10:
            c = pages.compact_blocks(caches, tables, now)
            tables = c.block_tables
    assert _lib.read_status() == 0


def test_beams_stay_apart(cuda):
    """What each beam has, read from the cache, and the token chosen for it: no two are the same, as no two (parent, token) pairs are."""
    model, beams = Model(cuda), 6
    kv = torch.zeros(2, LAYERS, BLOCKS, 256, HKV, D, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator().manual_seed(3)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    prompt = torch.randint(VOCAB, (251,), generator=g).to(cuda)
    tables, lens, tokens, scores = torch.full((1, 3), -1, dtype=torch.int32, device=cuda), i32([0]), prompt[-1:], torch.zeros(1, device=cuda)
    m = step_maps(i32([250]), lens, tables, pages.free_list(tables, lens, BLOCKS).free_blocks, 250)
    store(model, kv, prompt[:-1], m.slot_mapping)
    lens = i32([250])
    ids = {tuple(row): t for t, row in enumerate(model.k[0, :, 0, :8].view(torch.int16).tolist())}
    assert len(ids) == VOCAB  # a token's key tells which it is
    for step in range(9):
        m = step_maps(lens + 1, lens, tables, pages.free_list(tables, lens, BLOCKS).free_blocks, len(tokens))
        store(model, kv, tokens, m.slot_mapping)
        lens = lens + 1
        best = token_logprobs(model.hidden(tokens, kv, lens, tables) @ model.head.T, tokens, 2 * beams)
        scores, which = torch.topk((scores[:, None] + best.top_logprobs).flatten(), beams)
        parents, tokens = which // (2 * beams), best.top_tokens.flatten()[which]
        f = pages.fork_sequences((kv,), tables, lens, parents.to(torch.int32), pages.free_list(tables, lens, BLOCKS).free_blocks)
        tables, lens = f.block_tables, f.seq_lens
        paths = set()
        for row, n, token in zip(tables.tolist(), lens.tolist(), tokens.tolist()):
            at = torch.tensor([row[t // 256] * 256 + t % 256 for t in range(n)], device=cuda)
            had = [ids[tuple(k)] for k in kv[0, 0].view(-1, HKV, D)[at, 0, :8].view(torch.int16).tolist()]
            assert had[:251] == prompt.tolist()
            paths.add((*had, token))
        assert len(paths) == beams, f"step {step}"
