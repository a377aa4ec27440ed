"""The scoring and page calls from several threads at once, each on a stream and on tensors of its own: the same bits as alone."""
import threading

import pytest
import torch

from nano_vllm_b200 import _lib
from nano_vllm_b200.logprobs import head_logprobs, token_logprobs
from nano_vllm_b200.pages import compact_blocks, copy_blocks, fork_sequences, free_list

pytestmark = pytest.mark.gpu


class Work:
    def __init__(self, cuda, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        self.logits = torch.randn(37, 40_003, device=cuda, generator=g).bfloat16()
        self.tokens = torch.randint(3000, (300,), device=cuda, generator=g)
        self.states, self.weight = (torch.randn(n, 1104, device=cuda, generator=g).bfloat16() / 16 for n in (300, 3000))
        self.cache = torch.randn(2, 3, 12, 256, 2, 64, device=cuda, generator=g).bfloat16()
        self.table, self.lens = i32([[7, 3, 9], [1, 4, -1]]), i32([600 + seed, 300])
        self.parents, self.i32 = i32([1, 0, 0, 1]), i32

    def step(self):
        cache = self.cache.clone()
        a = token_logprobs(self.logits, self.tokens[:37], 20)
        b = head_logprobs(self.states, self.weight, self.tokens)
        free = free_list(self.table, self.lens, 12)
        fork = fork_sequences((cache,), self.table, self.lens, self.parents, free.free_blocks)
        moved = compact_blocks((cache,), fork.block_tables, fork.seq_lens)
        copy_blocks((cache,), moved.block_tables[0, :1], self.i32([11]))
        return [*a, *b, *free, *fork, *moved, cache.view(torch.int16)]


def test_threads_with_streams_of_their_own(cuda):
    _lib.read_status()
    work = [Work(cuda, seed) for seed in range(4)]
    want = [w.step() for w in work]
    torch.cuda.synchronize()
    got, errors = [[] for _ in work], []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(12):
                    got[k].append(work[k].step())
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k, steps in enumerate(got):
        assert len(steps) == 12
        for step in steps:
            assert all(torch.equal(a, b) for a, b in zip(step, want[k]))
    assert _lib.read_status() == 0
