"""Which tensors of `caches` reach the library, whatever they come in."""
import pytest
import torch

from nano_vllm_b200 import pages


class Host:
    """Stands for the compiled entry points and keeps what they are given."""

    def __getattr__(self, name):
        def call(caches, *args):
            self.caches = list(caches)
            return (0, 0, 0)
        return call


@pytest.mark.parametrize("make", [tuple, list, lambda c: (t for t in c), lambda c: iter(c), lambda c: {i: t for i, t in enumerate(c)}.values()])
def test_every_cache_is_given_on(monkeypatch, make):
    host, i = Host(), torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(pages, "_native", lambda t: host)
    c = [torch.zeros(2, 256, 1, 8, dtype=torch.bfloat16) for _ in range(3)]
    for call in (lambda: pages.copy_blocks(make(c), i, i), lambda: pages.fork_sequences(make(c), i.view(1, 1), i, i, i),
                 lambda: pages.compact_blocks(make(c), i.view(1, 1), i)):
        host.caches = None
        call()
        assert [t.data_ptr() for t in host.caches] == [t.data_ptr() for t in c]
