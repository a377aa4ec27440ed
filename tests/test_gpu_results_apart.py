"""`out` of the scoring and page calls: results that lie on one another or on what is still read are refused, in place is fine where a
row's result takes the place of what the row alone has read."""
import pytest
import torch

from nano_vllm_b200.logprobs import head_logprobs, token_logprobs
from nano_vllm_b200.pages import compact_blocks, fork_sequences, free_list

pytestmark = pytest.mark.gpu


def test_token_logprobs(cuda):
    g = torch.Generator("cuda").manual_seed(1)
    logits = torch.randn(300, 5000, device=cuda, generator=g)
    tokens, t = torch.randint(5000, (300,), device=cuda, generator=g), torch.rand(300, device=cuda, generator=g) + 0.5
    want = token_logprobs(logits, tokens, 1, t)
    for top in (1, 2):
        out = [torch.empty_like(x) for x in token_logprobs(logits, tokens, top, t)]
        wide = torch.zeros(301, device=cuda)
        for change in ({1: out[0]}, {0: out[3].view(-1)[:300]}, {0: logits.view(-1)[4000:4300]}, {1: logits[299, -300:]},
                       {0: tokens.view(torch.float32)[:300]}, {0: wide[:300], 1: wide[1:]}):
            bad = [change.get(i, x) for i, x in enumerate(out)]
            with pytest.raises(AssertionError, match="may not lie on"):
                token_logprobs(logits, tokens, top, t, bad)
        for shifted in (wide[:300], wide[1:]):
            other = wide[1:] if shifted.data_ptr() == wide.data_ptr() else wide[:300]
            with pytest.raises(AssertionError, match="arguments"):
                token_logprobs(logits, tokens, top, shifted, [other, *out[1:]])
    with pytest.raises(AssertionError, match="arguments"):
        wide = torch.zeros(300, 2, dtype=torch.int64, device=cuda)
        token_logprobs(logits, wide.view(-1)[:300], 2, t, [out[0], out[1], wide, out[3]])
    k, at = tokens.clone(), t.clone()  # the next tokens in the place of the last ones, a score in the place of a temperature
    got = token_logprobs(logits, k, 1, at, [at, out[1], k.view(300, 1), torch.empty(300, 1, device=cuda)])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(k, want.top_tokens[:, 0])


def test_head_logprobs(cuda):
    g = torch.Generator("cuda").manual_seed(2)
    x, w = (torch.randn(n, 128, device=cuda, generator=g).bfloat16() for n in (300, 900))
    tokens, t = torch.randint(900, (300,), device=cuda, generator=g), torch.rand(300, device=cuda, generator=g) + 0.5
    want = head_logprobs(x, w, tokens, t)
    out = [torch.empty_like(v) for v in want]
    for bad in ((out[0], out[0]), (x.view(torch.float32).view(-1)[:300], out[1]), (out[0], w.view(torch.float32).view(-1)[-300:]),
                (tokens.view(torch.float32)[:300], out[1])):
        with pytest.raises(AssertionError, match="may not lie on"):
            head_logprobs(x, w, tokens, t, bad)
    at = t.clone()
    got = head_logprobs(x, w, tokens, at, (out[0], at))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_pages(cuda):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    c = torch.zeros(1, 6, 256, 1, 8, dtype=torch.bfloat16, device=cuda)
    table, lens, one = i32(0, 1).view(1, 2), i32(300), i32(0)
    f, k, m = free_list(table, lens, 6), fork_sequences((c,), table, lens, one, i32(4, 5)), compact_blocks((c,), table, lens)
    for call in (lambda: free_list(table, lens, 6, None, (f[0], f[0], f[2])), lambda: free_list(table, lens, 6, None, (f[0], f[1], f[1][:1])),
                 lambda: fork_sequences((c,), table, lens, one, i32(4, 5), (k[0], k[1], k[1])),
                 lambda: fork_sequences((c,), table, lens, one, i32(4, 5), (k[0], k[0][0, :1], k[2])),
                 lambda: compact_blocks((c,), table, lens, None, (m[0], m[1], m[1][:1]))):
        with pytest.raises(AssertionError, match="may not lie on one another"):
            call()
    held = i32(0, 0, 3, 0, 0, 0)
    got = free_list(table, lens, 6, held, (held, f[1], f[2]))  # counted up in place
    assert got.ref_counts.tolist() == [1, 1, 3, 0, 0, 0] and got.free_blocks.tolist() == [3, 4, 5, -1, -1, -1] and got.num_free.tolist() == [3]
