"""How exact head_logprobs is over many rows: what its sums lose on average, and by how much its results scatter.

The bounds of single elements (oracle/logprobs_ref.py) hold for the worst order of signs, hundreds of times what happens.  These
hold for rows of random states.  A sum of H products is cut once for 16 of them, by 0 to 1 last places of what it is by then: half a
last place on average, which the kernel makes good, and sqrt(1/12) last places around that."""
import math

import pytest
import torch

from nano_vllm_b200.logprobs import head_logprobs
from oracle.logprobs_ref import assert_same, logprobs_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
# The logits' mean relative error.  The loss of a step is known in two digits (1.5e-8: half a unit of the last one, 5e-10, for 63
# steps), the scale that makes it good is rounded to fp32 (2^-24), and of 2048 rows whose results scatter by 2e-6 around a spread
# of 3.7 the mean is known to 3 * 2e-6 / (3.7 * sqrt(2048)).
SLOPE = 63 * 5e-10 + U + 3 * 2e-6 / (3.7 * math.sqrt(2048))


def rms(x):
    return x.square().mean().sqrt().item()


@pytest.mark.parametrize("rows", [100, 2048])
@pytest.mark.parametrize("hidden", [64, 512, 1024, 1280, 1472, 1536, 2048, 4096])
def test_states_of_random_rows(cuda, hidden, rows):
    vocab = 50003
    g = torch.Generator("cuda").manual_seed(hidden + rows)
    w = (torch.randn(vocab, hidden, device=cuda, generator=g) * (2.5 / math.sqrt(hidden))).bfloat16()
    tokens = torch.randint(vocab, (rows,), device=cuda, generator=g)
    tokens[:12] = torch.tensor([0, 1, 127, 128, 191, 192, 255, 256, 25000, vocab - 3, vocab - 2, vocab - 1], device=cuda)  # tiles' edges
    x = torch.randn(rows, hidden, device=cuda, generator=g) + 2 * torch.rand(rows, 1, device=cuda, generator=g) * w[tokens].float()
    x = x.bfloat16()
    got = head_logprobs(x, w, tokens)

    z = x.double() @ w.double().T
    log_z = torch.logsumexp(z, -1)
    log_p = z - log_z[:, None]
    p = log_p.exp()
    mean, given, entropy = (p * z).sum(-1), log_p.gather(1, tokens[:, None])[:, 0], -(p * log_p).sum(-1)
    var = (p * (z - mean[:, None]).square()).sum(-1)
    most = z.max(-1).values
    of_token = z.gather(1, tokens[:, None])[:, 0]
    off, off_entropy = got.logprobs.double() - given, got.entropy.double() - entropy

    # Logits all too large by a share s: d logprob = s (z_token - mean), d entropy = -s var
    spread = of_token - mean
    if rows == 2048:
        slope = (off * spread).sum() / spread.square().sum()
        assert abs(slope.item()) <= SLOPE, f"logits are {slope.item():.3g} off on average"
    # A logit's scatter: sqrt(H / 16 / 12) last places of a sum no larger than the logit and the spread of its row.  Then the
    # roundings of (z - m), its product and ln Z, weights that are 2^-22 off, sums of one addition for 32 columns and 60 that join.
    scatter = 2.0 ** -23 * math.sqrt(hidden / 16 / 12) * rms(of_token.abs() + z.std(-1)) + SLOPE * rms(spread)
    y, ln_z = (of_token - most).abs(), log_z - most
    sums = 2.0 ** -22 + math.sqrt(vocab / 32 / 148 + 60) * U
    bound = scatter + sums + U * (rms(2 * y + given.abs()) / math.sqrt(3) + 2 * rms(ln_z))
    assert rms(off) <= bound, f"log probabilities: {rms(off):.3g}, bound {bound:.3g}"
    # An entropy moves by sum p (ln p + entropy) d of its logits' errors d: no more than sqrt(var ln p) of their scatter, which here
    # is that of logits as large as the row's mean; and by the errors of both sums, of which the second is mean (m - z).
    scatter = 2.0 ** -23 * math.sqrt(hidden / 16 / 12) * rms(var.sqrt() * (mean.abs() + var.sqrt())) + SLOPE * rms(var)
    bound = scatter + 2 * sums * rms(1 + (most - mean)) + 2 * U * rms(ln_z + (most - mean))
    assert rms(off_entropy) <= bound, f"entropy: {rms(off_entropy):.3g}, bound {bound:.3g}"


@pytest.mark.parametrize("hidden", [8, 64, 1024, 1536, 4096])
@pytest.mark.parametrize("rows", [100, 300])
def test_sums_that_lose_nothing(cuda, hidden, rows):
    """Logits of one product are exact, and too large by the mean loss that is made good: no more than 63 steps' 1.5e-8."""
    g = torch.Generator().manual_seed(hidden)
    w = (torch.randn(3001, hidden, generator=g) * 2.0).bfloat16()
    tokens = torch.randint(3001, (rows,), generator=g)
    x = torch.zeros(rows, hidden)
    x[torch.arange(rows), torch.randint(hidden, (rows,), generator=g)] = 2.0
    x = x.bfloat16()
    got = head_logprobs(x.to(cuda), w.to(cuda), tokens.to(cuda))
    z = x.double() @ w.double().T
    given, entropy, _, _, (b0, b1, _) = logprobs_ref(z, tokens)
    log_p = z - torch.logsumexp(z, -1, keepdim=True)
    p = log_p.exp()
    mean = (p * z).sum(-1)
    var = (p * (z - mean[:, None]).square()).sum(-1)
    share = (63 * 1.5e-8 + U) * (min(hidden, 1024) > 16)
    assert_same(got.logprobs, given, b0 + share * (z.gather(1, tokens[:, None])[:, 0] - mean).abs(), "logprobs")
    assert_same(got.entropy, entropy, b1 + share * var, "entropy")
