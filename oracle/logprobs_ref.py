"""Log probabilities, entropy and alternatives in 64 bits, and how far 32-bit results may be from them."""
import torch


def logprobs_ref(logits, tokens, top=0, temperatures=None):
    """(logprobs, entropy, top_tokens, top_logprobs, bounds) of CPU tensors; bounds: of the first, the second and the fourth.

    Bounds, with y = (x - m) / T and p the distribution, u = 2^-24 half a step of fp32: a weight exp(y) has three roundings of its
    exponent (|y| u each, and c's own) and its exponential's 2^-22; a sum has `depth` additions one after the other and up to 40
    that join sums or rescale them."""
    x = logits.double()
    rows, vocab = x.shape
    t = torch.ones(rows, dtype=torch.float64)
    if temperatures is not None:
        t = torch.where(temperatures.double() > 0, temperatures.double(), t)
    m = x.max(-1, keepdim=True).values
    y = (x - m) / t[:, None]
    log_z = torch.log(torch.exp(y).sum(-1))
    log_p = y - log_z[:, None]
    p = torch.exp(log_p)
    held = torch.where(p == 0, 0.0, y)
    entropy = log_z - (p * held).sum(-1)
    given = torch.where(tokens < 0, 0.0, log_p.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0])
    given = torch.where(tokens >= vocab, torch.nan, given)
    ranked = torch.where(torch.isnan(x), -torch.inf, x)
    order = torch.sort(ranked, dim=-1, descending=True, stable=True).indices[:, :top]
    u, mean, square = 2.0 ** -24, (p * held.abs()).sum(-1), (p * held * held).sum(-1)
    depth = vocab / 512 + 40
    z = 4 * u * mean + 2.0 ** -22 + depth * u
    of = lambda q: torch.nan_to_num(q.abs(), nan=0.0, posinf=0.0)  # noqa: E731
    alternatives = log_p.gather(1, order)
    bounds = (z + 4 * u * of(y.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0]) + u * of(given) + u * of(log_z),
              z + 2 * mean * (2.0 ** -22 + depth * u) + 4 * u * square + 4 * u * (of(log_z) + mean),
              (z + u * of(log_z))[:, None] + 4 * u * of(y.gather(1, order)) + u * of(alternatives))
    return given, entropy, order, alternatives, bounds


def assert_same(got, want, bound, what):
    """Within the bound where finite, the same infinity or NaN elsewhere."""
    got, want = got.double().cpu(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN at other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: other infinities"
    off = (got - want).abs()[fine]
    assert bool((off <= bound.expand_as(want)[fine]).all()), f"{what}: off by {off.max().item():.3g}"


def head_logprobs_ref(hidden, weight, tokens, temperatures=None):
    """(logprobs, entropy, bounds of both) of CPU tensors.

    Bounds: a logit of H products is off by no more than H / 16 + 20 steps of 2^-23 of the sum of its products' sizes (a tensor core cuts
    its sum once for 16 products, and products of bf16 are exact); sums over the vocabulary as in logprobs_ref, in tiles of up to
    128 columns and 4 x 151936 / 128 of them."""
    x, w = hidden.double(), weight.double()
    given, entropy, _, _, (b0, b1, _) = logprobs_ref(x @ w.T, tokens, 0, temperatures)
    t = torch.ones(len(x), dtype=torch.float64)
    if temperatures is not None:
        t = torch.where(temperatures.double() > 0, temperatures.double(), t)
    off = (hidden.shape[1] / 16 + 20) * 2.0 ** -23 * (x.abs() @ w.abs().T).max(-1).values / t
    # d ln Z <= off; d entropy = sum p (ln p + entropy) d: no more than sqrt(var ln p) off, itself below 2 ln V + 2
    spread = 2 * torch.log(torch.tensor(float(len(w)), dtype=torch.float64)) + 2
    return given, entropy, (b0 + 2 * off, b1 + spread * off)
