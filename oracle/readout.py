"""CPU oracle of the readout -- TEST INFRASTRUCTURE ONLY, in float64: the
softmax of dan/readout.py:13-17 over whole rows, from its definition."""
import math

import torch


def log_softmax(x):
    """(log p, logsumexp [N]) of float64 rows. The maximum is subtracted first, so that log p keeps its bits whatever the rows' offset."""
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    z = torch.log(torch.exp(x - m).sum(1, keepdim=True))
    return torch.where(z == -math.inf, -math.inf, (x - m) - z), (m + z)[:, 0]


def token_logprobs(logits, tokens, top=0):
    """(logprobs [N, L], logsumexp, entropy, top_logprobs, top_ids); rows of -inf only: -inf, -inf, 0."""
    x = logits.double()
    logp, lse = log_softmax(x)
    p = logp.exp()
    entropy = -torch.where(p == 0, 0.0, p * logp).sum(1)
    given = torch.where(tokens < 0, 0.0, logp.gather(1, tokens.clamp(0, x.shape[1] - 1)))
    given = torch.where(tokens >= x.shape[1], math.nan, given)
    ids = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    return given, lse, entropy, logp.gather(1, ids), ids


def gradient(logits, tokens, top_ids=None, g=None, g_lse=None, g_entropy=None, g_top=None):
    """The logits' gradient by the formula (finite logits or -inf)."""
    x = logits.double()
    n, vocab = x.shape
    _, _, entropy, _, _ = token_logprobs(x, tokens[:, :0])
    logp, lse = log_softmax(x)
    p = logp.exp()
    grad = torch.zeros_like(x)
    pull = torch.zeros(n, 1, dtype=torch.float64)
    for ids, h in ((tokens, g), (top_ids, g_top)):
        if h is not None:
            h = torch.where(ids < 0, 0.0, h.double())
            grad.scatter_add_(1, ids.clamp(min=0), h)
            pull -= h.sum(1, keepdim=True)
    if g_lse is not None:
        pull += g_lse.double()[:, None]
    grad += p * pull
    if g_entropy is not None:
        grad -= g_entropy.double()[:, None] * torch.where(p == 0, 0.0, p * (logp + entropy[:, None]))
    return torch.where(lse[:, None] == -math.inf, 0.0, grad)
