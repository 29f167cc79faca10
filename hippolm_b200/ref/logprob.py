"""Pure-PyTorch oracle of the per-token scores (CPU execution path + test reference)."""
from __future__ import annotations

import torch


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0):
    """Log probability of ``ids[t]`` (0 where it is outside the vocabulary), entropy, and the ``top_k`` largest log probabilities with
    their tokens (descending, the lowest token first among equal ones; NaN counts as largest). Differentiable in the first two.
    A row of -inf only has log probability -inf, entropy 0 and no gradient."""
    z = logits.float()
    V = z.shape[-1]
    empty = (z == float("-inf")).all(-1)
    lp = torch.log_softmax(torch.where(empty.unsqueeze(1), 0.0, z), -1)
    scored = (ids >= 0) & (ids < V)
    own = lp.gather(1, ids.clamp(0, V - 1).unsqueeze(1)).squeeze(1)
    logprob = torch.where(scored, torch.where(empty, float("-inf"), own), 0.0)
    p = lp.exp()
    ent = -(p * torch.where(p == 0, 0.0, lp)).sum(-1)
    ent = torch.where(empty, 0.0, ent)
    if top_k == 0:
        return logprob, ent, None, None
    with torch.no_grad():
        idx = torch.sort(z + 0.0, dim=-1, descending=True, stable=True).indices              # NaN sorts first, equal values by index
        top = idx[:, :top_k]
        return logprob, ent, torch.where(empty.unsqueeze(1), float("-inf"), lp.gather(1, top)), top
