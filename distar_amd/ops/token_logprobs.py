"""Log probabilities of given tokens, entropy and top alternatives.

One call gives, for each row of logits, the log probability of the row's given
token, the entropy of the row's distribution, and its ``top_k`` likeliest
tokens, from a single reading of the logits; the first two have gradients.  It
takes float32, bfloat16 and float16 logits as they are (no float32 copy) with an
optional mask of allowed tokens and a temperature.  `ops/ce_loss.py` and
`ops/rl_rowwise.py` hold the same quantities one by one for float32 rows.

On a GPU the kernels in `ops/hip/token_logprobs.hip` run; CPU tensors (and
``DISTAR_AMD_DISABLE_HIP=1``) take the eager composition.
"""
import math
from typing import NamedTuple, Optional

import torch

from . import hip_ext

MAX_TOP_K = 64


class TokenLogProbs(NamedTuple):
    logprob: torch.Tensor                    # (...) float32
    entropy: torch.Tensor                    # (...) float32
    top_logprobs: Optional[torch.Tensor]     # (..., k) float32, no gradient
    top_tokens: Optional[torch.Tensor]       # (..., k) int64


def _eager(logits, tokens, mask, temperature, top_k, ignore_index):
    raw = logits if logits.dtype == torch.float64 else logits.float()
    if mask is not None:
        raw = raw.masked_fill(~mask, -math.inf)
    top = raw.detach().amax(-1, keepdim=True)
    empty = top == -math.inf
    gone = raw == -math.inf
    x = (raw.masked_fill(gone, 0.) - top.masked_fill(empty, 0.)) / temperature
    # infinities make NaN as they do in x itself, but never through a gradient
    e = torch.exp(x).masked_fill(gone, 0.)
    total = e.sum(-1, keepdim=True)
    logp = x - torch.log(total.masked_fill(empty, 1.))
    bad = ~torch.isfinite(total) | (top == math.inf)
    p = e / total.masked_fill(empty, 1.)
    entropy = -(p * logp.masked_fill(gone, 0.)).sum(-1)
    # added, not filled in: a masked token's -inf still falls with log(total)
    logp = logp + torch.zeros_like(logp).masked_fill(gone, -math.inf)
    logp = logp.masked_fill(bad, math.nan)
    entropy = entropy.masked_fill(bad.squeeze(-1), math.nan)
    classes = logits.shape[-1]
    inside = (tokens >= 0) & (tokens < classes)
    given = logp.gather(-1, tokens.clamp(0, classes - 1).unsqueeze(-1)).squeeze(-1)
    given = torch.where(inside, given, math.nan)
    logprob = given.masked_fill(tokens == ignore_index, 0.)
    k = min(top_k, classes)
    with torch.no_grad():
        order = torch.sort(raw, dim=-1, descending=True, stable=True)[1][..., :k]
        missing = (raw.gather(-1, order) == -math.inf) | bad
        top_lp = logp.gather(-1, order).masked_fill(missing, -math.inf)
        top_lp = top_lp.masked_fill(bad, math.nan)
        top_t = order.masked_fill(missing, -1)
    out = torch.promote_types(torch.float32, logits.dtype)
    return logprob.to(out), entropy.to(out), top_lp.to(out), top_t


def token_logprobs(logits, tokens, mask=None, temperature=1.0, top_k=0,
                   ignore_index=-100):
    """Log probabilities of `tokens` under ``softmax(logits / temperature)``.

    logits: (..., C) float32, bfloat16 or float16.
    tokens: (...) integers in [0, C), or `ignore_index`.
    mask: bool, broadcast to logits; only tokens where it is True are possible.
        What the logits hold elsewhere (NaN included) has no influence, and no
        gradient.  A logit of -inf counts as masked.
    top_k: 0 to 64 alternatives, the largest logits first, equal ones by index.

    Returns a `TokenLogProbs`.  A row's logprob is 0 (without gradient) where its
    token is `ignore_index`, -inf where the token is masked (with a gradient at the
    possible tokens alone), NaN (without gradient) where it is outside [0, C).  A row
    without any possible token has entropy 0, logprob -inf and no gradient;
    alternatives that do not exist are token -1 with -inf.  A NaN or +inf among a
    row's possible logits makes that row's results NaN (and its alternatives -1).
    """
    ext = hip_ext.maybe_ext(logits)
    if ext is not None:
        return TokenLogProbs(*ext.token_logprobs(logits, tokens, mask, temperature, top_k,
                                                 ignore_index))
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError('logits need a last dimension of at least one element')
    if not logits.is_floating_point():
        raise TypeError(f'logits must be floating point, not {logits.dtype}')
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f'tokens have shape {tuple(tokens.shape)}, but logits have '
                         f'{tuple(logits.shape)}')
    if tokens.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8):
        raise TypeError(f'tokens must be integers, not {tokens.dtype}')
    if mask is not None and mask.dtype != torch.bool:
        raise TypeError(f'mask must be bool, not {mask.dtype}')
    if not 0 <= top_k <= MAX_TOP_K:
        raise ValueError(f'top_k must be 0 to {MAX_TOP_K}, got {top_k}')
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f'temperature must be positive, 1e-30 to 1e30, got {temperature}')
    tokens = tokens.long()
    if mask is not None:
        try:
            mask = mask.expand(logits.shape)
        except RuntimeError:
            raise ValueError(f'mask of shape {tuple(mask.shape)} does not broadcast to '
                             f'logits of shape {tuple(logits.shape)}') from None
    got = _eager(logits, tokens, mask, temperature, top_k, ignore_index)
    return TokenLogProbs(got[0], got[1], *(got[2:] if top_k else (None, None)))
