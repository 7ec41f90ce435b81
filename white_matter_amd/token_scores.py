"""Scores of given tokens under rows of logits: log probability, entropy and
the top alternatives, with the gradient of the logits.

The same numbers serve a draft's verification (the log probability of each
drafted token, the entropy and the alternatives that a sampler takes in its
place) and training on given tokens (their log probabilities and entropy,
differentiated). The HIP path reads each logit once (wmx_score) and in the
gradient once more, writing one value for it (wmx_score_bwd); nothing of the
logits' size is kept between them. The operators are white_matter::token_scores
and white_matter::token_scores_bwd.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native, portable

_native.load_ops()


# token_scores(logits, tokens, top_k, ignore_index) -> (log_probs, entropy,
#     top_log_probs, top_indices, lse), differentiable in logits; and its
#     argument checks alone, for any device
_token_scores = torch.ops.white_matter.token_scores.default
_token_scores_check = torch.ops.white_matter.token_scores_check.default


class TokenLogProbs(NamedTuple):
    """Results of token_log_probs, one row of logits each, float32."""

    log_probs: torch.Tensor  # (...) log probability of the given token
    entropy: torch.Tensor  # (...) of the row's distribution, in nats
    top_log_probs: torch.Tensor  # (..., top_k) log probabilities of the top alternatives
    top_indices: torch.Tensor  # (..., top_k) int64, the alternatives


@torch.library.register_fake("white_matter::token_scores")
def _(logits, tokens, top_k, ignore_index):
    rows = [logits.new_empty(tokens.shape, dtype=torch.float32) for _ in range(3)]
    top = logits.new_empty((*tokens.shape, top_k), dtype=torch.float32)
    return rows[0], rows[1], top, tokens.new_empty((*tokens.shape, top_k), dtype=torch.int64), rows[2]


@torch.library.register_fake("white_matter::token_scores_bwd")
def _(logits, *args):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def token_log_probs(
    logits: torch.Tensor, tokens: torch.Tensor, *, top_k: int = 0, ignore_index: int = -100
) -> TokenLogProbs:
    """Log probabilities of `tokens` under softmax(logits), the entropy of each
    row and its top_k alternatives.

    logits (..., V) float32, bfloat16 or float16, rows of any alignment; tokens
    (...) integer. Arithmetic and results are float32. The alternatives are the
    top_k (up to 32) largest logits in order, equal ones by their index, lowest
    first. Differentiable (once) in logits through log_probs, entropy and
    top_log_probs.

    A token equal to ignore_index (padding) has log probability 0 and takes no
    gradient; another one outside [0, V) has NaN. Logits of -inf (banned
    tokens) have probability 0; a row of nothing else has log probabilities
    -inf, entropy 0 and no gradient. A row with a NaN or +inf has NaN results.
    """
    # (shapes, types and devices are checked by the operator)
    if logits.is_cuda:
        scores = _token_scores(logits, tokens, top_k, ignore_index)
        return TokenLogProbs(scores[0], scores[1], scores[2], scores[3])
    _token_scores_check(logits, tokens, top_k)
    return TokenLogProbs(*portable.token_log_probs_portable(logits, tokens.long(), top_k, ignore_index))
