"""Log probabilities of given tokens, with entropy and the most probable alternatives.

Both sides of a weight sync compute them: the rollout returns them with the tokens it samples,
the trainer recomputes them on the same tokens and differentiates its policy loss through them.
``WeightSender.check_policy`` compares the two.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._ext import ext

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                  # fp32, the tokens' shape
    entropy: torch.Tensor                   # fp32, the tokens' shape (nats)
    top_logprobs: Optional[torch.Tensor]    # fp32, [..., top_k]; None without top_k
    top_ids: Optional[torch.Tensor]         # int64, [..., top_k]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, vocab: int | None = None, temperature: float = 1.0,
                   top_k: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """``log softmax(logits / temperature)`` at ``tokens``, the entropy of every row and its
    ``top_k`` most probable columns.

    ``logits``: [..., columns] bf16, fp16 or fp32 on a CUDA device; the last dimension is
    contiguous, the leading ones may be strided (``logits[:, :-1]`` is not copied).  ``tokens``:
    int64 or int32, the leading shape.  ``vocab``: how many leading columns are real; the others
    (vocabulary padding) take no part and get a zero gradient.  ``top_k``: 0 to 32 alternatives
    ordered by logit, ties by the lower id (of at most 2^21 columns); they carry no gradient.

    For the tokens one position on, ``logits[:, :-1]`` does for scoring; where a gradient is taken give
    the whole logits and ``ignore_index`` as the last position's token: torch's backward of the
    slice would zero and fill a whole gradient behind the kernel, more than it moves itself.

    Rows whose token is ``ignore_index`` are not read: log probability and entropy 0, gradient
    0, alternatives -1 at -inf.  Columns of -inf have probability 0; a row that has no other is
    empty: log probability -inf, entropy 0, gradient 0.  NaN or +inf in a row, or a token
    outside the vocabulary, make its log probability NaN.

    Differentiable once in ``logits`` through ``logprobs`` and ``entropy``, in reverse mode (a tensor
    with a forward mode derivative is refused); the gradient has the logits' type.  Results are fp32 and held in 32 bits throughout.  Runs on the current stream
    of the logits' device and can be captured into a CUDA graph.
    """
    return TokenLogprobs(*ext().token_logprobs(logits, tokens, vocab, temperature, top_k, ignore_index))
