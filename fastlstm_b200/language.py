"""The operators around a language model of LSTM layers: tokens in, regularisation between the layers, predictions out.

Each is a call on CUDA tensors (float32, float16 or bfloat16) that runs on the current stream, allocates through torch and
is differentiable once.  Invalid arguments raise ValueError.  A token outside of the vocabulary is found on the device: its
embedding or log probability is NaN, its row gives no gradient, and `check_status()` or a later call raises BlstmError.
What a call does on the host is csrc/host_language.cpp; the kernels are csrc/embedding.cu, csrc/dropout.cu and
csrc/log_probs.cu."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib


def _whole(v, name: str, low: int = -2 ** 63, high: int = 2 ** 63 - 1) -> int:
    try:
        n = int(v)
    except (TypeError, ValueError, OverflowError):
        n = None
    if n is None or n != v:
        raise ValueError(f"{name} must be a whole number, got {v!r}")
    if not low <= n <= high:
        raise ValueError(f"{name} must be a whole number in the range [{low}, {high}], got {n}")
    return n


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * weight[tokens]: tokens [...] (int64 or int32, any strides), weight [vocabulary, width] -> [..., width].

    The gradient of the table is dense and in the table's type; equal tokens' rows are added in 32 bits in an order that the
    tokens alone fix (results repeat bit by bit) and rounded once.  padding_idx names a token that gets no gradient."""
    return _lib.host().embedding(tokens, weight, float(scale), None if padding_idx is None else _whole(padding_idx, "padding_idx"))


def dropout(x: torch.Tensor, p: float, seed, *, offset: int = 0, shared_dim: Optional[int] = None, training: bool = True) -> torch.Tensor:
    """x with every element set to zero with probability p and divided by 1 - p otherwise.

    The mask is a function of (seed, offset, the element's row-major number): the same for every type, every layout and in
    backward, which draws it again instead of reading it.  Calls that should differ get different offsets (a layer's number,
    say) or seeds; both are whole numbers in [0, 2^64).  seed may also be a CUDA tensor of one int64, read when the kernel
    runs: a captured graph that changes it between replays draws new masks.
    shared_dim: all positions along that dimension share one mask (one mask for all steps of a sequence); the
    product of the dimensions up to it is below 2^31.
    Elements that are dropped are 0 whatever they held."""
    if not training:
        return x
    at = seed if isinstance(seed, torch.Tensor) else None
    return _lib.host().dropout(x, float(p), 0 if at is not None else _whole(seed, "seed", 0, 2 ** 64 - 1), at,
                               _whole(offset, "offset", 0, 2 ** 64 - 1), None if shared_dim is None else _whole(shared_dim, "shared_dim"))


class TokenLogProbs(NamedTuple):
    """What token_log_probs returns; the top fields are None where no alternatives were asked for."""
    log_probs: torch.Tensor                  # [...]      of the given tokens
    entropy: torch.Tensor                    # [...]      of the distribution, in nats
    top_log_probs: Optional[torch.Tensor]    # [..., top] of the likeliest tokens, largest first
    top_tokens: Optional[torch.Tensor]       # [..., top] equal logits in the order of their numbers


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, temperature: float = 1.0,
                    ignore_index: int = -100) -> TokenLogProbs:
    """Log probabilities of `tokens` [...] under softmax(logits / temperature), logits [..., vocabulary], in float32.

    With them the distribution's entropy and, for top > 0 (at most 32), the likeliest tokens; log_probs, entropy and
    top_log_probs are differentiable.  Logits may be strided as long as the vocabulary is dense (a padded one, cut, is).
    Logits of -inf are impossible tokens.  A row of nothing else: log_probs and top_log_probs -inf, entropy 0, the first
    tokens, no gradient.  NaN or +inf in a row makes its results NaN.  Rows whose token is ignore_index count for
    nothing, whatever they hold: log_probs 0, entropy 0, top_log_probs -inf, top_tokens -1, no gradient.  Entropy and alternatives of a row whose token
    is outside of the vocabulary are its own, without a gradient."""
    return TokenLogProbs(*_lib.host().token_log_probs(logits, tokens, _whole(top, "top"), float(temperature),
                                                       _whole(ignore_index, "ignore_index")))
