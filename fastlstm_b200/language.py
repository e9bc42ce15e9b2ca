"""The operators around a language model of LSTM layers: tokens in, regularisation between the layers, predictions out.

Each is a call on CUDA tensors (float32, float16 or bfloat16; reorder_states takes any type) that runs on the current stream
and allocates through torch.  embedding, dropout, token_log_probs and rms_norm are differentiable once, the others not.  A backward pass
can be captured as long as no graph from before the capture has the default stream add up its leaves' gradients.  Invalid arguments raise ValueError.  A token outside of the vocabulary is found on the device: its
embedding or log probability is NaN, its row gives no gradient, and `check_status()` or a later call raises BlstmError.
What a call does on the host is csrc/host_language.cpp, csrc/host_norm.cpp and csrc/host_beam.cpp; the kernels are csrc/embedding.cu,
csrc/dropout.cu, csrc/log_probs.cu, csrc/rms_norm.cu and csrc/beam.cu."""
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


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, h = x; with a residual [of x's shape] h = x + residual, and
    the result is (y, h): what goes into the next layer, and the next one's residual.

    h is rounded to the tensors' type before the norm is taken of it.  y and h are dense; all of x, residual and weight are
    differentiable, the weight's gradient is added up in 32 bits in an order that sizes, strides and alignment fix.  Squares are added up in 32
    bits too: rows whose squares come to 2^128 or more (magnitudes from 2^63 on) give zeros, and with an eps of 0 those whose squares vanish (up to 2^-75) infinities."""
    return _lib.host().rms_norm(x, weight, residual, float(eps))


class EightBitRows(NamedTuple):
    """What rms_norm_e4m3 returns: values * scales[..., None] is the norm; sum is None where there was no residual."""
    values: torch.Tensor                     # [..., width] float8_e4m3fn
    scales: torch.Tensor                     # [...]        float32: the row's largest magnitude / 448, or 0
    sum: Optional[torch.Tensor]              # [..., width] x + residual


def rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, *, residual: Optional[torch.Tensor] = None, eps: float = 1e-6) -> EightBitRows:
    """rms_norm with its output in 8 bits and a scale for every row, for products of 8-bit operands; without gradients.

    Values are rounded once, from 32 bits.  A row of zeros, or of magnitudes up to 2^-110, has scale 0 and values 0."""
    return EightBitRows(*_lib.host().rms_norm_e4m3(x, weight, residual, float(eps)))


class BeamStep(NamedTuple):
    """What beam_step returns, the best hypothesis of every sentence first; finished and lengths are None where they were not asked for."""
    scores: torch.Tensor                     # [batch, width] float32: log probabilities of the hypotheses so far
    parents: torch.Tensor                    # [batch, width] int64: the hypothesis each goes on from
    tokens: torch.Tensor                     # [batch, width] int64: what it goes on with
    finished: Optional[torch.Tensor]         # [batch, width] bool: whether it has ended, with this token or before
    lengths: Optional[torch.Tensor]          # [batch, width] int64: tokens up to its end


def beam_step(logits: torch.Tensor, scores: torch.Tensor, *, width: Optional[int] = None, end_token: Optional[int] = None,
              finished: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, length_penalty: float = 0.0) -> BeamStep:
    """The `width` best continuations of every sentence's hypotheses; without gradients.

    logits [batch, hypotheses, vocabulary] are the hypotheses' next predictions, scores [batch, hypotheses] (float32) their log
    probabilities so far; the first step has one hypothesis of score 0 and a width of its own (at most 32; the number of hypotheses by
    default).  A continuation's score is its hypothesis' plus the log softmax of the logits.  A hypothesis in `finished` (bool) goes
    on with end_token alone, at its own score; its logits are not read, nor are those of a hypothesis whose score is -inf.
    With a length_penalty (0 to 4) continuations are ranked by score / length ** length_penalty (scores stay what they are); lengths
    (int64) counts the tokens of hypotheses, to which a continuation adds one unless its hypothesis is finished; in ranks they count
    as 1 at least and 2 ** 24 at most.

    Sums are ranked in 64 bits, equal ones in the order of (hypothesis, token).  Where fewer than `width` continuations are possible,
    impossible ones (score -inf) follow.  NaN or +inf among a hypothesis' logits makes its continuations NaN, which come first."""
    whole = lambda v, name: None if v is None else _whole(v, name)
    return BeamStep(*_lib.host().beam_step(logits, scores, whole(width, "width"), whole(end_token, "end_token"), finished, lengths, float(length_penalty)))


def reorder_states(states, parents: torch.Tensor, *, dim: int = 1):
    """What belongs to hypotheses in the order of those that go on: states [..., batch * hypotheses, ...] -> [..., batch * width, ...] along
    dim, where row b * width + j is row b * hypotheses + parents[b, j].

    states: a tensor or a (nested) list or tuple of tensors of any types, in which `None` stays: the (h, c) [layers, rows, width] of a
    FastLSTM, several of them, and token histories [steps, rows] in one launch.  parents [batch, width] (int64 or int32) are those of
    beam_step.  A parent that is none gives zeros, and `check_status()` or a later call raises BlstmError.  Without gradients."""
    return _lib.host().reorder(states, parents, _whole(dim, "dim"))
