"""What the entry points of the operators around a language model refuse before anything runs on a device: addresses and numbers
that are none."""
import ctypes

import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200 import _lib

from test_language import EMBED, PTR, SCORE, _desc


@pytest.mark.parametrize("bits,shift", [(64, 4), (64, 1), (32, 2), (32, 1)])
def test_misaligned_tokens_are_refused(bits, shift):
    lib, st = _lib.load(), (ctypes.c_int64 * 2)(0, 10)
    e, s = _desc(_lib.EmbedDesc, **{**EMBED, "token_bits": bits}), _desc(_lib.ScoreDesc, **{**SCORE, "token_bits": bits})
    assert lib.blstm_embedding(e, PTR + shift, PTR, PTR, None) == 1
    assert lib.blstm_embedding_grad(e, PTR + shift, PTR, PTR, None, 0, None) == 1
    assert lib.blstm_token_log_probs(s, PTR, PTR + shift, PTR, PTR, PTR, PTR, PTR, None) == 1
    assert lib.blstm_token_log_probs_grad(s, PTR, PTR + shift, PTR, PTR, PTR, st, PTR, st, PTR, PTR, st, None) == 1


def test_misaligned_results_and_statistics_are_refused():
    lib, st = _lib.load(), (ctypes.c_int64 * 2)(0, 10)
    d = _desc(_lib.ScoreDesc, **SCORE)
    for i, shift in ((2, 2), (3, 2), (4, 2), (5, 4), (6, 2)):        # log_probs, entropy, top_log_probs, top_tokens, stats
        a = [PTR] * 7
        a[i] += shift
        assert lib.blstm_token_log_probs(d, *a, None) == 1
    for i, shift in ((2, 2), (3, 4), (4, 2), (6, 2), (8, 2)):        # stats, top_tokens, g_log_probs, g_entropy, g_top
        a = [PTR, PTR, PTR, PTR, PTR, st, PTR, st, PTR, PTR, st]
        a[i] += shift
        assert lib.blstm_token_log_probs_grad(d, *a, None) == 1


def test_numbers_outside_of_64_bits_are_refused():
    x, t = torch.zeros(3, 4), torch.zeros(3, dtype=torch.long)
    for call in (lambda v: F.embedding(t, x, padding_idx=v), lambda v: F.dropout(x, 0.5, 1, shared_dim=v), lambda v: F.token_log_probs(x, t, top=v),
                 lambda v: F.token_log_probs(x, t, ignore_index=v), lambda v: F.dropout(x, 0.5, v), lambda v: F.dropout(x, 0.5, 1, offset=v)):
        for v in (2 ** 64, -2 ** 64):
            with pytest.raises(ValueError, match="range"):
                call(v)
        with pytest.raises(ValueError, match="whole number"):
            call(1.5)
    with pytest.raises(ValueError, match="CUDA"):
        F.dropout(x, 0.5, 2 ** 64 - 1, offset=2 ** 64 - 1)
