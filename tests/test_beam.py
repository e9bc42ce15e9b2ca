"""Beam search without a GPU: the oracle against enumeration, and what the entry points refuse before anything runs on a device."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200 import _lib
from oracle import language_oracle as O

from test_language import PTR, _desc


def test_oracle_finds_the_best_sequences():
    """A width of all sequences that there are keeps them all, in the order of their log probabilities."""
    g = np.random.RandomState(0)
    V, steps = 3, 3
    first, step = g.randn(V), g.randn(V, V)         # logits of the first token, and of the next given the last
    lsm = lambda z: z - np.log(np.exp(z).sum(-1, keepdims=True))
    scores, paths = np.zeros((1, 1)), [()]
    for t in range(steps):
        logits = (first[None] if t == 0 else np.stack([step[p[-1]] for p in paths]))[None]
        s, parents, tokens, _, _ = O.beam_step(logits, scores, min(V ** (t + 1), 27))
        scores, paths = s, [paths[k] + (int(v),) for k, v in zip(parents[0], tokens[0])]
    want = sorted(((lsm(first)[p[0]] + sum(lsm(step)[a][b] for a, b in zip(p, p[1:])), p) for p in itertools.product(range(V), repeat=steps)), reverse=True)
    assert paths == [p for _, p in want]
    np.testing.assert_allclose(scores[0], [s for s, _ in want], atol=1e-12)


def test_oracle_of_ended_and_dead_hypotheses():
    z = np.random.RandomState(1).randn(1, 3, 4)
    z[0, 1] = np.nan
    s, parents, tokens, ended, lengths = O.beam_step(z, np.array([[-1.0, -0.5, -np.inf]]), 6, end=2, finished=np.array([[False, True, False]]),
                                                     lengths=np.array([[3, 2, 3]]))
    assert (parents[0, 0], tokens[0, 0], s[0, 0], ended[0, 0], lengths[0, 0]) == (1, 2, -0.5, True, 2)
    assert parents[0].tolist() == [1, 0, 0, 0, 0, 1] and tokens[0, 5] == 0 and np.isneginf(s[0, 5])


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        F.beam_step(torch.zeros(1, 2, 3), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="CUDA"):
        F.reorder_states([torch.zeros(2, 4)], torch.zeros(2, 2, dtype=torch.long))
    for bad in (dict(width=1.5), dict(end_token=0.5), dict(width=2 ** 70)):
        with pytest.raises(ValueError, match="whole"):
            F.beam_step(torch.zeros(1, 2, 3), torch.zeros(1, 2), **bad)
    with pytest.raises(ValueError, match="lists or tuples"):
        F.reorder_states({"h": torch.zeros(2, 4)}, torch.zeros(2, 2, dtype=torch.long))


def test_descriptor_layouts_match_the_library():
    assert ctypes.sizeof(_lib.BeamDesc) == 64 and ctypes.sizeof(_lib.ReorderItem) == 48


BEAM = dict(dtype=_lib.BF16, width=4, batch=2, beams=3, vocab=10, logits_stride=(30, 10), end_token=1, length_penalty=0.5)


@pytest.mark.parametrize("change", [dict(dtype=4), dict(width=0), dict(width=33, vocab=100), dict(width=31), dict(batch=-1), dict(batch=2 ** 30), dict(beams=0),
                                    dict(beams=33), dict(vocab=0), dict(vocab=2 ** 31), dict(end_token=-2), dict(end_token=10),
                                    dict(length_penalty=-1.0), dict(length_penalty=float("nan")), dict(length_penalty=float("inf")), dict(length_penalty=4.001)])
def test_descriptors_refused(change):
    lib, d = _lib.load(), _desc(_lib.BeamDesc, **{**BEAM, **change})
    assert lib.blstm_beam_step(d, *[PTR] * 10, 1 << 30, None) == 1
    assert lib.blstm_beam_workspace(d) == 0


def test_more_continuations_than_are_counted_are_refused():
    """A sentence's candidates are counted in 32 bits."""
    lib = _lib.load()
    for beams, vocab, fits in ((4, 2 ** 30, False), (32, 2 ** 27, False), (3, 2 ** 31 - 2, False), (4, 2 ** 30 - 1, True), (1, 2 ** 31 - 2, True)):
        d = _desc(_lib.BeamDesc, **{**BEAM, "beams": beams, "vocab": vocab, "logits_stride": (beams * vocab, vocab)})
        assert (lib.blstm_beam_workspace(d) > 0) == fits
        if not fits:
            assert lib.blstm_beam_step(d, *[PTR] * 10, 1 << 30, None) == 1


def test_pointers_refused():
    lib, d = _lib.load(), _desc(_lib.BeamDesc, **BEAM)
    need = lib.blstm_beam_workspace(d)
    assert need > 0 and need % 256 == 0
    good = [PTR] * 9          # logits, scores, finished, lengths, out_scores, parents, tokens, out_finished, out_lengths
    for i, v in ((0, None), (1, None), (3, None), (4, None), (5, None), (6, None), (0, PTR + 1), (1, PTR + 2), (3, PTR + 4), (4, PTR + 2), (5, PTR + 4),
                 (6, PTR + 4), (8, PTR + 4)):
        a = list(good)
        a[i] = v
        assert lib.blstm_beam_step(d, *a, PTR, need, None) == 1
    assert lib.blstm_beam_step(_desc(_lib.BeamDesc, **{**BEAM, "end_token": -1}), *good, PTR, need, None) == 1
    plain = _desc(_lib.BeamDesc, **{**BEAM, "length_penalty": 0.0})
    assert lib.blstm_beam_step(plain, PTR, PTR, None, None, PTR, PTR, PTR, None, PTR, PTR, need, None) == 1      # out_lengths without lengths
    for ws, n in ((None, need), (PTR + 16, need), (PTR, need - 1)):
        assert lib.blstm_beam_step(d, *good, ws, n, None) == 3
    assert lib.blstm_beam_step(_desc(_lib.BeamDesc, **{**BEAM, "batch": 0}), *[None] * 10, 0, None) == 0


def test_reorder_refused():
    lib = _lib.load()

    def call(n=1, parents=PTR, bits=64, batch=2, beams=3, width=4, **given):
        item = (_lib.ReorderItem * 1)(_lib.ReorderItem(**{**dict(src=PTR, dst=PTR, outer=1, inner_bytes=8, outer_stride=0, row_stride=8), **given}))
        return lib.blstm_reorder(item if n else None, abs(n), parents, bits, batch, beams, width, None) if n >= 0 else lib.blstm_reorder(
            item, n, parents, bits, batch, beams, width, None)
    for bad in (dict(n=-1), dict(parents=None), dict(parents=PTR + 4), dict(bits=16), dict(batch=-1), dict(beams=0), dict(width=0), dict(batch=2 ** 30),
                dict(src=None), dict(dst=None), dict(outer=-1), dict(inner_bytes=-1), dict(inner_bytes=2 ** 40)):
        assert call(**bad) == 1, bad
    assert lib.blstm_reorder(None, 1, PTR, 64, 2, 3, 4, None) == 1
    assert call(n=0) == 0 and call(outer=0) == 0 and call(batch=0, parents=None) == 0


def test_reorder_of_rows_near_2_to_the_32_pieces_is_refused():
    """The kernel counts a row's pieces, and 512 more at a time, in 32 bits."""
    lib = _lib.load()
    for odd in (2 ** 32 - 1, 2 ** 32 - 511, 2 ** 32 + 1):                # in pieces of one byte
        item = (_lib.ReorderItem * 1)(_lib.ReorderItem(src=PTR, dst=PTR, outer=1, inner_bytes=odd, outer_stride=0, row_stride=odd))
        assert lib.blstm_reorder(item, 1, PTR, 64, 1, 1, 1, None) == _lib.E_TOO_LARGE
