"""The operators around a language model, without a GPU: the oracle against torch in 64 bits and published values, and what
the entry points refuse before anything runs on a device."""
import ctypes

import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200 import _lib
from oracle import language_oracle as O


def test_oracle_philox_known_answers():
    # known-answer vectors published with the generator
    ff = [0xFFFFFFFF] * 4
    for counter, key, want in (([0, 0, 0, 0], [0, 0], [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
                               (ff, ff[:2], [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
                               ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
                                [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])):
        assert O.philox4x32(np.array(counter), np.array(key)).tolist() == want


def test_oracle_log_probs_match_torch():
    g = torch.Generator().manual_seed(3)
    z = (torch.randn(7, 11, generator=g, dtype=torch.float64) * 3).requires_grad_()
    tokens = torch.randint(0, 11, (7,), generator=g)
    w = [torch.randn(7, generator=g, dtype=torch.float64) for _ in range(2)] + [torch.randn(7, 3, generator=g, dtype=torch.float64)]
    lp = torch.log_softmax(z / 0.7, -1)
    top = lp.topk(3, -1)
    outs = lp.gather(1, tokens[:, None])[:, 0], -(lp.exp() * lp).sum(1), top.values
    (dz,) = torch.autograd.grad(outs, z, w)
    r = O.token_log_probs(z.detach().numpy(), tokens.numpy(), 3, 0.7)
    for a, b in zip(outs, (r["log_probs"], r["entropy"], r["top_log_probs"])):
        np.testing.assert_allclose(a.detach().numpy(), b, atol=1e-12)
    assert (r["top_tokens"] == top.indices.numpy()).all()
    d, _ = O.token_log_probs_grad(z.detach().numpy(), tokens.numpy(), *(t.numpy() for t in w), temperature=0.7)
    np.testing.assert_allclose(dz.numpy(), d, atol=1e-12)


def test_oracle_embedding_grad_matches_torch():
    g = torch.Generator().manual_seed(4)
    W = torch.randn(9, 5, generator=g, dtype=torch.float64, requires_grad=True)
    tokens, dout = torch.randint(0, 9, (4, 6), generator=g), torch.randn(4, 6, 5, generator=g, dtype=torch.float64)
    out = torch.nn.functional.embedding(tokens, W, padding_idx=2) * 1.5
    (dW,) = torch.autograd.grad(out, W, dout)
    np.testing.assert_allclose(out.detach().numpy(), O.embedding(tokens.numpy(), W.detach().numpy(), 1.5), atol=1e-12)
    np.testing.assert_allclose(dW.numpy(), O.embedding_grad(tokens.numpy(), dout.numpy(), 9, 1.5, 2)[0], atol=1e-12)


def test_cpu_tensors_are_refused():
    x, t = torch.randn(3, 4), torch.zeros(3, dtype=torch.long)
    for call in (lambda: F.embedding(t, x), lambda: F.dropout(x, 0.5, 1), lambda: F.token_log_probs(x, t)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()
    assert F.dropout(x, 0.5, 1, training=False) is x
    for bad in (dict(seed=-1), dict(seed=2 ** 64), dict(seed=1, offset=-1), dict(seed=1, offset=2 ** 64)):
        with pytest.raises(ValueError, match="range"):
            F.dropout(x, 0.5, **bad)


def test_descriptor_layouts_match_the_library():
    # (the library asserts the same sizes when it is compiled)
    assert [ctypes.sizeof(c) for c in (_lib.EmbedDesc, _lib.DropoutDesc, _lib.ScoreDesc)] == [88, 72, 80]


def _desc(cls, **given):
    d = cls()
    for k, v in given.items():
        setattr(d, k, (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v)
    return d


EMBED = dict(dtype=_lib.BF16, token_bits=64, n0=1, n1=8, token_stride=(0, 1), vocab=10, width=16, row_stride=(16, 16), padding=-1, scale=1.0)
DROP = dict(dtype=_lib.BF16, shared=-1, n0=1, n1=4, cols=16, stride=(64, 16), p=0.5, seed=1, offset=0)
SCORE = dict(dtype=_lib.BF16, token_bits=64, n0=1, n1=8, token_stride=(0, 1), vocab=10, logits_stride=(0, 10), ignore=-100, top=2, temperature=1.0)
PTR = 0x10000     # (never touched: every check comes before the first CUDA call)


@pytest.mark.parametrize("change", [dict(dtype=7), dict(token_bits=16), dict(n0=-1), dict(n0=2 ** 20, n1=2 ** 20), dict(vocab=0),
                                    dict(vocab=2 ** 31), dict(width=0)])
def test_embedding_descriptors_refused(change):
    lib = _lib.load()
    d = _desc(_lib.EmbedDesc, **{**EMBED, **change})
    assert lib.blstm_embedding(d, PTR, PTR, PTR, None) == 1
    assert lib.blstm_embedding_grad(d, PTR, PTR, PTR, PTR, 1 << 30, None) == 1
    assert lib.blstm_embedding_grad_workspace(d) == 0


def test_embedding_pointers_refused():
    lib = _lib.load()
    d = _desc(_lib.EmbedDesc, **EMBED)
    for a in ((None, PTR, PTR), (PTR, None, PTR), (PTR, PTR, None), (PTR, PTR + 1, PTR), (PTR, PTR, PTR + 1)):
        assert lib.blstm_embedding(d, *a, None) == 1
    assert lib.blstm_embedding_grad_workspace(d) == 0            # (few tokens)
    d.n1 = 100000
    need = lib.blstm_embedding_grad_workspace(d)
    assert need > 0 and need % 256 == 0
    for a in ((None, PTR, PTR), (PTR, None, PTR), (PTR, PTR, None), (PTR, PTR + 1, PTR)):
        assert lib.blstm_embedding_grad(d, *a, PTR, need, None) == 1
    assert lib.blstm_embedding_grad(d, PTR, PTR, PTR, None, need, None) == 3
    assert lib.blstm_embedding_grad(d, PTR, PTR, PTR, PTR + 16, need, None) == 3
    assert lib.blstm_embedding_grad(d, PTR, PTR, PTR, PTR, 256, None) == 3
    assert lib.blstm_embedding(None, PTR, PTR, PTR, None) == 1
    assert lib.blstm_embedding(_desc(_lib.EmbedDesc, **{**EMBED, "n1": 0}), None, None, None, None) == 0


@pytest.mark.parametrize("change", [dict(dtype=-1), dict(shared=2), dict(shared=-2), dict(cols=-1), dict(n0=2 ** 20, n1=2 ** 20),
                                    dict(p=-0.1), dict(p=1.5), dict(p=float("nan"))])
def test_dropout_descriptors_refused(change):
    assert _lib.load().blstm_dropout(_desc(_lib.DropoutDesc, **{**DROP, **change}), PTR, None, PTR, None) == 1


def test_dropout_pointers_refused():
    lib, d = _lib.load(), _desc(_lib.DropoutDesc, **DROP)
    for x, seed, y in ((None, None, PTR), (PTR, None, None), (PTR + 1, None, PTR), (PTR, PTR + 4, PTR)):
        assert lib.blstm_dropout(d, x, seed, y, None) == 1
    assert lib.blstm_dropout(_desc(_lib.DropoutDesc, **{**DROP, "n1": 0}), None, None, None, None) == 0


@pytest.mark.parametrize("change", [dict(dtype=3), dict(token_bits=8), dict(n1=-2), dict(vocab=0), dict(top=-1), dict(top=33, vocab=100),
                                    dict(top=11), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                                    dict(temperature=float("inf"))])
def test_score_descriptors_refused(change):
    lib, d = _lib.load(), _desc(_lib.ScoreDesc, **{**SCORE, **change})
    st = (ctypes.c_int64 * 2)(0, 10)
    assert lib.blstm_token_log_probs(d, PTR, PTR, PTR, PTR, PTR, PTR, PTR, None) == 1
    assert lib.blstm_token_log_probs_grad(d, PTR, PTR, PTR, PTR, PTR, st, PTR, st, PTR, PTR, st, None) == 1


def test_score_pointers_refused():
    lib, d = _lib.load(), _desc(_lib.ScoreDesc, **SCORE)
    for i in range(6):                    # logits, tokens, log_probs, entropy, top_log_probs, top_tokens
        a = [PTR] * 7
        a[i] = None
        assert lib.blstm_token_log_probs(d, *a, None) == 1
    st, other = (ctypes.c_int64 * 2)(0, 10), (ctypes.c_int64 * 2)(0, 11)
    good = [PTR, PTR, PTR, PTR, PTR, st, PTR, st, PTR, PTR, st]
    for i, v in ((0, None), (1, None), (2, None), (3, None), (5, None), (7, None), (9, None), (9, PTR + 2), (10, None), (10, other)):
        a = list(good)
        a[i] = v
        assert lib.blstm_token_log_probs_grad(d, *a, None) == 1
