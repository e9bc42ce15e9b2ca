"""The root-mean-square norm without a GPU: the oracle against torch in 64 bits, and what the entry points refuse before anything
runs on a device."""
import ctypes

import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200 import _lib
from oracle import language_oracle as O

from test_language import PTR, _desc


def test_oracle_matches_torch():
    g = torch.Generator().manual_seed(1)
    h, w, dy, dh = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 5, 7), (7,), (3, 5, 7), (3, 5, 7)))
    h.requires_grad_(), w.requires_grad_()
    y = torch.nn.functional.rms_norm(h, (7,), w, 1e-6)
    dx, dw = torch.autograd.grad(y, (h, w), dy)
    got = O.rms_norm_grad(h.detach().numpy(), w.detach().numpy(), dy.numpy(), dh.numpy())
    np.testing.assert_allclose(O.rms_norm(h.detach().numpy(), w.detach().numpy())[0], y.detach().numpy(), atol=1e-13)
    np.testing.assert_allclose(got[0], (dx + dh).numpy(), atol=1e-13)
    np.testing.assert_allclose(got[1], dw.numpy(), atol=1e-13)


def test_oracle_rounds_to_e4m3():
    x = torch.cat([torch.linspace(-448, 448, 5003), torch.linspace(-0.1, 0.1, 5003), 2.0 ** -torch.arange(0, 14.0)])
    assert (O.e4m3(x.numpy()) == x.to(torch.float8_e4m3fn).double().numpy()).all()


def test_cpu_tensors_and_wrong_shapes_are_refused():
    x, w = torch.randn(3, 4), torch.randn(4)
    for call in (F.rms_norm, F.rms_norm_e4m3):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call(x, w)


def test_descriptor_layout_matches_the_library():
    assert ctypes.sizeof(_lib.NormDesc) == 80


NORM = dict(dtype=_lib.BF16, eps=1e-6, n0=1, n1=8, width=16, x_stride=(128, 16), residual_stride=(128, 16), dy_stride=(128, 16))


@pytest.mark.parametrize("change", [dict(dtype=5), dict(n0=-1), dict(n0=2 ** 20, n1=2 ** 20), dict(width=0), dict(width=2 ** 31), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(eps=float("inf"))])
def test_descriptors_refused(change):
    lib, d = _lib.load(), _desc(_lib.NormDesc, **{**NORM, **change})
    assert lib.blstm_rms_norm(d, PTR, PTR, PTR, PTR, PTR, PTR, None) == 1
    assert lib.blstm_rms_norm_e4m3(d, PTR, PTR, PTR, PTR, PTR, PTR, None) == 1
    assert lib.blstm_rms_norm_grad(d, PTR, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 1 << 30, None) == 1
    assert lib.blstm_rms_norm_grad_workspace(d) == 0


def test_pointers_refused():
    lib, d = _lib.load(), _desc(_lib.NormDesc, **NORM)
    good = [PTR] * 6                      # x, residual, weight, y, sum, rstd
    for i, v in ((0, None), (1, None), (2, None), (3, None), (4, None), (0, PTR + 1), (1, PTR + 1), (2, PTR + 1), (3, PTR + 1), (4, PTR + 1), (5, PTR + 2)):
        a = list(good)
        a[i] = v
        assert lib.blstm_rms_norm(d, *a, None) == 1
    for i, v in ((0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (4, PTR + 2), (1, PTR + 1)):      # ..., values, scales, sum
        a = list(good)
        a[i] = v
        assert lib.blstm_rms_norm_e4m3(d, *a, None) == 1
    need = lib.blstm_rms_norm_grad_workspace(d)
    assert need > 0 and need % 256 == 0
    good = [PTR] * 7                      # dy, dsum, h, weight, rstd, dx, dweight
    for i, v in ((0, None), (2, None), (3, None), (4, None), (5, None), (0, PTR + 1), (1, PTR + 1), (4, PTR + 2), (5, PTR + 1), (6, PTR + 1)):
        a = list(good)
        a[i] = v
        assert lib.blstm_rms_norm_grad(d, *a, PTR, need, None) == 1
    assert lib.blstm_rms_norm_grad(d, *good, None, need, None) == 3
    assert lib.blstm_rms_norm_grad(d, *good, PTR + 16, need, None) == 3
    assert lib.blstm_rms_norm_grad(d, *good, PTR, need - 1, None) == 3
    empty = _desc(_lib.NormDesc, **{**NORM, "n1": 0})
    assert lib.blstm_rms_norm(empty, *[None] * 6, None) == 0
    assert lib.blstm_rms_norm_grad(empty, *[None] * 8, 0, None) == 0
    assert lib.blstm_rms_norm(None, *good[:6], None) == 1
