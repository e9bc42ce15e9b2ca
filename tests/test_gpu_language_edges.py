"""The operators around a language model where their promises end: overlapping rows, addresses, tokens and numbers that are none,
masks held to bounds of their own.  Tolerances as in test_gpu_language.py unless a test derives its own."""
import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200 import _lib
from oracle import language_oracle as O

from test_gpu_language import DT, U, check_dropout, check_scores, gen, make_logits

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- log probabilities
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("vocab,step", [(10, 2), (77, 76), (1300, 8), (6007, 1), (700, 0)])
def test_scores_of_overlapping_rows(vocab, step, dtype):
    """Rows that share elements (windows of one tensor): every row of the gradient is its own."""
    g = gen(30)
    base = make_logits(g, 3 * vocab + 12 * step + 16, dtype=dtype)
    tokens = torch.randint(0, vocab, (12,), generator=g, device="cuda")
    windows = base.as_strided((12, vocab), (step, 1))
    for v, t in ((windows, tokens), (windows[None], tokens[None]), (windows[:, None], tokens[:, None]), (windows.view(3, 4, vocab), tokens.view(3, 4)),
                 (base.as_strided((2, 3, 2, vocab), (step, step, step, 1), 3), tokens.view(2, 3, 2)),
                 (base.as_strided((4, 3, vocab), (step, vocab + 1, 1)), tokens.view(4, 3))):
        check_scores(v, t, dtype, 2)


def test_scores_gradient_of_windows_adds_up_in_the_tensor():
    base = make_logits(gen(31), 400, dtype="fp32").requires_grad_()
    tokens = torch.arange(20, device="cuda")
    (d,) = torch.autograd.grad(F.token_log_probs(base.unfold(0, 210, 10), tokens).log_probs.sum(), base)
    ref = base.detach().double().requires_grad_()
    lp = torch.log_softmax(ref.unfold(0, 210, 10), -1)
    (want,) = torch.autograd.grad(lp.gather(1, tokens[:, None]).sum(), ref)
    # 20 windows, each gradient at most 1 and with distances of up to D = 35 powers of two off by (6 D + 16) u of it
    assert float((d.double() - want).abs().max()) <= 20 * (6 * 35 + 16) * U


@pytest.mark.parametrize("vocab", [40, 100, 129, 300, 700, 1000, 1500, 9000, 40000])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_scores_alternatives_of_rows_with_nan(vocab, dtype):
    """NaN comes before all logits, and equal ones by their number: all NaN; one at number 0 or 1 or the last before equal logits."""
    nan, top = float("nan"), min(32, vocab)
    z = torch.full((4, vocab), 1.5, device="cuda").to(DT[dtype])
    z[0] = nan
    for row, j in ((1, 0), (2, 1), (3, vocab - 1)):
        z[row, j] = nan
    r = F.token_log_probs(z, torch.zeros(4, dtype=torch.long, device="cuda"), top=top)
    want = [list(range(top))] + [([j] + [k for k in range(top + 1) if k != j])[:top] for j in (0, 1, vocab - 1)]
    assert r.top_tokens.tolist() == want
    assert r.log_probs.isnan().all() and r.entropy.isnan().all() and r.top_log_probs.isnan().all()


@pytest.mark.parametrize("vocab,top", [(60, 2), (700, 0), (1500, 3), (5000, 3), (40000, 5)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_scores_of_tokens_outside_of_the_vocabulary_give_no_gradient(vocab, top, dtype):
    """Neither through the entropy nor through the alternatives, which have the row's own values."""
    z = make_logits(gen(32), 5, vocab, dtype=dtype).requires_grad_()
    good = torch.tensor([0, 1, 5, 2, 3], device="cuda")
    want = F.token_log_probs(z, good, top=top)
    n = 3 if top else 2
    ups = [torch.randn(t.shape, generator=gen(33), device="cuda") for t in want[:n]]
    (ref,) = torch.autograd.grad(want[:n], z, ups)
    for bad in (vocab, -1, 2 ** 40):
        tokens = good.clone()
        tokens[2] = bad
        r = F.token_log_probs(z, tokens, top=top)
        with pytest.raises(_lib.BlstmError, match="at position 2"):
            F.check_status()
        assert r.log_probs[2].isnan()
        for a, b in list(zip(r, want))[1:2 + 2 * (top > 0)]:
            assert torch.equal(a, b)
        (d,) = torch.autograd.grad(r[:n], z, ups)
        F.check_status()
        rows = torch.arange(5, device="cuda") != 2
        assert not d[2].any() and torch.equal(d[rows], ref[rows])


# ---------------------------------------------------------------- arguments
def test_scales_beyond_32_bits_are_refused():
    x, t = torch.randn(3, 4, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    for scale in (1e39, -1e300, float("inf")):
        with pytest.raises(ValueError, match="scale must be finite"):
            F.embedding(t, x, scale=scale)


def test_numbers_that_are_none_are_refused():
    x, t = torch.randn(3, 4, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    for call in (lambda v: F.dropout(x, 0.5, v), lambda v: F.dropout(x, 0.5, 1, offset=v), lambda v: F.token_log_probs(x, t, top=v),
                 lambda v: F.token_log_probs(x, t, ignore_index=v), lambda v: F.embedding(t, x, padding_idx=v), lambda v: F.dropout(x, 0.5, 1, shared_dim=v)):
        for v in (0.5, "1", float("nan"), float("inf")):
            with pytest.raises(ValueError, match="whole number"):
                call(v)
    # whole numbers of other types are none the worse
    assert torch.equal(F.dropout(x, 0.5, np.int64(7), offset=2.0, shared_dim=np.int32(0)), F.dropout(x, 0.5, 7, offset=2, shared_dim=0))
    assert torch.equal(F.embedding(t, x, padding_idx=np.int64(1)), F.embedding(t, x))
    assert F.token_log_probs(x, t, top=np.int64(2), ignore_index=np.int64(-5)).top_tokens.shape == (3, 2)


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,width,cut", [(700, 64, 8), (700, 64, 5), (513, 33, 1), (1, 96, 32), (4099, 3, 2)])
def test_dropout_of_rows_apart(rows, width, cut, dtype):
    """[rows, width] with gaps between its rows is read in place, forward and backward."""
    wide = torch.randn(rows, width + cut, generator=gen(34), device="cuda").to(DT[dtype])
    for x in (wide[:, :width], wide[:, cut:], wide[::2, :width], wide[:1, :width].expand(rows, width)):
        for d in (None, 0):
            check_dropout(x, 0.3, 11, 4, d, grad=wide[: x.shape[0], :width])
    check_dropout(torch.randn(width, rows, generator=gen(35), device="cuda").to(DT[dtype]).t(), 0.3, 11, 4, 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_dropout_of_more_dimensions_apart(dtype):
    x = torch.randn(3, 4, 5, 6, 40, generator=gen(36), device="cuda").to(DT[dtype])
    for v in (x[..., :32], x[..., 3:], x[:, :, :, ::2], x.transpose(1, 2), x.transpose(0, 3)[..., :8], x[:, :1].expand_as(x), x.permute(4, 0, 1, 2, 3)):
        for d in (None, 0, 2, 3):
            check_dropout(v, 0.3, 13, 4, d)


@pytest.mark.parametrize("shape,shared_dim", [((4096,), None), ((4096,), 0), ((16, 256), None), ((16, 256), 1), ((4, 4, 256), None)])
def test_dropout_of_rows_apart_copies_nothing(shape, shared_dim):
    x = torch.randn(*shape, 1024 + 8, device="cuda")[..., :1024]
    F.dropout(x, 0.5, 1)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = F.dropout(x, 0.5, 1, shared_dim=shared_dim)
    assert torch.cuda.max_memory_allocated() - before == y.numel() * 4


def test_dropout_of_more_than_2_to_31_rows():
    n0, n1 = 2 ** 16, 2 ** 15 + 3
    x = torch.ones(n0, n1, 2, device="cuda", dtype=torch.bfloat16)[:, :, :1]
    y = F.dropout(x, 0.25, 9, offset=2).view(-1)
    for first in (0, 2 ** 31 - 2048, n0 * n1 // 4 * 4 - 4096):
        assert torch.equal(y[first:first + 4096] != 0, torch.from_numpy(O.kept(4096, 0.25, 9, 2, first)).cuda())
    del y
    y = F.dropout(x, 0.25, 9, offset=2, shared_dim=0)
    mask = torch.from_numpy(O.kept(n1, 0.25, 9, 2)).cuda()
    assert (y.view(n0, n1)[::4093] != 0).eq(mask).all()
    with pytest.raises(ValueError, match="more than 2\\^31 - 1 rows"):
        F.dropout(x, 0.25, 9, shared_dim=1)


# ---------------------------------------------------------------- C ABI
def descriptor(cls, **given):
    d = cls()
    for k, v in given.items():
        setattr(d, k, type(getattr(d, k))(*v) if isinstance(v, tuple) else v)
    return d


@pytest.mark.parametrize("at", [0, 1, 2, 3])
@pytest.mark.parametrize("width", [16, 7])
def test_reports_reach_a_mailbox_on_any_int(width, at):
    lib = _lib.load()
    tokens, W, out = torch.tensor([3, 1, 9, 0], device="cuda"), torch.ones(5, width, device="cuda"), torch.zeros(4, width, device="cuda")
    mail = torch.zeros(16, dtype=torch.int32).pin_memory()
    d = descriptor(_lib.EmbedDesc, dtype=_lib.F32, token_bits=64, n0=1, n1=4, token_stride=(0, 1), vocab=5, width=width, row_stride=(width, 0), padding=-1, scale=1.0)
    stream = torch.cuda.current_stream().cuda_stream
    lib.blstm_set_mailbox(mail.data_ptr() + 4 * at)
    try:
        assert lib.blstm_embedding(d, tokens.data_ptr(), W.data_ptr(), out.data_ptr(), stream) == 0
    finally:
        lib.blstm_set_mailbox(None)
    torch.cuda.synchronize()
    assert mail.tolist() == [0] * at + [0, _lib.E_TOKEN, 2, 9] + [0] * (12 - at)
    assert out[2].isnan().all() and torch.equal(out[[0, 1, 3]], W[:3])
