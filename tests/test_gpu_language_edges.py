"""The operators around a language model where their promises end: overlapping rows, addresses, tokens and numbers that are none,
masks held to bounds of their own.  Tolerances as in test_gpu_language.py unless a test derives its own."""
import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200 import _lib
from oracle import language_oracle as O

from test_gpu_language import DT, EPS, TINY, U, check_dropout, check_scores, gen, make_logits, np64

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


def masked_rows(vocab, dtype):
    z = make_logits(gen(38), 9, vocab, dtype=dtype)
    low = torch.finfo(DT[dtype]).min
    z[1, ::2] = -float("inf")
    z[2, 1:] = -float("inf")                    # one token possible
    z[3] = -float("inf")                        # none
    z[4, : vocab - 3] = low
    z[5] = low                                  # all equal
    z[6, 5:] = -float("inf")
    z[7, torch.rand(vocab, generator=gen(39), device="cuda") < 0.7] = low
    return z


@pytest.mark.parametrize("temperature", [1.0, 1.5])
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("vocab", [40, 600, 3000, 40000])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_scores_of_masked_rows_to_bounds_of_their_own(dtype, vocab, top, temperature):
    """Every row and every logit has its own bound, over what counts in that row.

    With D the largest distance in powers of two of a logit whose probability is not 0 in 32 bits (e^-104), a power of two is
    relatively off by (3 D + 4) u, the sum over a row by V / 64 u more.  A log probability lp adds roundings of its own size: (8 |lp| +
    3 D + 8 + V / 64) u.  The entropy H, a mean of distances (at most H) over that sum: (H + 1) (6 D + 20 + V / 32) u.  A gradient,
    p (g + g_H (lp + H)) / T, whose p is relatively off by (6 D + 12 + V / 64) u and which rounds sums of at most 5 terms and the entropy:
    (6 D + 88 + V / 64) u of its terms' size, p |g_H| times the entropy's bound, 40 u of itself, and what 2^-126 cuts off; then the type's rounding.
    """
    z = masked_rows(vocab, dtype).requires_grad_()
    raw, V = np64(z), vocab
    for token in (0, vocab - 1):
        tokens = torch.full((9,), token, device="cuda")
        r = F.token_log_probs(z, tokens, top=top, temperature=temperature)
        want = O.token_log_probs(raw, tokens.cpu().numpy(), top, temperature)
        lp = want["lp"]
        D = np.where(lp > -104, np.abs(lp), 0).max(1) / np.log(2) + 1

        def check(got, ref, bound, small, what):
            fine = np.isfinite(ref)
            assert np.array_equal(got[~fine], ref[~fine]), what
            assert (bound[fine] <= small[fine]).all(), what + ": the bound would hold anything"
            err = np.abs(got[fine] - ref[fine])
            assert (err <= bound[fine]).all(), (what, err.max())

        def of_log_probs(ref, D):
            with np.errstate(invalid="ignore"):
                return (8 * np.abs(ref) + 3 * D + 8 + V / 64) * U, 1e-4 * (1 + np.abs(ref))
        check(np64(r.log_probs), want["log_probs"], *of_log_probs(want["log_probs"], D), "log_probs")
        H = want["entropy"]
        of_H = (H + 1) * (6 * D + 20 + V / 32) * U
        check(np64(r.entropy), H, of_H, 2e-4 * (1 + H), "entropy")
        if top:
            assert np.array_equal(r.top_tokens.cpu().numpy(), want["top_tokens"])
            check(np64(r.top_log_probs), want["top_log_probs"], *of_log_probs(want["top_log_probs"], D[:, None]), "top_log_probs")
        outs = [r.log_probs, r.entropy] + ([r.top_log_probs] if top else [])
        ups = [torch.randn(t.shape, generator=gen(40), device="cuda") for t in outs]
        (d,) = torch.autograd.grad(outs, z, ups)
        g = [np64(u) for u in ups]
        ref, size = O.token_log_probs_grad(raw, tokens.cpu().numpy(), g[0], g[1], g[2] if top else None, temperature)
        g_all = np.abs(g[0]) + (np.abs(g[2]).sum(1) if top else 0) + np.abs(g[1]) * (200 + H)
        p = np.exp(lp)
        inner = ((6 * D + 88 + V / 64)[:, None] * U * size + p * (np.abs(g[1]) * of_H / temperature)[:, None] + 40 * U * np.abs(ref)
                 + 2.0 ** -126 * g_all[:, None] / temperature)
        check(np64(d), ref, inner + EPS[dtype] * np.abs(ref) + TINY[dtype],
              1e-3 * (p * g_all[:, None] / temperature + np.abs(ref)) + EPS[dtype] * np.abs(ref) + TINY[dtype] + 1e-34, "dlogits")


# ---------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", [1, 2, 3, 7, 33, 302])
@pytest.mark.parametrize("bad", [[0], [22], [5, 6], [3, 11, 12, 13], list(range(23))])
def test_lookups_of_tokens_outside_of_the_vocabulary_in_odd_widths(width, bad, dtype):
    """Rows that begin and end inside of 16-byte pieces: a row of NaN ends where it should, and is reported."""
    W = torch.randn(7, width, generator=gen(37), device="cuda").to(DT[dtype]).requires_grad_()
    good = torch.arange(23, device="cuda") % 7
    rows = torch.ones(23, dtype=torch.bool, device="cuda")
    rows[bad] = False
    for wrong, scale, kind in ((7, 1.0, torch.int64), (-1, 3.0, torch.int64), (2 ** 40 + 3, 1.0, torch.int64), (-2 ** 31, 1.0, torch.int32)):
        tokens = torch.where(rows, good, wrong).to(kind)
        out = F.embedding(tokens, W, scale=scale)
        with pytest.raises(_lib.BlstmError, match="token %d at position" % min(wrong, 2 ** 31 - 1)) as e:
            F.check_status()
        assert e.value.code == _lib.E_TOKEN and int(str(e.value).split("position ")[1].split(":")[0]) in bad
        F.check_status()
        want = (W.detach().float() * scale).to(W.dtype)[good]
        assert out[~rows].isnan().all() and torch.equal(out[rows], want[rows])
        (dW,) = torch.autograd.grad(out, W, torch.ones_like(out))
        count = torch.bincount(good[rows], minlength=7).float()[:, None] * scale
        assert torch.equal(dW.float(), count.expand(7, width))


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
