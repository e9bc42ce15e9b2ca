"""The operators around a language model where their promises end: overlapping rows, addresses, tokens and numbers that are none,
masks held to bounds of their own.  Tolerances as in test_gpu_language.py unless a test derives its own."""
import pytest
import torch

import fastlstm_b200 as F
from test_gpu_language import U, check_scores, gen, make_logits

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
