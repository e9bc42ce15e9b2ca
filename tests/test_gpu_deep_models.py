"""Norms, AdamW and beam search together, as a deep language model of LSTM layers uses them: the example's model with residual layers."""
import itertools
import math

import pytest
import torch

import fastlstm_b200 as F

from test_gpu_language import _example, gen

pytestmark = pytest.mark.gpu


def reference(model, dtype=torch.float64):
    """(table, norms, torch.nn.LSTM layers) with the model's numbers."""
    table = model.table.detach().to(dtype).requires_grad_()
    norms = [w.detach().to(dtype).requires_grad_() for w in model.norms]
    layers = [torch.nn.LSTM(table.shape[1], table.shape[1], dtype=dtype, device="cuda") for _ in model.layers]
    for a, b in zip(layers, model.layers):
        a.load_state_dict({k: v.to(dtype) for k, v in b.state_dict().items()})
    return table, norms, layers


def ref_logits(tokens, table, norms, layers, padding=None):
    h = torch.nn.functional.embedding(tokens, table, padding_idx=padding) * table.shape[1] ** 0.5
    n = lambda x, w: torch.nn.functional.rms_norm(x, (x.shape[-1],), w, 1e-6)
    for layer, w in zip(layers, norms):
        h = h + layer(n(h, w))[0]
    return n(h, norms[-1]) @ table.t()


def test_gradients_match_torch():
    """One step of a residual model against torch's own layers in 64 bits: each of the nine operators that the gradients pass through is
    within 1e-5 of its tensor's norm in fp32."""
    m = _example()
    torch.manual_seed(3)
    model = m.LanguageModel(70, 48, layers=3, dropout=0.0, dtype=torch.float32, residual=True)
    with torch.no_grad():
        for w in model.norms:
            w.add_(0.2 * torch.randn(48, device="cuda"))
    tokens, targets = m.batch(70, 12, 5, gen(1))
    grads = torch.autograd.grad(model.loss(tokens, targets, entropy_weight=0.1), list(model.parameters()))
    table, norms, layers = reference(model)
    lp = torch.log_softmax(ref_logits(tokens, table, norms, layers, m.PADDING), -1)
    live = targets != m.PADDING
    want = -((lp.gather(2, targets[..., None])[..., 0] - 0.1 * (lp.exp() * lp).sum(-1)) * live).sum() / live.sum()
    ref = torch.autograd.grad(want, [table] + [p for layer in layers for p in layer.parameters()] + norms)
    assert len(ref) == len(grads)
    for (name, _), a, b in zip(model.named_parameters(), grads, ref):
        assert float((a.double() - b).norm()) <= 9e-5 * float(b.norm()), name


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_repeats(dtype, bits):
    """The same run twice: losses, weights and states bit by bit."""
    m = _example()

    def once():
        torch.manual_seed(5)
        model = m.LanguageModel(60, 64, layers=3, dropout=0.1, dtype={"fp32": torch.float32, "bf16": torch.bfloat16}[dtype], residual=True)
        o = F.AdamW(model.parameters(), lr=3e-3, state_bits=bits, max_norm=1.0, seed=3)
        return model, o, m.train(model, 8, T=24, B=32, optimiser=o)
    (a, o, losses), (b, n, again) = once(), once()
    assert losses == again and all(math.isfinite(v) for v in losses)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q) and all(torch.equal(o.state[p][k].float(), n.state[q][k].float()) for k in o.state[p])
    assert all(int(o.state[p]["step"]) == 8 for p in a.parameters())


def test_search_finds_the_best_sequences():
    """With as many hypotheses as there are pairs of tokens, sequences of three tokens are found in the order of their log probabilities,
    which a model in 64 bits gives (distances of less than 1e-4 do not decide)."""
    m = _example()
    torch.manual_seed(6)
    model = m.LanguageModel(5, 32, layers=2, dropout=0.0, dtype=torch.float32, residual=True)
    with torch.no_grad():
        model.table.mul_(2)
    model.eval()
    start = torch.tensor([[1, 4], [2, 3]], device="cuda")
    found, scores = model.search(start, 3, beams=25)
    assert found.shape == (2, 25, 3) and scores.shape == (2, 25) and (scores[:, :-1] >= scores[:, 1:]).all()
    table, norms, layers = reference(model)
    every = torch.tensor(list(itertools.product(range(5), repeat=3)), device="cuda")
    with torch.no_grad():
        for b in range(2):
            tokens = torch.cat([start[:, b, None].expand(2, 125), every.t()[:2]])
            lp = torch.log_softmax(ref_logits(tokens, table, norms, layers), -1)[1:]
            total = lp.gather(2, every.t()[..., None])[..., 0].sum(0)
            place = (found[b] * torch.tensor([25, 5, 1], device="cuda")).sum(1)
            assert place.unique().numel() == 25
            assert float((total[place] - scores[b]).abs().max()) <= 1e-4
            assert float((total[place] - total.topk(25).values).abs().max()) <= 1e-4


def test_search_stops_at_the_end_token():
    m = _example()
    torch.manual_seed(7)
    model = m.LanguageModel(7, 32, layers=1, dropout=0.0, dtype=torch.bfloat16, residual=True)
    model.eval()
    met = 0
    for end in range(7):                     # (a model that has learnt nothing repeats what it was given: which tokens it comes to is its own matter)
        found, scores = model.search(torch.tensor([[1, 2, 3]], device="cuda"), 12, beams=6, end=end, length_penalty=1.0)
        there = found == end
        assert (there == (there.cumsum(-1) > 0)).all() and scores.isfinite().all()      # nothing but the end token behind it
        met += int(there.any(-1).sum())
    assert met > 0
    F.check_status()
