"""A step of beam search and the reordering of states against their oracle in 64 bits, at the sizes, strides, masks and ties where they
can go wrong.

Tolerances.  u = 2^-24.  A logit's distance of D powers of two from its row's maximum carries an error of D u, its exponential 4 u more, a sum
over V terms V / 64 u (no thread adds up more in a row): C u with C = 4 D + 16 + V / 64 bounds what a row's sum adds to its totals; outputs
are rounded to 32 bits.  Two hypotheses' continuations whose ranks are nearer than twice that may come in either order; within one
hypothesis the order is that of the logits, always."""
import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200._lib import BlstmError, E_PARENT
from oracle import language_oracle as O

from test_gpu_language import DT, U, gen, np64

pytestmark = pytest.mark.gpu


def host(t):
    return None if t is None else t.cpu().numpy()


def check(logits, scores, width=None, end=None, finished=None, lengths=None, penalty=0.0):
    B, n, V = logits.shape
    W = n if width is None else width
    r = F.beam_step(logits, scores, width=width, end_token=end, finished=finished, lengths=lengths, length_penalty=penalty)
    again = F.beam_step(logits, scores, width=width, end_token=end, finished=finished, lengths=lengths, length_penalty=penalty)
    F.check_status()
    for a, b in zip(r, again):
        assert (a is None and b is None) or torch.equal(a, b) or torch.equal(a.isnan(), b.isnan())
    assert r.scores.shape == r.parents.shape == r.tokens.shape == (B, W) and r.scores.dtype == torch.float32
    assert r.parents.dtype == r.tokens.dtype == torch.int64
    z, s, f, l = np64(logits), np64(scores), host(finished), host(lengths)
    want_s, want_p, want_t, want_f, want_l = O.beam_step(z, s, W, end, f, l, penalty)
    rank, total = O.beam_ranks(z, s, end, f, l, penalty)
    p, t = host(r.parents), host(r.tokens)
    rows = np.arange(B)[:, None]
    with np.errstate(all="ignore"):
        far = np.nan_to_num(np.where(np.isfinite(z), z.max(-1, keepdims=True) - z, 0)) / np.log(2)
        D = min(float(far.max()) if far.size else 0, 160)
    bound = (4 * D + 16 + V / 64) * U
    got_total, got_rank, ideal = total[rows, p, t], rank[rows, p, t], rank[rows, want_p, want_t]
    same = (p == want_p) & (t == want_t)
    with np.errstate(all="ignore"):
        assert (same | (np.abs(got_rank - ideal) <= 2 * bound)).all(), "another continuation than the oracle's"
        near = np.abs(np64(r.scores) - got_total) <= bound + U * np.abs(got_total)
    assert (near | (np64(r.scores) == got_total) | (np.isnan(np64(r.scores)) & np.isnan(got_total))).all(), "scores"
    for b in range(B):                                   # never the same continuation twice
        assert len(set(zip(p[b], t[b]))) == W
    if end is not None:
        ended = np.zeros((B, n), bool) if f is None else f
        assert (host(r.finished) == (ended[rows, p] | (t == end))).all()
    else:
        assert r.finished is None
    if l is not None:
        ended = np.zeros((B, n), bool) if f is None else f
        assert (host(r.lengths) == l[rows, p] + ~ended[rows, p]).all()
    else:
        assert r.lengths is None
    return r, same.all()


def make(g, B, n, V, dtype="bf16", std=2.5):
    logits = (torch.randn(B, n, V, generator=g, device="cuda") * std).to(DT[dtype])
    return logits, -torch.rand(B, n, generator=g, device="cuda") * 6


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,n,V,W", [(1, 1, 1, 1), (1, 1, 50, 4), (2, 3, 7, 5), (1, 3, 2, 6), (2, 32, 1, 32), (3, 4, 205, 4), (2, 5, 1000, 8), (2, 4, 1024, 4), (2, 4, 1025, 4),
                                     (3, 10, 2053, 10), (2, 8, 4099, 32), (1, 4, 50000, 4), (1, 32, 9001, 32), (40, 2, 3001, 2), (2, 3, 131072, 16),
                                     (700, 3, 64, 3), (5, 1, 20011, 24), (150, 5, 5003, 1)])
def test_sizes(dtype, B, n, V, W):
    g = gen(B + n + V)
    check(*make(g, B, n, V, dtype), width=W)


@pytest.mark.parametrize("penalty", [0.0, 0.6, 2.0])
@pytest.mark.parametrize("V", [60, 700, 5003, 40000])
def test_ended_hypotheses_and_lengths(V, penalty):
    g = gen(V)
    B, n = 6, 5
    logits, scores = make(g, B, n, V)
    finished = torch.rand(B, n, generator=g, device="cuda") < 0.4
    finished[0], finished[1] = True, False
    lengths = torch.randint(1, 40, (B, n), generator=g, device="cuda")
    for end in (0, 3, V - 1):
        logits[finished] = float("nan")                  # (never looked at)
        r, _ = check(logits, scores, 7, end, finished, lengths, penalty)
        assert not r.scores.isnan().any()
    check(logits.nan_to_num(), scores, None, V - 1)
    check(logits.nan_to_num(), scores, None, None, None, lengths, penalty)


@pytest.mark.parametrize("V", [40, 600, 3000, 40000])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_masks(V, dtype):
    """Rows that leave fewer tokens than the width, one, none; the type's lowest value in place of -inf; hypotheses that are dead."""
    g = gen(V)
    B, n, W = 7, 4, 6
    logits, scores = make(g, B, n, V, dtype)
    inf = float("inf")
    logits[0, :, 2:] = -inf                              # two tokens each: 8 continuations
    logits[1, :, 1:] = -inf                              # four continuations for a width of 6
    logits[2] = -inf                                     # none
    logits[3, 1:] = -inf
    logits[4, torch.rand(n, V, generator=g, device="cuda") < 0.9] = torch.finfo(DT[dtype]).min
    scores[5, 1:] = -inf
    logits[5, 1:] = float("nan")                         # (dead: never looked at)
    scores[6] = -inf
    r, _ = check(logits, scores, W)
    assert (r.scores[1] == -inf).sum() == 2 and (r.scores[2] == -inf).all() and (r.parents[5] == 0).all() and (r.scores[6] == -inf).all()
    assert r.parents[2].tolist() == [0] * W and r.tokens[2].tolist() == list(range(W)) and r.tokens[6].tolist() == list(range(W))


@pytest.mark.parametrize("V", [48, 720, 5008, 40000])
@pytest.mark.parametrize("kind", ["equal", "few values", "rising", "falling", "block at the end"])
def test_ties(V, kind):
    """Equal logits and equal hypotheses: the first hypothesis, the first token.  (Rows of whole 16-byte pieces, whose sums are alike.)"""
    g = gen(V)
    B, n = 3, 4
    i = torch.arange(V, device="cuda").float()
    row = {"equal": i * 0, "few values": i % 3, "rising": (i / 64).floor(), "falling": (-i / 64).floor(),
           "block at the end": (i >= V - 20).float() * 5}[kind]
    logits = row.expand(B, n, V).bfloat16()
    r, same = check(logits, torch.full((B, n), -2.0, device="cuda"), 9)
    assert same
    spread = torch.tensor([-1.0, -1.0, -1.5, -1.5], device="cuda").expand(B, n)
    assert check(logits, spread, 9)[1]


@pytest.mark.parametrize("V", [40, 3001, 40000])
@pytest.mark.parametrize("low", [-1e4, -1e9, -1e30, torch.finfo(torch.float32).min])
def test_scores_that_stand_for_dead_hypotheses(V, low):
    """First steps with one hypothesis of score 0 and others that are out by their scores; sentences of nothing but those, whose totals may
    all be one number: the first hypothesis, the first tokens."""
    g = gen(V)
    logits, scores = make(g, 4, 5, V)
    scores[0], scores[1], scores[2, 1:] = low, low, low
    scores[0, 3] = 0
    r, _ = check(logits, scores)
    assert (r.parents[0] == 3).all() and (r.parents[2] == 0).all()
    if low <= -1e30:
        assert (r.parents[1] == 0).all() and r.tokens[1].tolist() == list(range(5))
    lengths = torch.randint(1, 9, (4, 5), generator=g, device="cuda")
    if low > -1e30:
        check(logits, scores, 7, 1, None, lengths, 0.7)


@pytest.mark.parametrize("scale", [1e3, 1e6])
def test_scores_of_any_size_and_sign(scale):
    """Scores that cancel against what the logits come to."""
    g = gen(9)
    logits, scores = make(g, 3, 6, 9001, "fp32")
    logits[1] *= 40
    scores = torch.randn(3, 6, generator=g, device="cuda") * scale
    check(logits, scores)
    check(logits, scores - scores.amax(1, keepdim=True) + logits.amax(-1), 4)


@pytest.mark.parametrize("V", [100, 2000, 20000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_a_number_and_infinity_come_first(V, bad):
    g = gen(V)
    logits, scores = make(g, 3, 3, V, "fp32")
    logits[1, 2, V // 3] = bad
    r = F.beam_step(logits, scores, width=2)
    assert r.scores[1].isnan().all() and (r.parents[1] == 2).all() and not r.scores[[0, 2]].isnan().any()
    clean = logits.clone()
    clean[1] = 0
    want = F.beam_step(clean, scores, width=2)
    for a, b in zip(r[:3], want[:3]):
        assert torch.equal(a[[0, 2]], b[[0, 2]])


def spoiled(call):
    """A call whose results lie in memory that holds something else; what it returns twice is the same, bit by bit."""
    results = []
    for fill in (-7, 13):
        junk = [torch.full((n,), fill, dtype=torch.int64, device="cuda") for n in (8, 64, 128, 192, 256, 512) for _ in range(8)]
        del junk
        results.append(call())
    F.check_status()
    for a, b in zip(*results):
        assert (a is None and b is None) or torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    return results[0]


@pytest.mark.parametrize("V", [9, 40, 600, 4000, 40000])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_a_number_and_infinity_beside_masked_logits(V, dtype, bad):
    """A bad logit makes all of its hypothesis' continuations NaN, the masked ones too: they come first, in the order of (hypothesis, token),
    and what is possible behind them.  (One healthy hypothesis a sentence: its order is that of its logits.)"""
    g = gen(V)
    inf = float("inf")
    for W in (1, 2, 8, 31, 32):
        for at in (0, V // 3, V - 1):
            n = 4
            logits, scores = make(g, 6, n, V, dtype)
            logits[:, 1:] = -inf
            scores[:, 3] = -inf                          # (dead)
            logits[0, 1, at] = bad                       # one bad logit, nothing else possible; the healthy one in front
            logits[1, 0] = -inf
            logits[1, 0, at] = bad                       # the same in the first hypothesis; the second has nothing possible
            logits[2, 2] = make(g, 1, 1, V, dtype)[0][0, 0]
            logits[2, 2, torch.rand(V, generator=g, device="cuda") < 0.9] = -inf
            logits[2, 2, at] = bad                       # some finite ones besides
            logits[3, 1:3, at] = bad                     # two bad hypotheses
            logits[4, 2, at:] = bad
            scores[5, 0] = bad                           # a bad score over logits of which some are masked
            logits[5, 0, ::2] = -inf
            w = min(W, n * V)
            finished = torch.zeros(6, n, dtype=torch.bool, device="cuda")
            finished[4, 1], scores[4, 1] = True, 0       # (ended, in front of all that go on)
            lengths = torch.randint(1, 9, (6, n), generator=g, device="cuda")
            for kw in (dict(), dict(end_token=V // 2, finished=finished, lengths=lengths, length_penalty=0.7)):
                r = spoiled(lambda: F.beam_step(logits, scores, width=w, **kw))
                z, s = np64(logits), np64(scores)
                f, l = (host(finished), host(lengths)) if kw else (None, None)
                want_s, want_p, want_t, want_f, want_l = O.beam_step(z, s, w, V // 2 if kw else None, f, l, kw.get("length_penalty", 0.0))
                assert (host(r.parents) == want_p).all() and (host(r.tokens) == want_t).all()
                got = np64(r.scores)
                assert (np.isnan(got) == np.isnan(want_s)).all()
                sure = np.isfinite(want_s)
                assert (got[~sure & ~np.isnan(got)] == want_s[~sure & ~np.isnan(got)]).all()
                assert (np.abs(got[sure] - want_s[sure]) <= (4 * 160 + 16 + V / 64) * U + U * np.abs(want_s[sure])).all()
                if kw:
                    assert (host(r.finished) == want_f).all() and (host(r.lengths) == want_l).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_scores_of_hypotheses_that_cannot_go_on(bad):
    """A score of NaN or +inf over logits of nothing but -inf: NaN, not a quiet end."""
    logits, scores = torch.full((1, 2, 700), -float("inf"), device="cuda"), torch.tensor([[-1.0, bad]], device="cuda")
    r = spoiled(lambda: F.beam_step(logits, scores, width=5))
    assert r.scores.isnan().all() and r.parents.tolist() == [[1] * 5] and r.tokens.tolist() == [list(range(5))]


@pytest.mark.parametrize("V", [77, 512, 1300, 6007, 40003])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(V, dtype):
    """Logits that are turned, cut from a padded vocabulary, expanded; scores, lengths and flags that are views."""
    g = gen(V)
    B, n = 3, 4
    logits, scores = make(g, B, n, V + 5, dtype)
    check(logits[..., :V], scores)
    check(logits[..., 5:], scores)
    check(make(g, n, B, V, dtype)[0].transpose(0, 1), scores)
    check(make(g, B, 1, V, dtype)[0].expand(B, n, V), scores)
    check(make(g, V, B, n, dtype)[0].permute(1, 2, 0), scores)
    wide = torch.rand(n, B, 2, generator=g, device="cuda")
    check(logits[..., :V], -wide[..., 1].t(), 5, 3, (wide[..., 0] < 0.3).t(), (wide[..., 0] * 20).long().t() + 1, 1.0)


def test_no_sentences_and_refusals():
    r = F.beam_step(torch.zeros(0, 3, 5, device="cuda"), torch.zeros(0, 3, device="cuda"), end_token=1)
    assert r.scores.shape == r.finished.shape == (0, 3) and r.lengths is None
    z, s = torch.zeros(2, 3, 5, device="cuda"), torch.zeros(2, 3, device="cuda")
    f, l = torch.zeros(2, 3, device="cuda", dtype=torch.bool), torch.zeros(2, 3, device="cuda", dtype=torch.long)
    for a, k in (((z[0], s), {}), ((z, s[:1]), {}), ((z, s.half()), {}), ((z.double(), s), {}), ((z, s.cpu()), {}), ((z, s), dict(width=0)),
                 ((z, s), dict(width=16)), ((z, s), dict(end_token=5)), ((z, s), dict(end_token=-1)), ((z, s), dict(finished=f)),
                 ((z, s), dict(end_token=1, finished=f.long())), ((z, s), dict(end_token=1, finished=f[:1])), ((z, s), dict(lengths=l.int())),
                 ((z, s), dict(length_penalty=0.5)), ((z, s), dict(lengths=l, length_penalty=-0.5)), ((z, s), dict(lengths=l, length_penalty=float("nan"))),
                 ((z[..., :0], s), {}), ((z[:, :0], s[:, :0]), {}), ((torch.zeros(1, 33, 5, device="cuda"), torch.zeros(1, 33, device="cuda")), {}),
                 ((torch.zeros(1, 2, 50, device="cuda"), torch.zeros(1, 2, device="cuda")), dict(width=33)), ((z.requires_grad_(), s), {})):
        with pytest.raises(ValueError):
            F.beam_step(*a, **k)
    with torch.no_grad():
        F.beam_step(z, s)


@pytest.mark.parametrize("penalty", [0.6, 4.0])
@pytest.mark.parametrize("V", [3, 60, 5003])
def test_lengths_that_are_none(V, penalty):
    """Lengths of zero, below it and far above any, of hypotheses that go on, have ended or are dead: nothing is divided by 0, and what
    is impossible comes behind."""
    g = gen(V)
    logits, scores = make(g, 4, 6, V)
    finished = torch.zeros(4, 6, dtype=torch.bool, device="cuda")
    finished[:, 1] = finished[:, 3] = True
    scores[0, 2:], scores[1, 1:], scores[2, :5], scores[3, 3] = -torch.inf, -torch.inf, -torch.inf, 0
    lengths = torch.tensor([0, 0, -7, -1, 2 ** 62, 12], device="cuda").repeat(4, 1)
    lengths[1], lengths[2] = -1, 1 << 40
    check(logits, scores, 9, 1, finished, lengths, penalty)
    with pytest.raises(ValueError, match="length_penalty"):
        F.beam_step(logits, scores, lengths=lengths, length_penalty=4.5)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,n,V,W", [(2, 32, 1, 32), (3, 4, 205, 4), (2, 4, 1025, 4), (3, 10, 2053, 10), (2, 8, 4099, 32), (1, 32, 9001, 32), (700, 3, 64, 3), (2, 3, 131072, 16),
                                     (5, 1, 20011, 24), (64, 5, 20003, 5)])
def test_runs_repeat_bit_by_bit(dtype, B, n, V, W):
    """All of a step's results, also of equal logits, which overflow the candidates' buffer in whatever order they come."""
    g = gen(B + n + V)
    logits, scores = make(g, B, n, V, dtype)
    few = (logits * 0.5).round()
    finished = torch.rand(B, n, generator=g, device="cuda") < 0.2
    lengths = torch.randint(1, 30, (B, n), generator=g, device="cuda")
    for z in (logits, few, torch.zeros_like(logits)):
        for s in (scores, torch.zeros_like(scores)):
            first = spoiled(lambda: F.beam_step(z, s, width=W))
            for _ in range(4):
                assert all(torch.equal(a, b) for a, b in zip(first[:3], F.beam_step(z, s, width=W)[:3]))
            spoiled(lambda: F.beam_step(z, s, width=W, end_token=V - 1, finished=finished, lengths=lengths, length_penalty=0.6))


def test_captured_and_replayed_and_on_another_stream():
    g = gen(3)
    logits, scores = make(g, 4, 5, 9000)
    state = torch.randn(2, 20, 64, generator=g, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = F.beam_step(logits, scores)
        moved = F.reorder_states(state, side.parents)
    torch.cuda.current_stream().wait_stream(s)
    want = F.beam_step(logits, scores)
    assert all(torch.equal(a, b) for a, b in zip(side[:3], want[:3])) and torch.equal(moved, F.reorder_states(state, want.parents))
    graphs, results = [], []
    for _ in range(2):                                   # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = F.beam_step(logits, scores)
            results.append((r, F.reorder_states(state, r.parents)))
        graphs.append(graph)
    for k in range(4):
        logits.copy_(make(gen(10 + k), 4, 5, 9000)[0])
        graphs[k % 2].replay()
        want = F.beam_step(logits, scores)
        r, moved = results[k % 2]
        assert all(torch.equal(a, b) for a, b in zip(r[:3], want[:3])) and torch.equal(moved, F.reorder_states(state, want.parents))


def test_calls_at_once():
    """Searches and reorderings on two streams side by side, and two layers' states behind each."""
    g = gen(12)
    data = [(*make(g, 7, 6, 9001), torch.randn(2, 42, 96, generator=g, device="cuda")) for _ in range(2)]

    def step(logits, scores, state):
        r = F.beam_step(logits, scores)
        again = F.beam_step(logits, r.scores)
        return [*r[:3], *again[:3], *F.reorder_states((state, r.tokens.view(1, -1)), again.parents)]
    want = [step(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(step(*d))
    torch.cuda.synchronize()
    for k, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[k % 2]))


def test_logits_beyond_32_bits():
    """More than 2^31 logits (4.4 GB): the last sentence is what it is alone."""
    B, n, V = 66, 32, 2 ** 20 + 3
    logits = torch.zeros(B, n, V, device="cuda", dtype=torch.bfloat16)
    g = gen(4)
    last, scores = make(g, 1, n, V)
    logits[-1] = last[0]
    all_scores = scores.expand(B, n).contiguous()
    r, want = F.beam_step(logits, all_scores, width=8), F.beam_step(logits[-1:].clone(), scores, width=8)
    # (the copy may begin on another boundary: sums in another order, 2^-22 apart)
    assert torch.equal(r.parents[-1:], want.parents) and torch.equal(r.tokens[-1:], want.tokens)
    assert float((r.scores[-1:] - want.scores).abs().max()) <= 2e-5


# ---------------------------------------------------------------- reordering
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64, torch.int64, torch.int32, torch.int16, torch.uint8, torch.bool,
                                   torch.float8_e4m3fn, torch.complex64])
@pytest.mark.parametrize("inner", [(), (1,), (3,), (7,), (64,), (5, 12)])
def test_reorder_types_and_sizes(dtype, inner):
    g = gen(5)
    B, n, W = 3, 4, 6
    parents = torch.randint(0, n, (B, W), generator=g, device="cuda")
    for outer in ((), (1,), (3,), (2, 5)):
        raw = torch.randint(0, 2, (*outer, B * n, *inner), generator=g, device="cuda") if dtype == torch.bool else torch.randint(0, 100, (*outer, B * n, *inner), generator=g, device="cuda")
        x = raw.to(dtype)
        got = F.reorder_states(x, parents, dim=len(outer))
        rows = (torch.arange(B, device="cuda")[:, None] * n + parents).view(-1)
        want = raw.index_select(len(outer), rows).to(dtype)
        assert got.dtype == dtype and got.shape == want.shape and got.is_contiguous()
        assert torch.equal(got.view(-1).view(torch.uint8), want.reshape(-1).view(torch.uint8))
        assert torch.equal(F.reorder_states(x, parents.int(), dim=len(outer) - x.dim()).view(-1).view(torch.uint8), want.reshape(-1).view(torch.uint8))


def test_reorder_layouts_and_nests():
    g = gen(6)
    B, n = 5, 3
    parents = torch.randint(0, n, (B, n), generator=g, device="cuda")
    rows = (torch.arange(B, device="cuda")[:, None] * n + parents).view(-1)
    make_state = lambda *s: torch.randn(*s, generator=g, device="cuda")
    views = [make_state(2, B * n, 40)[..., 3:30], make_state(B * n, 2, 16).transpose(0, 1), make_state(16, B * n, 2).transpose(0, 2), make_state(2, 1, 8).expand(2, B * n, 8),
             make_state(2, 2 * B * n, 8)[:, ::2], make_state(4, B * n, 8)[::2], make_state(1, B * n, 8), make_state(7, B * n).bfloat16()[1:],
             make_state(2 * B * n * 8 + 1)[1:].view(2, B * n, 8), make_state(B * n, 4).t()]
    for v in views:
        assert torch.equal(F.reorder_states(v, parents), v[:, rows])
    nest = [(views[0], views[1]), [views[2], None], views[3]]
    got = F.reorder_states(nest, parents)
    assert isinstance(got, list) and isinstance(got[0], tuple) and isinstance(got[1], list) and got[1][1] is None
    for a, b in zip((got[0][0], got[0][1], got[1][0], got[2]), views):
        assert torch.equal(a, b[:, rows])
    from collections import namedtuple
    Pair = namedtuple("Pair", "h c")
    pair = F.reorder_states([Pair(views[0], None)], parents)[0]
    assert type(pair) is Pair and torch.equal(pair.h, got[0][0]) and pair.c is None
    z = torch.view_as_complex(make_state(2, B * n, 8, 2))
    for lazy in (z.conj(), z.conj().imag):               # (numbers whose signs are still to be turned)
        assert torch.equal(F.reorder_states(lazy, parents), lazy[:, rows])
    many = [make_state(1 + k % 3, B * n, 1 + k % 5) for k in range(100)]
    for a, b in zip(F.reorder_states(many, parents.t().contiguous().t()), many):
        assert torch.equal(a, b[:, rows])
    assert F.reorder_states([], parents) == []
    assert F.reorder_states(make_state(2, 0, 5), parents[:0]).shape == (2, 0, 5)
    assert F.reorder_states(make_state(2, B * n, 0), parents).shape == (2, B * n, 0)


def test_reorder_parents_that_are_none():
    state = torch.ones(3, 8, 5, device="cuda")
    for bad in (-1, 4, 2 ** 40):
        parents = torch.tensor([[0, 1, 2, 3], [3, bad, 1, 0]], device="cuda")
        got = F.reorder_states((state, state[0]), parents, dim=-2)
        with pytest.raises(BlstmError, match="at position 5") as e:
            F.check_status()
        assert e.value.code == E_PARENT
        assert not got[0][:, 5].any() and got[0][:, :5].all() and got[0][:, 6:].all() and not got[1][5].any()


def test_reorder_refusals():
    x, p = torch.zeros(2, 6, 4, device="cuda"), torch.zeros(2, 3, device="cuda", dtype=torch.long)
    for a, k in (((x, p[0]), {}), ((x, p.float()), {}), ((x, p.cpu()), {}), ((x.cpu(), p), {}), ((x, p), dict(dim=3)), ((x, p), dict(dim=-4)), ((x[:, :5], p), {}),
                 ((x[:, :0], p), {}), (([x, x[:, :4]], p), {}), ((x, p[:, :0]), {}), ((x, p[:0]), {}), ((x.clone().requires_grad_(), p), {}), ((3, p), {}),
                 ((x.to_sparse(), p), {})):
        with pytest.raises(ValueError):
            F.reorder_states(*a, **k)


def test_reorder_beyond_32_bits():
    """A state of 4.5 GB, and one whose pieces are numbered above 2^32."""
    B, n = 3, 2
    parents = torch.tensor([[1, 0], [0, 0], [1, 1]], device="cuda")
    x = torch.zeros(2, B * n, 3 * 2 ** 27 + 16, device="cuda", dtype=torch.uint8)
    x[:, :, -9:] = torch.arange(12, device="cuda", dtype=torch.uint8).view(2, 6, 1) + 1
    got = F.reorder_states(x, parents)
    assert got[:, :, -1].tolist() == [[2, 1, 3, 3, 6, 6], [8, 7, 9, 9, 12, 12]] and not got[:, :, :-9].any()
    del got
    odd = x.view(-1)[1:-11].view(2, B * n, -1)
    got = F.reorder_states(odd, parents)
    assert torch.equal(got[1, 5], odd[1, 5]) and torch.equal(got[1, 0], odd[1, 1])
