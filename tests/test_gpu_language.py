"""The operators around a language model against their oracle in 64 bits, at the sizes, strides and masks where they can go
wrong.

Tolerances.  u = 2^-24 is the rounding of 32 bits, e that of the type (2^-24, 2^-11, 2^-8), tiny the spacing of fp16's
subnormal numbers.  Embedding: one product and one rounding; the table's gradient adds n terms, an error of at most
(n + 2) u sum |terms| before it is rounded.  Dropout: one product in 32 bits and one rounding, so the expected result is known
exactly.  Log probabilities: a distance of D powers of two from the maximum carries an error of D u, its power of two a
relative one of (D + 4) u, a sum over V terms V / 64 u more (no thread adds up more in a row); C u with
C = 4 D + 16 + V / 64 bounds a log probability, C (D + 4) u the entropy, whose terms are multiplied by up to D."""
import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200._lib import BlstmError, E_TOKEN
from oracle import language_oracle as O

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
U, TINY = 2.0 ** -24, {"fp32": 1e-44, "fp16": 2.0 ** -25, "bf16": 1e-40}


def np64(t):
    return t.detach().double().cpu().numpy()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound, what):
    err = np.abs(got - want)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, the worst by {np.nanmax(err - bound):.3e} over a bound of {np.max(bound):.3e}"


# ---------------------------------------------------------------- embedding
def check_embedding(tokens, W, dtype, scale=1.0, padding=None, dout=None):
    W = W.detach().requires_grad_()
    out = F.embedding(tokens, W, scale=scale, padding_idx=padding)
    assert out.shape == (*tokens.shape, W.shape[1]) and out.dtype == W.dtype and out.is_contiguous()
    want = (W.detach().float() * torch.tensor(scale, dtype=torch.float32)).to(W.dtype)[tokens.long()]
    assert torch.equal(out, want)
    if dout is None:
        dout = torch.randn(out.shape, generator=gen(5), device="cuda").to(W.dtype)
    (dW,) = torch.autograd.grad(out, W, dout, retain_graph=True)
    (again,) = torch.autograd.grad(out, W, dout)
    F.check_status()
    assert dW.dtype == W.dtype and torch.equal(dW, again)
    ref, size, terms = O.embedding_grad(tokens.cpu().numpy(), np64(dout), W.shape[0], scale, padding)
    within(np64(dW), ref, (terms[:, None] + 2) * U * size + EPS[dtype] * np.abs(ref) + TINY[dtype], "dW")


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,width,vocab", [(1, 1, 1), (1, 512, 1000), (2, 8, 5), (31, 33, 7), (33, 40, 511), (64, 2048, 64), (1000, 301, 513),
                                           (2047, 7, 100), (2049, 24, 1), (4096, 130, 33), (5000, 64, 40000)])
def test_embedding_sizes(dtype, n, width, vocab):
    g = gen(n + width)
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    W = torch.randn(vocab, width, generator=g, device="cuda").to(DT[dtype])
    check_embedding(tokens, W, dtype, scale=1.0 if n % 2 else width ** 0.5)


@pytest.mark.parametrize("n,vocab", [(70001, 300007), (65536, 1 << 18), (65537, 262143), (140000, 600)])
def test_embedding_large_sorts(n, vocab):
    g = gen(n)
    tokens = (torch.rand(n, generator=g, device="cuda") ** 3 * vocab).long()
    W = torch.randn(vocab, 8, generator=g, device="cuda").bfloat16()
    check_embedding(tokens, W, "bf16")


@pytest.mark.parametrize("n,width", [(40, 64), (1500, 36), (3000, 520), (30000, 16)])
@pytest.mark.parametrize("kind", ["one", "two", "mostly one", "runs"])
def test_embedding_many_equal_tokens(n, width, kind):
    g = gen(7)
    i = torch.arange(n, device="cuda")
    tokens = {"one": i * 0 + 3, "two": i % 2 * 8, "mostly one": torch.where(i % 97 == 0, i % 50, 11), "runs": i // 32 % 50}[kind]
    check_embedding(tokens, torch.randn(50, width, generator=g, device="cuda").half(), "fp16", scale=0.5)


@pytest.mark.parametrize("n", [100, 5000])
@pytest.mark.parametrize("padding", [0, 3, -1])
def test_embedding_padding(n, padding):
    g = gen(8)
    tokens = torch.randint(0, 9, (n,), generator=g, device="cuda")
    W = torch.randn(9, 20, generator=g, device="cuda").requires_grad_()
    out = F.embedding(tokens, W, padding_idx=padding)
    dout = torch.randn(out.shape, generator=g, device="cuda")
    (dW,) = torch.autograd.grad(out, W, dout)
    ref, size, terms = O.embedding_grad(tokens.cpu().numpy(), np64(dout), 9, 1.0, padding % 9)
    assert not dW[padding].any() and torch.equal(out, W.detach()[tokens])
    within(np64(dW), ref, (terms[:, None] + 2) * U * size + U * np.abs(ref), "dW")
    # nothing but padding
    out = F.embedding(torch.full((n,), padding % 9, device="cuda"), W, padding_idx=padding)
    assert not torch.autograd.grad(out.sum(), W)[0].any()


@pytest.mark.parametrize("T,B,width", [(9, 5, 24), (70, 40, 64), (11, 6, 37)])
def test_embedding_layouts(T, B, width):
    """Tokens and gradients that are views: turned, cut, 32-bit, spread out; rows of a wider table."""
    g = gen(9)
    W = torch.randn(50, width, generator=g, device="cuda").bfloat16()
    tokens = torch.randint(0, 50, (B, T), generator=g, device="cuda")
    turned = torch.randn(B, T, width, generator=g, device="cuda").bfloat16().transpose(0, 1)
    check_embedding(tokens.t(), W, "bf16", dout=turned)
    check_embedding(tokens.t().int(), W, "bf16", dout=turned[:, :1].expand(T, B, width))
    check_embedding(tokens.repeat_interleave(2, 1)[:, ::2].t(), W, "bf16", dout=torch.randn(width, T, B, generator=g, device="cuda").bfloat16().permute(1, 2, 0))
    check_embedding(tokens.view(1, B, T, 1).expand(2, B, T, 3), W, "bf16")
    check_embedding(tokens[0, 0], W, "bf16")
    wide = torch.randn(50, width + 3, generator=g, device="cuda").bfloat16()
    for cut in (wide[:, :width], wide[:, 3:], torch.randn(width, 50, generator=g, device="cuda").bfloat16().t()):
        check_embedding(tokens, cut, "bf16")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [2048, 2049, 16384, 16385, 32768, 32769, 65536, 262144, 262145])
def test_embedding_at_the_lines_between_sorts(n, dtype):
    g = gen(n)
    tokens = (700 ** torch.rand(n, generator=g, device="cuda")).long()
    check_embedding(tokens, torch.randn(700, 12, generator=g, device="cuda").to(DT[dtype]), dtype, padding=0)


@pytest.mark.parametrize("n,vocab,width,dtype", [(700, 60000, 640, "fp16"), (3000, 150000, 512, "bf16"), (3000, 40001, 700, "fp32"),
                                                 (40000, 120000, 512, "fp16"), (33000, 60000, 800, "fp32"), (33000, 70001, 301, "fp32")])
def test_embedding_rows_that_no_token_names(n, vocab, width, dtype):
    """Tables larger than what is cleared beside the sort; the memory that the gradient gets held NaN before."""
    g = gen(n + width)
    tokens = torch.cat([torch.randint(0, vocab, (n - 3,), generator=g, device="cuda"), torch.tensor([vocab - 1, 0, vocab - 1], device="cuda")])
    W = torch.zeros(vocab, width, device="cuda", dtype=DT[dtype]).requires_grad_()
    out = F.embedding(tokens, W, padding_idx=5)
    dout = torch.randn(n, width, generator=g, device="cuda").to(W.dtype)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    poison = torch.full_like(W, float("nan"))
    del poison
    (dW,) = torch.autograd.grad(out, W, dout)
    met = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    met[tokens] = True
    met[5] = False
    assert not dW[~met].any()
    want = torch.zeros(vocab, width, device="cuda", dtype=torch.float64).index_add_(0, tokens, dout.double())
    size = torch.zeros(vocab, width, device="cuda", dtype=torch.float64).index_add_(0, tokens, dout.double().abs())
    terms = torch.bincount(tokens, minlength=vocab).double()[:, None]
    bound = (terms + 2) * U * size + EPS[dtype] * want.abs() + TINY[dtype]
    assert ((dW.double() - want).abs() <= bound)[met].all()


def test_embedding_without_tokens():
    W = torch.randn(5, 3, device="cuda", requires_grad=True)
    out = F.embedding(torch.zeros(0, 4, dtype=torch.long, device="cuda"), W)
    assert out.shape == (0, 4, 3)
    assert not torch.autograd.grad(out.sum(), W)[0].any()


@pytest.mark.parametrize("n", [50, 4000])
def test_embedding_tokens_outside_of_the_vocabulary(n):
    W = torch.randn(7, 16, device="cuda", requires_grad=True)
    for bad in (7, -1, 2 ** 40 + 3):
        tokens = torch.arange(n, device="cuda") % 7
        tokens[n // 2] = bad
        out = F.embedding(tokens, W)
        with pytest.raises(BlstmError, match="at position %d" % (n // 2)) as e:
            F.check_status()
        assert e.value.code == E_TOKEN
        F.check_status()                       # once
        rows = torch.arange(n, device="cuda") != n // 2
        assert out[n // 2].isnan().all() and torch.equal(out[rows], W.detach()[tokens[rows]])
        (dW,) = torch.autograd.grad(out, W, torch.ones_like(out))
        count = torch.bincount(tokens[rows], minlength=7).float()
        assert torch.equal(dW, count[:, None].expand(7, 16))


def test_embedding_gradient_against_differences():
    """The operator is linear: a difference along a direction is the gradient's product with it, to rounding."""
    g = gen(10)
    tokens, W = torch.randint(0, 30, (40, 3), generator=g, device="cuda"), torch.randn(30, 12, generator=g, device="cuda").requires_grad_()
    w, v = torch.randn(40, 3, 12, generator=g, device="cuda"), torch.randn(30, 12, generator=g, device="cuda")
    (dW,) = torch.autograd.grad(F.embedding(tokens, W, scale=2.0), W, w)
    f = lambda t: (F.embedding(tokens, t.detach(), scale=2.0).double() * w.double()).sum()
    left, right = float((dW.double() * v.double()).sum()), float((f(W + v) - f(W - v)) / 2)
    # every output of some 4 in size is rounded twice, weighed by |w| and added: 1440 terms
    assert abs(left - right) <= 1440 * 16 * U * 4


def test_embedding_offsets_beyond_32_bits():
    V, D = 70000, 32768                        # 2.3e9 elements
    W = torch.empty(V, D, device="cuda", dtype=torch.float16)
    W[-3:] = torch.randn(3, D, generator=gen(11), device="cuda").half()
    tokens = torch.tensor([V - 1, V - 3, V - 1], device="cuda")
    W.requires_grad_()
    out = F.embedding(tokens, W)
    assert torch.equal(out, W.detach()[tokens])
    dout = torch.ones_like(out)
    (dW,) = torch.autograd.grad(out, W, dout)
    assert (dW[-3:] == torch.tensor([1.0, 0.0, 2.0], device="cuda", dtype=torch.float16)[:, None]).all()
    assert not dW[:-3].any()


# ---------------------------------------------------------------- dropout
def expected_dropout(x, p, seed, offset=0, shared_dim=None):
    shape = list(x.shape)
    if shared_dim is not None:
        shape[shared_dim] = 1
    mask = torch.from_numpy(O.kept(int(np.prod(shape)), p, seed, offset).reshape(shape)).to(x.device)
    scale = torch.tensor(1 / (1 - p) if p < 1 else 0.0, dtype=torch.float32)
    return torch.where(mask, x.detach().float() * scale, 0.0).to(x.dtype)


def check_dropout(x, p, seed, offset=0, shared_dim=None, grad=None):
    x = x.detach().requires_grad_()
    y = F.dropout(x, p, seed, offset=offset, shared_dim=shared_dim)
    assert y.is_contiguous() and y.dtype == x.dtype
    assert torch.equal(y, expected_dropout(x, p, seed, offset, shared_dim))
    grad = torch.randn(x.shape, generator=gen(6), device="cuda").to(x.dtype) if grad is None else grad
    (dx,) = torch.autograd.grad(y, x, grad)
    assert torch.equal(dx, expected_dropout(grad, p, seed, offset, shared_dim))
    return y


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", [(1,), (3,), (17,), (1, 1, 512), (2, 3, 8), (5, 7, 33), (19, 3, 301), (64, 16, 256), (3, 5, 2, 24), (4097,)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout_sizes(dtype, shape, p):
    x = torch.randn(shape, generator=gen(len(shape)), device="cuda").to(DT[dtype])
    check_dropout(x, p, seed=1234567 + len(shape), offset=3)
    for d in range(len(shape) - 1):
        check_dropout(x, p, 99, shared_dim=d)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,T,H", [(6, 10, 64), (5, 9, 33), (3, 130, 20)])
def test_dropout_layouts(dtype, B, T, H):
    g = gen(12)
    x = torch.randn(B, T, H, generator=g, device="cuda").to(DT[dtype])
    wide = torch.randn(B, T, H + 5, generator=g, device="cuda").to(DT[dtype])
    for v in (x.transpose(0, 1), wide[:, :, :H], wide[:, :, 5:], wide[:, ::2, :H].transpose(0, 1), x.permute(2, 0, 1), x[:, :1].expand(B, T, H),
              x.flatten()[1:], x.flatten()[3:-2]):
        for d in (None, 0, 1):
            if d is None or d < v.dim() - 1:
                check_dropout(v, 0.3, 7, 1, d)
    check_dropout(x, 0.3, 7, grad=x.transpose(0, 1).contiguous().transpose(0, 1))
    check_dropout(x, 0.3, 7, shared_dim=1, grad=torch.ones((), device="cuda", dtype=x.dtype).expand(B, T, H))


@pytest.mark.parametrize("seed,offset", [(0, 0), (1, 0), (0, 1), (2 ** 32, 5), (2 ** 64 - 1, 2 ** 64 - 1), (0x123456789ABCDEF, 2 ** 40)])
def test_dropout_seeds(seed, offset):
    x = torch.randn(33, 65, generator=gen(13), device="cuda")
    y = check_dropout(x, 0.4, seed, offset)
    assert torch.equal(y, F.dropout(x, 0.4, seed, offset=offset))
    assert not torch.equal(y, F.dropout(x, 0.4, seed, offset=offset ^ 1))
    if seed < 2 ** 63:
        at = torch.tensor([seed], device="cuda")
        assert torch.equal(y, F.dropout(x, 0.4, at, offset=offset))


@pytest.mark.parametrize("p", [0.0, 1.0, 1e-12, 1 - 1e-12])
def test_dropout_extremes(p):
    x = torch.randn(40, 50, generator=gen(14), device="cuda").bfloat16()
    y = check_dropout(x, p, 5) if p != 1 - 1e-12 else F.dropout(x, p, 5)
    assert torch.equal(y, x) if p < 0.5 else not y.any()


def test_dropout_share_and_dropped_values():
    n = 1 << 20
    x = torch.full((n,), float("inf"), device="cuda")
    x[::2] = float("nan")
    y = F.dropout(x, 0.3, 77)
    kept = torch.from_numpy(O.kept(n, 0.3, 77)).cuda()
    assert not y[~kept].any() and not y[kept].isfinite().any()
    # a binomial share, six standard deviations
    assert abs(float(kept.double().mean()) - 0.7) <= 6 * (0.21 / n) ** 0.5


def test_dropout_seed_on_the_gpu_changes_between_replays():
    x, seed = torch.randn(64, 128, device="cuda"), torch.tensor(3, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.dropout(x, 0.5, seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F.dropout(x, 0.5, seed)
    for s in (3, 4):
        seed.fill_(s)
        graph.replay()
        assert torch.equal(y, expected_dropout(x, 0.5, s))
    # a seed that changes between forward and backward would draw another mask: refused
    v = x.detach().requires_grad_()
    out = F.dropout(v, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_dropout_without_elements():
    for shape in ((0,), (0, 4, 5), (4, 0, 5), (4, 5, 0)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        y = F.dropout(x, 0.5, 1)
        assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape


def test_dropout_offsets_beyond_32_bits():
    n = 2 ** 32 + 4 * 5003
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = F.dropout(x, 0.25, 9, offset=2)
    for first, count in ((0, 4096), (2 ** 31 - 2048, 4096), (2 ** 32 - 2048, 4096), (n - 4096, 4096)):
        want = torch.from_numpy(O.kept(count, 0.25, 9, 2, first)).cuda()
        assert torch.equal(y[first:first + count] != 0, want)
    del y
    rows = x[:2 ** 32].view(2 ** 16, 2 ** 11, 32).transpose(0, 1)
    y = F.dropout(rows, 0.25, 9, offset=2)
    assert torch.equal(y.view(-1)[-4096:] != 0, torch.from_numpy(O.kept(4096, 0.25, 9, 2, 2 ** 32 - 4096)).cuda())


# ---------------------------------------------------------------- log probabilities
def check_scores(logits, tokens, dtype, top=0, temperature=1.0, ignore=-100, grads=True):
    """logits and tokens may have any leading dimensions and strides."""
    logits = logits.detach().requires_grad_(grads)
    V = logits.shape[-1]
    r = F.token_log_probs(logits, tokens, top=top, temperature=temperature, ignore_index=ignore)
    assert r.log_probs.shape == r.entropy.shape == tokens.shape
    assert all(t is None for t in r[2:]) if top == 0 else r.top_log_probs.shape == r.top_tokens.shape == (*tokens.shape, top)
    z, t = np64(logits).reshape(-1, V), tokens.cpu().numpy().reshape(-1)
    want = O.token_log_probs(z, t, top, temperature, ignore)
    finite = np.where(np.isfinite(want["lp"]), want["lp"], 0)
    D = float(np.abs(finite).max(initial=0)) * 1.4427 + 1
    C = (4 * D + 16 + V / 64) * U
    names = ["log_probs", "entropy"] + (["top_log_probs"] if top else [])
    for name, bound in zip(names, (C, C * (D + 4), C)):
        got, ref = np64(getattr(r, name)).reshape(want[name].shape), want[name]
        fine = np.isfinite(ref)
        assert np.array_equal(got[~fine], ref[~fine], equal_nan=True), name
        within(got[fine], ref[fine], bound, name)
    if top:
        assert np.array_equal(r.top_tokens.cpu().numpy().reshape(-1, top), want["top_tokens"])
    if not grads:
        return
    g = gen(15)
    ups = [torch.randn(getattr(r, n).shape, generator=g, device="cuda") for n in names]
    outs = [getattr(r, n) for n in names]
    (dz,) = torch.autograd.grad(outs, logits, ups, retain_graph=True)
    assert dz.shape == logits.shape and dz.dtype == logits.dtype
    flat = [np64(u).reshape(len(t), -1) for u in ups]
    ref, size = O.token_log_probs_grad(z, t, flat[0][:, 0], flat[1][:, 0], flat[2] if top else None, temperature, ignore)
    bound = (C * (D + 4) * size + 8 * U * np.abs(ref)) + EPS[dtype] * np.abs(ref) + TINY[dtype] + C / temperature * 1e-6
    within(np64(dz).reshape(ref.shape), ref, bound, "dlogits")
    # of one output alone
    if not len(t):
        return
    (dz,) = torch.autograd.grad(outs[0], logits, ups[0].reshape(-1)[0].expand(outs[0].shape), retain_graph=True)
    ref, size = O.token_log_probs_grad(z, t, np.full(len(t), flat[0][0, 0]), None, None, temperature, ignore)
    within(np64(dz).reshape(ref.shape), ref, C * (D + 4) * size + (EPS[dtype] + 8 * U) * np.abs(ref) + TINY[dtype] + C / temperature * 1e-6, "dlogits of log_probs")


def make_logits(g, *shape, dtype="bf16", std=3.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,vocab", [(1, 1), (1, 2), (3, 31), (40, 64), (17, 205), (9, 1000), (5, 1023), (5, 1024), (5, 1025), (4, 2048), (6, 4099),
                                     (3, 10007), (2, 33001), (1, 131072), (700, 513), (300, 2500)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_scores_sizes(dtype, n, vocab, top):
    g = gen(n + vocab)
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    check_scores(make_logits(g, n, vocab, dtype=dtype), tokens, dtype, min(top, vocab), 1.0 if n % 2 else 0.7)


@pytest.mark.parametrize("vocab", [50, 700, 1500, 9000, 70000])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few values", "two far", "block at the end"])
def test_scores_ties_and_orders(vocab, kind):
    """Where the alternatives sit must not matter: equal logits everywhere, sorted ones, all the large ones side by side."""
    j = torch.arange(vocab, device="cuda").float()
    row = {"equal": j * 0 + 2.5, "rising": j / vocab * 4, "falling": -j / vocab * 4, "few values": j % 7,
           "two far": torch.where((j == 3) | (j == vocab - 1), 100.0, 0.0), "block at the end": torch.where(j >= vocab - 45, 5.0, -1.0)}[kind]
    tokens = torch.tensor([0, vocab - 1], device="cuda")
    for dtype in ("fp32", "bf16"):
        check_scores(row.to(DT[dtype]).expand(2, vocab), tokens, dtype, top=min(32, vocab))
        check_scores(row.to(DT[dtype]).expand(2, vocab), tokens, dtype, top=1, grads=False)


@pytest.mark.parametrize("vocab", [40, 600, 3000, 40000])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_scores_masks(vocab, dtype):
    g = gen(16)
    z = make_logits(g, 8, vocab, dtype=dtype)
    low = torch.finfo(DT[dtype]).min
    z[1, ::2] = -float("inf")
    z[2, 1:] = -float("inf")                    # one token possible
    z[3] = -float("inf")                        # none
    z[4, : vocab - 3] = low
    z[5] = low                                  # all equal
    z[6, 5:] = -float("inf")                    # fewer than there are alternatives
    tokens = torch.zeros(8, dtype=torch.long, device="cuda")
    check_scores(z, tokens, dtype, top=20)
    check_scores(z, tokens, dtype, top=0, temperature=1.5)
    r = F.token_log_probs(z.requires_grad_(), tokens, top=2)
    assert r.log_probs[3] == -float("inf") and r.entropy[3] == 0 and r.top_tokens[3].tolist() == [0, 1]
    assert r.log_probs[2] == 0 and r.entropy[2] == 0 and r.top_log_probs[2].tolist() == [0, -float("inf")]
    d = torch.autograd.grad(r.log_probs[2:4].sum() + r.entropy.sum(), z)[0]
    assert not d[3].any() and not d[2].any() and d.isfinite().all()


@pytest.mark.parametrize("vocab", [100, 2000, 20000])
def test_scores_not_a_number_and_infinity(vocab):
    z = make_logits(gen(17), 4, vocab, dtype="fp32")
    z[1, vocab // 2] = float("nan")
    z[2, vocab - 1] = float("inf")
    tokens = torch.ones(4, dtype=torch.long, device="cuda")
    z.requires_grad_()
    r = F.token_log_probs(z, tokens, top=3)
    for t in (r.log_probs, r.entropy, r.top_log_probs):
        assert t[1:3].isnan().all() and t[::3].isfinite().all()
    assert r.top_tokens[1, 0] == vocab // 2 and r.top_tokens[2, 0] == vocab - 1
    (d,) = torch.autograd.grad(r.log_probs.sum(), z)
    assert d[1:3].isnan().all() and d[::3].isfinite().all()


@pytest.mark.parametrize("offset", [1000.0, -20000.0])
def test_scores_common_offset(offset):
    """Only differences count: logits that are exact in 32 bits next to a large offset give what they give without it."""
    z = torch.randint(-40, 40, (5, 3001), generator=gen(18), device="cuda").float() / 8
    tokens = torch.arange(5, device="cuda")
    a, b = F.token_log_probs(z, tokens, top=4), F.token_log_probs(z + offset, tokens, top=4)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_scores_ignored_rows():
    g = gen(19)
    for n, vocab, ignore in ((6, 300, -100), (5, 5000, 0), (7, 40, 3)):
        z = make_logits(g, n, vocab)
        tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
        tokens[1::2] = ignore
        z[1::2] = float("nan")                  # not read
        zn = z.clone()
        zn[1::2] = 0
        r = F.token_log_probs(z, tokens, top=2, ignore_index=ignore)
        assert not r.log_probs[1::2].any() and not r.entropy[1::2].any()
        assert (r.top_log_probs[1::2] == -float("inf")).all() and (r.top_tokens[1::2] == -1).all()
        check_scores(zn, tokens, "bf16", 2, 1.0, ignore)
        v = z.requires_grad_()
        assert not torch.autograd.grad(F.token_log_probs(v, tokens, ignore_index=ignore).log_probs.sum(), v)[0][1::2].any()
        check_scores(zn, torch.full_like(tokens, ignore), "bf16", 2, 1.0, ignore)


@pytest.mark.parametrize("vocab", [77, 512, 1300, 6007])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_scores_layouts(vocab, dtype):
    g = gen(20)
    T, B = 5, 3
    tokens = torch.randint(0, vocab, (B, T), generator=g, device="cuda")
    z = make_logits(g, B, T, vocab, dtype=dtype)
    wide = make_logits(g, B, T, vocab + 9, dtype=dtype)
    for v in (z, wide[..., :vocab], wide[..., 9:], wide[..., 1:vocab + 1], make_logits(g, vocab, B, T, dtype=dtype).permute(1, 2, 0), z[:, :1].expand(B, T, vocab)):
        check_scores(v.transpose(0, 1), tokens.t(), dtype, 3)
        check_scores(v[:, -1], tokens[:, -1].int(), dtype, 1)
        check_scores(v[0, 0], tokens[0, 0], dtype, 2)
    check_scores(z.view(1, B, T, vocab).expand(2, B, T, vocab), tokens.expand(2, B, T), dtype, 1)


def test_scores_without_rows():
    z = torch.randn(0, 7, device="cuda", requires_grad=True)
    r = F.token_log_probs(z, torch.zeros(0, dtype=torch.long, device="cuda"), top=2)
    assert r.log_probs.shape == (0,) and r.top_tokens.shape == (0, 2)
    assert torch.autograd.grad(r.log_probs.sum(), z)[0].shape == (0, 7)


@pytest.mark.parametrize("vocab", [60, 5000])
def test_scores_tokens_outside_of_the_vocabulary(vocab):
    z = make_logits(gen(21), 5, vocab, dtype="fp32").requires_grad_()
    for bad in (vocab, -1, -2 ** 50):
        tokens = torch.tensor([0, 1, bad, 2, 3], device="cuda")
        r = F.token_log_probs(z, tokens, top=1)
        with pytest.raises(BlstmError, match="at position 2"):
            F.check_status()
        assert r.log_probs[2].isnan() and r.log_probs[[0, 1, 3, 4]].isfinite().all() and r.entropy.isfinite().all()
        (d,) = torch.autograd.grad(r.log_probs.nan_to_num().sum(), z)
        F.check_status()
        assert not d[2].any() and d[0].any()


def test_scores_gradient_against_differences():
    """A central difference along a direction v, in 32 bits: its own error is h^2/6 times the third derivative (of some
    |v|_inf^3 |w| per row, here below 30) and the outputs' 4 u |lp| over h."""
    g = gen(22)
    for vocab, top in ((90, 3), (2000, 3)):
        z = make_logits(g, 6, vocab, dtype="fp32").requires_grad_()
        tokens = torch.randint(0, vocab, (6,), generator=g, device="cuda")
        v = torch.randn(6, vocab, generator=g, device="cuda")
        w = [torch.randn(6, generator=g, device="cuda"), torch.randn(6, generator=g, device="cuda"), torch.randn(6, top, generator=g, device="cuda")]

        def f(x):
            r = F.token_log_probs(x, tokens, top=top, temperature=0.9)
            return sum((a.double() * b.double()).sum() for a, b in zip(r[:3], w))
        r = F.token_log_probs(z, tokens, top=top, temperature=0.9)
        (d,) = torch.autograd.grad(r[:3], z, w)
        h = 2.0 ** -9
        with torch.no_grad():
            slope = float((f(z + h * v) - f(z - h * v)) / (2 * h))
        assert abs(slope - float((d.double() * v.double()).sum())) <= 30 * 30 * h * h + 30 * 20 * 4 * U / h


def test_scores_offsets_beyond_32_bits():
    V, n = 50000, 43008                         # 2.15e9 logits
    z = torch.zeros(n, V, device="cuda", dtype=torch.bfloat16)
    z[-2:] = make_logits(gen(23), 2, V)
    tokens = torch.arange(n, device="cuda") % V
    z.requires_grad_()
    r = F.token_log_probs(z, tokens, top=2)
    want = O.token_log_probs(np64(z[-2:]), tokens[-2:].cpu().numpy(), 2)
    assert np.array_equal(r.top_tokens[-2:].cpu().numpy(), want["top_tokens"]) and (r.top_tokens[:-2] == torch.tensor([0, 1], device="cuda")).all()
    np.testing.assert_allclose(np64(r.log_probs[-2:]), want["log_probs"], atol=2e-3)
    assert torch.allclose(r.log_probs[:-2], torch.tensor(-float(np.log(V)), device="cuda"), atol=2e-4)
    (d,) = torch.autograd.grad(r.log_probs, z, torch.ones_like(r.log_probs))
    ref, _ = O.token_log_probs_grad(np64(z[-2:]), tokens[-2:].cpu().numpy(), np.ones(2))
    np.testing.assert_allclose(np64(d[-2:]), ref, rtol=2e-2, atol=1e-6)
    i = torch.arange(0, n - 2, 997, device="cuda")
    assert (d[i, tokens[i]] > 0.99).all() and (d[i, (tokens[i] + 1) % V] < 0).all()


# ---------------------------------------------------------------- all of them
def test_refusals():
    x, t = torch.randn(3, 4, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    cases = [
        (lambda: F.embedding(t.cpu(), x), "must be a CUDA"), (lambda: F.embedding(t.float(), x), "dtype"), (lambda: F.embedding(t, x[0]), "expected weight"),
        (lambda: F.embedding(t, x.double()), "unsupported dtype"), (lambda: F.embedding(t, x[:0]), "expected weight"),
        (lambda: F.embedding(t, x, padding_idx=3), "padding_idx"), (lambda: F.embedding(t, x, padding_idx=-4), "padding_idx"),
        (lambda: F.embedding(t, x, scale=float("nan")), "scale"),
        (lambda: F.dropout(x, 1.1, 0), "p must"), (lambda: F.dropout(x, float("nan"), 0), "p must"), (lambda: F.dropout(x.long(), 0.5, 0), "unsupported dtype"),
        (lambda: F.dropout(x, 0.5, 0, shared_dim=1), "shared_dim"), (lambda: F.dropout(x, 0.5, 0, shared_dim=-1), "shared_dim"),
        (lambda: F.dropout(x, 0.5, 0, shared_dim=2), "shared_dim"), (lambda: F.dropout(x, 0.5, t), "seed"),
        (lambda: F.dropout(x, 0.5, x[0, :1]), "seed"), (lambda: F.dropout(x, 0.5, t[:1].cpu()), "seed"),
        (lambda: F.token_log_probs(x, t[:2]), "tokens have shape"), (lambda: F.token_log_probs(x, t, top=5), "top must"), (lambda: F.token_log_probs(x, t, top=-1), "top must"),
        (lambda: F.token_log_probs(x.expand(3, 3, 4), t), "tokens have shape"), (lambda: F.token_log_probs(x, t, temperature=0), "temperature"),
        (lambda: F.token_log_probs(torch.randn(3, 40, device="cuda"), t, top=33), "top must"), (lambda: F.token_log_probs(x[:, :0], t), "expected logits"),
        (lambda: F.token_log_probs(x, t.float()), "dtype"), (lambda: F.token_log_probs(x.double(), t), "unsupported dtype"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()


def test_gradients_of_gradients_are_refused():
    x, t = torch.randn(3, 4, device="cuda", requires_grad=True), torch.zeros(3, dtype=torch.long, device="cuda")
    for out in (F.embedding(t, x), F.dropout(x, 0.5, 0), F.token_log_probs(x, t).log_probs):
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_forward_mode_gradients_are_refused():
    from torch.autograd import forward_ad
    x, t = torch.randn(3, 4, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: F.embedding(t, dual), lambda: F.dropout(dual, 0.5, 0), lambda: F.token_log_probs(dual, t)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_another_stream_and_no_gradients():
    """Calls on a side stream are ordered with it, and what they return without gradients is the same."""
    g = gen(24)
    W, t = torch.randn(500, 64, generator=g, device="cuda", requires_grad=True), torch.randint(0, 500, (4000,), generator=g, device="cuda")

    def all_of_them():
        e = F.embedding(t, W, scale=2.0)
        return [e, F.dropout(e, 0.5, 3), *F.token_log_probs(e, t % 64, top=3)]
    want = all_of_them()
    grads = torch.autograd.grad([want[1], want[2]], W, [torch.ones_like(want[1]), torch.ones_like(want[2])])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = all_of_them()
        again = torch.autograd.grad([got[1], got[2]], W, [torch.ones_like(got[1]), torch.ones_like(got[2])])
    side.synchronize()
    with torch.no_grad():
        free = all_of_them()
    assert not any(v.requires_grad for v in free)
    for a, b, c in zip(want, got, free):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert torch.equal(grads[0], again[0])


# ---------------------------------------------------------------- together
def _example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "language_model.py")
    spec = importlib.util.spec_from_file_location("language_model", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_language_model_gradients_match_torch():
    """One step of the example's model without dropout against torch's own layers in 64 bits: each of the four operators that the
    gradients pass through is within 1e-5 of its tensor's norm in fp32."""
    m = _example()
    torch.manual_seed(3)
    model = m.LanguageModel(70, 48, layers=2, dropout=0.0, dtype=torch.float32)
    tokens, targets = m.batch(70, 12, 5, gen(1))
    loss = model.loss(tokens, targets, entropy_weight=0.1)
    grads = torch.autograd.grad(loss, list(model.parameters()))
    table = model.table.detach().double().requires_grad_()
    layers = [torch.nn.LSTM(48, 48, dtype=torch.float64, device="cuda") for _ in range(2)]
    for a, b in zip(layers, model.layers):
        a.load_state_dict({k: v.double() for k, v in b.state_dict().items()})
    x = torch.nn.functional.embedding(tokens, table, padding_idx=m.PADDING) * 48 ** 0.5
    for layer in layers:
        x, _ = layer(x)
    lp = torch.log_softmax(x @ table.t(), -1)
    live = targets != m.PADDING
    want = -((lp.gather(2, targets[..., None])[..., 0] - 0.1 * (lp.exp() * lp).sum(-1)) * live).sum() / live.sum()
    ref = torch.autograd.grad(want, [table] + [p for layer in layers for p in layer.parameters()])
    assert abs(float(loss.detach()) - float(want.detach())) <= 4e-5 * abs(float(want.detach()))
    for (name, _), a, b in zip(model.named_parameters(), grads, ref):
        assert float((a.double() - b).norm()) <= 4e-5 * float(b.norm()), name


def test_language_model_learns_and_repeats():
    m = _example()

    def once():
        torch.manual_seed(5)
        model = m.LanguageModel(60, 64, layers=2, dropout=0.1, dtype=torch.float32)
        return model, m.train(model, 60, T=24, B=32)
    model, losses = once()
    assert losses == once()[1]
    assert sum(losses[-5:]) < 0.5 * sum(losses[:5])
    model.eval()
    start = 1 + torch.arange(8, device="cuda")[:, None] * torch.tensor([1, 2], device="cuda")
    tokens, lp, top_tokens, top_lp = model.go_on(start, 4, top=3)
    assert tokens.shape == lp.shape == (4, 2) and top_tokens.shape == top_lp.shape == (4, 2, 3)
    assert torch.equal(tokens, top_tokens[..., 0]) and (top_lp[..., :-1] >= top_lp[..., 1:]).all()
