"""The root-mean-square norm against its oracle in 64 bits, at the sizes, strides and values where it can go wrong.

Tolerances.  u = 2^-24 is the rounding of 32 bits, e that of the type, tiny the spacing of fp16's subnormal numbers.  A sum over D
products is added up by 32 threads at least, none of which adds more than D / 32 + 40 terms in a row, and joined in ten steps: a
relative error of C u, C = D / 32 + 50; the inverse root has half of that and three roundings of its own (two in the last place of
the reciprocal root).  y is two products behind it: (C / 2 + 6) u relative, and e.  dx: each of its two terms has the errors of i
(squared in one), of the sum and of four products: (2 C + 16) u of the terms' magnitudes, and e.  dw: N terms: (N + 60 + C / 2) u of
their magnitudes, and e.  In 8 bits a value is off by half a step, 2^-4 of itself or 2^-10 of the scale, besides."""
import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from oracle import language_oracle as O

from test_gpu_language import DT, EPS, TINY, U, gen, np64, within

pytestmark = pytest.mark.gpu


def check(x, w, dtype, residual=None, eps=1e-6, dy=None, dh=None):
    D = x.shape[-1]
    C = D / 32 + 50
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    r = None if residual is None else residual.detach().requires_grad_()
    out = F.rms_norm(x, w, residual=r, eps=eps)
    y, h = out if r is not None else (out, x)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous() and h.dtype == x.dtype
    if r is not None:
        assert torch.equal(h, (x.float() + r.float()).to(x.dtype)) and h.is_contiguous()
    want, _ = O.rms_norm(np64(h), np64(w), eps)
    within(np64(y), want, ((C / 2 + 6) * U + EPS[dtype]) * np.abs(want) + TINY[dtype], "y")
    # without gradients: the same numbers
    with torch.no_grad():
        again = F.rms_norm(x, w, residual=r, eps=eps)
    assert torch.equal(again if r is None else again[0], y) and (r is None or torch.equal(again[1], h))
    # in 8 bits
    q = F.rms_norm_e4m3(x.detach(), w.detach(), residual=None if r is None else r.detach(), eps=eps)
    assert q.values.dtype == torch.float8_e4m3fn and q.values.shape == x.shape and q.scales.shape == x.shape[:-1] and q.scales.dtype == torch.float32
    assert (q.sum is None) if r is None else torch.equal(q.sum, h)
    most = np.abs(want).max(-1) / 448
    within(np64(q.scales), most, (C / 2 + 8) * U * most, "scales")
    scale = np64(q.scales)[..., None]
    within(np64(q.values) * scale, want, (2.0 ** -4 + (C / 2 + 12) * U) * np.abs(want) + 2.0 ** -10 * scale, "values")
    # gradients
    g = gen(3)
    dy = torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) if dy is None else dy
    if r is not None:
        dh = torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) if dh is None else dh
    outs, ups, ins = ([y], [dy], [x, w]) if r is None else ([y, h], [dy, dh], [x, r, w])
    grads = torch.autograd.grad(outs, ins, ups, retain_graph=True)
    repeat = torch.autograd.grad(outs, ins, ups)
    assert all(torch.equal(a, b) and a.dtype == x.dtype for a, b in zip(grads, repeat))
    dx, dw, size, size_w = O.rms_norm_grad(np64(h), np64(w), np64(dy), None if r is None else np64(dh), eps)
    for t in grads[:-1]:
        assert t.shape == x.shape
        within(np64(t), dx, (2 * C + 16) * U * size + EPS[dtype] * np.abs(dx) + TINY[dtype], "dx")
    N = x.numel() // D
    within(np64(grads[-1]), dw, (N + 60 + C / 2) * U * size_w + EPS[dtype] * np.abs(dw) + TINY[dtype], "dw")


def rows(g, *shape, dtype="bf16", std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,width", [(1, 1), (1, 8), (3, 7), (5, 16), (17, 33), (4, 255), (9, 256), (6, 301), (33, 512), (5, 520), (7, 1000), (6, 1024),
                                     (3, 1025), (5, 2048), (3, 2053), (2, 4096), (3, 4099), (2, 8192), (2, 8200), (3, 16400)])
@pytest.mark.parametrize("residual", [False, True])
def test_sizes(dtype, n, width, residual):
    g = gen(n + width)
    check(rows(g, n, width, dtype=dtype), 1 + rows(g, width, dtype=dtype, std=0.3), dtype, rows(g, n, width, dtype=dtype) if residual else None)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", [7, 64, 301, 512, 2053, 16400])
def test_eight_bits_of_tiny_rows(dtype, width):
    """448 over a magnitude below 2^-119 is infinite: such rows are zeros; those above 2^-110 have their values as ever."""
    x = rows(gen(width), 5, width, dtype=dtype)
    x[:, 0] = 0
    x[1] = 0
    q = F.rms_norm_e4m3(x, torch.full((width,), 2.0 ** -122, dtype=DT[dtype], device="cuda"))
    assert (q.scales == 0).all() and (q.values.float() == 0).all()
    w = torch.full((width,), 2.0 ** -105, dtype=DT[dtype], device="cuda")
    q = F.rms_norm_e4m3(x, w)
    C = width / 32 + 50
    want, _ = O.rms_norm(np64(x), np64(w), 1e-6)
    most = np.abs(want).max(-1) / 448
    within(np64(q.scales), most, (C / 2 + 8) * U * most, "scales")
    scale = np64(q.scales)[..., None]
    within(np64(q.values) * scale, want, (2.0 ** -4 + (C / 2 + 12) * U) * np.abs(want) + 2.0 ** -10 * scale, "values")


@pytest.mark.parametrize("dtype,n,width", [("bf16", 20011, 64), ("fp32", 7001, 301), ("fp16", 5003, 515), ("bf16", 3001, 1536), ("bf16", 1201, 7000)])
def test_many_rows(dtype, n, width):
    """More rows than blocks, so that each has several."""
    g = gen(width)
    check(rows(g, n, width, dtype=dtype), 1 + rows(g, width, dtype=dtype, std=0.3), dtype, rows(g, n, width, dtype=dtype))


@pytest.mark.parametrize("width", [64, 40, 33, 1100, 1101])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype, width):
    """Views: turned, cut out of wider rows, on odd addresses, expanded, of more and fewer dimensions, with a last dimension that is
    not dense."""
    g, B, T = gen(width), 5, 9
    w = 1 + rows(g, width, dtype=dtype, std=0.3)
    a, b = rows(g, B, T, width, dtype=dtype), rows(g, T, B, width, dtype=dtype)
    check(a.transpose(0, 1), w, dtype, b)
    check(b, w, dtype, a.transpose(0, 1), dy=rows(g, T, 1, width, dtype=dtype).expand(T, B, width), dh=rows(g, B, T, width, dtype=dtype).transpose(0, 1))
    check(rows(g, T, B, width + 3, dtype=dtype)[..., 1:-2], w, dtype, rows(g, T, B, width + 8, dtype=dtype)[..., :width])
    flat = rows(g, T * B * width + 5, dtype=dtype)
    for shift in (1, 2, 5):
        check(flat[shift:shift + T * B * width].view(T, B, width), w, dtype, b)
    check(b[:, :1].expand(T, B, width), w, dtype, b)
    check(rows(g, 2, T, 1, B, width, dtype=dtype), w, dtype, rows(g, T, 2, 1, B, width, dtype=dtype).transpose(0, 1))
    check(b[0, 0], w, dtype, b[1, 0])
    check(rows(g, width, T, dtype=dtype).t(), rows(g, width, 2, dtype=dtype)[:, 1], dtype, dy=rows(g, width, T, dtype=dtype).t())
    check(b, rows(g, width + 1, dtype=dtype)[1:], dtype)


def test_no_rows():
    for residual in (False, True):
        x, w = torch.zeros(0, 5, 24, device="cuda", requires_grad=True), torch.ones(24, device="cuda", requires_grad=True)
        out = F.rms_norm(x, w, residual=x.detach() if residual else None)
        y = out[0] if residual else out
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == dx.shape == x.shape and not dw.any()
        assert F.rms_norm_e4m3(x.detach(), w.detach()).scales.shape == (0, 5)


@pytest.mark.parametrize("width", [24, 301, 3000, 20000])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_values(dtype, width):
    """Rows of zeros, of large and of small numbers; rows with NaN or infinity are NaN and leave the others alone."""
    g = gen(4)
    x = rows(g, 6, width, dtype=dtype)
    x[1] = 0
    x[2] *= 1000
    x[3] *= 1e-3
    w = 1 + rows(g, width, dtype=dtype, std=0.3)
    check(x, w, dtype)
    q = F.rms_norm_e4m3(x, w)
    assert float(q.scales[1]) == 0 and not q.values[1].float().any()
    bad = x.clone()
    bad[0, width // 2], bad[4, width - 1] = float("nan"), float("inf")
    y, good = F.rms_norm(bad, w), F.rms_norm(x, w)
    assert y[0].isnan().all() and y[4, width - 1].isnan() and not y[4, :-1].float().any()
    assert torch.equal(y[[1, 2, 3, 5]], good[[1, 2, 3, 5]])
    s = F.rms_norm_e4m3(bad, w)
    assert s.scales[0].isnan() and s.scales[4].isnan() and torch.equal(s.scales[[1, 2, 3, 5]], q.scales[[1, 2, 3, 5]])


@pytest.mark.parametrize("eps", [0.0, 1e-12, 0.5, 1e30])
def test_eps(eps):
    g = gen(5)
    check(rows(g, 5, 96, dtype="fp32"), rows(g, 96, dtype="fp32"), "fp32", eps=eps)


@pytest.mark.parametrize("width", [40, 301, 2500])
def test_gradient_against_differences(width):
    """<gradient, direction> against (f(+d) - f(-d)) / 2 of the operator in fp32; the weighted sum itself is taken in 64 bits.  Each of
    the two values carries 2^-24 of the terms' magnitudes at most times C / 2 + 7, divided by the step; the third derivative times the step
    squared is below 1e-4 of the result's size for steps of 1/64 of a standard deviation."""
    g = gen(width)
    x, r, d = (rows(g, 3, width, dtype="fp32") for _ in range(3))
    w, dw = 1 + rows(g, width, dtype="fp32", std=0.3), rows(g, width, dtype="fp32")
    up = [rows(g, 3, width, dtype="fp32").double() for _ in range(2)]

    def f(x, w):
        y, h = F.rms_norm(x, w, residual=r)
        return (y.double() * up[0]).sum() + (h.double() * up[1]).sum()
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y, h = F.rms_norm(a, b, residual=r)
    gx, gw = torch.autograd.grad((y, h), (a, b), [t.float() for t in up])
    step = 1 / 64
    size = float((y.detach().double() * up[0]).abs().sum() + (h.detach().double() * up[1]).abs().sum())
    for got, plus, minus in ((float((gx.double() * d).sum()), f(x + step * d, w), f(x - step * d, w)),
                             (float((gw.double() * dw).sum()), f(x, w + step * dw), f(x, w - step * dw))):
        assert abs(got - float(plus - minus) / (2 * step)) <= size * ((width / 64 + 32) * U / step + 1e-4)


def test_only_some_inputs_need_gradients():
    g = gen(6)
    x, r, w = rows(g, 7, 64), rows(g, 7, 64), rows(g, 64)
    up = rows(g, 7, 64)
    full = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = F.rms_norm(full[0], full[2], residual=full[1])
    want = torch.autograd.grad((y, h), full, (up, up))
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        t = [v.clone().requires_grad_(bool(n)) for v, n in zip((x, r, w), need)]
        y, h = F.rms_norm(t[0], t[2], residual=t[1])
        assert h.requires_grad == bool(need[0] or need[1]) and y.requires_grad
        outs = (y, h) if h.requires_grad else (y,)
        got = iter(torch.autograd.grad(outs, [v for v, n in zip(t, need) if n], (up, up)[:len(outs)]))
        for k in range(3):
            if need[k]:
                assert torch.equal(next(got), want[k])
    # only one of the two outputs is used
    t = [v.clone().requires_grad_() for v in (x, r, w)]
    y, h = F.rms_norm(t[0], t[2], residual=t[1])
    gx, gr, gw = torch.autograd.grad(h, t, up, allow_unused=True, retain_graph=True)
    assert torch.equal(gx, up) and torch.equal(gr, up) and (gw is None or not gw.any())
    gx, gr, gw = torch.autograd.grad(y, t, up)
    alone = [v.clone().requires_grad_() for v in (h.detach(), w)]
    hx, hw = torch.autograd.grad(F.rms_norm(alone[0], alone[1]), alone, up)
    assert torch.equal(gx, hx) and torch.equal(gr, hx) and torch.equal(gw, hw)


def test_one_tensor_as_both_terms_and_one_weight_twice():
    """Gradients of a leaf that is met twice add up."""
    g = gen(7)
    x, w = rows(g, 9, 48, dtype="fp32").requires_grad_(), rows(g, 48, dtype="fp32").requires_grad_()
    y, h = F.rms_norm(x, w, residual=x)
    z = F.rms_norm(y, w)
    (z.sum() + h.sum()).backward()
    a, b = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    f = lambda t: torch.nn.functional.rms_norm(t, (48,), b, 1e-6)
    (f(f(2 * a)).sum() + 2 * a.sum()).backward()
    assert float((x.grad - a.grad).abs().max()) <= 1e-4 * float(a.grad.abs().max())
    assert float((w.grad - b.grad).abs().max()) <= 1e-4 * float(b.grad.abs().max())


def test_saved_tensors_that_change_are_noticed():
    x, w, r = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((4, 32), (32,), (4, 32)))
    y, h = F.rms_norm(x, w, residual=r)
    with torch.no_grad():
        h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed on new inputs, while an eager graph of other leaves lives."""
    g = gen(8)
    x, r, w = rows(g, 65, 300, dtype="fp32"), rows(g, 65, 300, dtype="fp32"), rows(g, 300, dtype="fp32")
    up = rows(g, 65, 300, dtype="fp32")

    def step(a, b, c):
        y, h = F.rms_norm(a, c, residual=b)
        return (y, h, *torch.autograd.grad((y, h), (a, b, c), (up, up)))
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*leaves)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*leaves)
    for k in range(2):
        new = [rows(g, *t.shape, dtype="fp32") for t in leaves]
        with torch.no_grad():
            for a, b in zip(leaves, new):
                a.copy_(b)
        graph.replay()
        want = step(*[t.requires_grad_() for t in new])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    x, w = torch.randn(9, 40, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
    eager = F.rms_norm(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: F.rms_norm(x, w), lambda: F.rms_norm(x.detach(), w), lambda: F.dropout(x, 0.5, 1),
                     lambda: F.embedding(torch.zeros(3, dtype=torch.long, device="cuda"), x),
                     lambda: F.token_log_probs(x, torch.zeros(9, dtype=torch.long, device="cuda"))):
            with pytest.raises(RuntimeError, match="before the capture lives"):
                call()
    want = torch.autograd.grad(eager.sum(), (x, w))
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(F.rms_norm(x, w).sum(), (x, w))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


class Around(torch.nn.Module):
    """Every operator with a gradient, on leaves."""

    def __init__(self, seed):
        super().__init__()
        g = gen(seed)
        self.table = torch.nn.Parameter(torch.randn(50, 40, generator=g, device="cuda"))
        self.weight = torch.nn.Parameter(1 + 0.1 * torch.randn(40, generator=g, device="cuda"))
        self.tokens = torch.randint(0, 50, (9,), generator=g, device="cuda")

    def forward(self, x):
        y, h = F.rms_norm(F.dropout(x, 0.25, 7), self.weight, residual=F.embedding(self.tokens, self.table))
        r = F.token_log_probs(F.rms_norm(h, self.weight), self.tokens % 40, top=2)
        return r.log_probs.sum() + r.entropy.sum() + r.top_log_probs.sum() + y.sum()


def test_captures_beside_graphs_of_side_streams():
    """A graph from a side stream may live: its leaves' gradients are joined into the capture (torch.cuda.make_graphed_callables warms up on
    such a stream and keeps its last outputs)."""
    model, plain = Around(1), Around(1)
    x = torch.randn(9, 40, generator=gen(2), device="cuda", requires_grad=True)
    graphed = torch.cuda.make_graphed_callables(model, (x.detach().clone().requires_grad_(),))
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(9, 40, generator=gen(3 + k), device="cuda"))
        got = torch.autograd.grad(graphed(x), [x, *model.parameters()])
        want = torch.autograd.grad(plain(x), [x, *plain.parameters()])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_backward_captured_beside_a_graph_of_a_side_stream():
    """The same with gradients that are added up in the leaves."""
    model, plain = Around(4), Around(4)
    x = torch.randn(9, 40, generator=gen(5), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept = model(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model(x).backward()
    graph.replay()
    plain(x).backward()
    for a, b in zip(model.parameters(), plain.parameters()):
        assert torch.equal(a.grad, b.grad)
    kept.backward()
    for a, b in zip(model.parameters(), plain.parameters()):
        assert torch.equal(a.grad, 2 * b.grad)


def test_calls_at_once():
    """Forward and backward on two streams side by side."""
    g = gen(11)
    data = [[rows(g, 3001, 520), rows(g, 520), rows(g, 3001, 520)] for _ in range(2)]

    def step(x, w, up):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(F.rms_norm(a, b), (a, b), up)
    want = [step(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(8):
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(step(*d))
    torch.cuda.synchronize()
    for k, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[k % 2]))


def test_lazily_negated_inputs():
    """Numbers whose signs are still to be turned, in tensors that are dense all the same (rows of one element)."""
    g = gen(21)
    lazy = lambda *s: torch.view_as_complex(torch.randn(*s, 2, generator=g, device="cuda")).conj().imag
    x, r, w, up = lazy(5, 1), lazy(5, 1), lazy(1), lazy(5, 1)
    assert x.is_neg() and w.is_neg() and w.is_contiguous()
    plain = [t.clone() for t in (x, r, w, up)]
    assert not plain[0].is_neg()

    def norm(x, r, w, up):
        x, r, w = (t.detach().requires_grad_() for t in (x, r, w))
        y, h = F.rms_norm(x, w, residual=r, eps=0.5)
        q = F.rms_norm_e4m3(x.detach(), w.detach(), residual=r.detach())
        return [y, h, q.values.float(), q.scales, *torch.autograd.grad((y, h), (x, r, w), (up, up))]

    def others(x, r, w, up):
        zero = torch.zeros(5, dtype=torch.long, device="cuda")
        leaf = x.detach().requires_grad_()
        drop = F.dropout(leaf[:1], 0.0, 1)
        out = [drop, *torch.autograd.grad(drop, leaf, up[:1]), F.embedding(zero, w[None]), *F.token_log_probs(x.expand(5, 3), zero)[:2]]
        s = F.token_log_probs(leaf.expand(5, 3), zero, top=1)
        out += torch.autograd.grad((s.log_probs, s.top_log_probs), leaf, (up[:, 0], up), allow_unused=True)
        b = F.beam_step(x.view(5, 1, 1), r)
        out += [b.scores, *b[1:3]]
        p = w.clone().requires_grad_()
        p.grad = up[:1, 0]
        F.AdamW([p]).step()
        return out + [p.detach()]
    for f in (norm, others):
        for a, b in zip(f(x, r, w, up), f(*plain)):
            assert torch.equal(a, b)
    p = w.requires_grad_()
    p.grad = torch.ones(1, device="cuda")
    with pytest.raises(ValueError, match="negated"):
        F.AdamW([p]).step()


def test_another_stream():
    g = gen(9)
    x, w = rows(g, 513, 640), rows(g, 640)
    want = F.rms_norm(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = F.rms_norm(x, w)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    x, w = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda")
    for a, k in (((x, w[:7]), {}), ((x, w.half()), {}), ((x.double(), w.double()), {}), ((x, w.cpu()), {}), ((x, w), dict(residual=x[:2])),
                 ((x, w), dict(residual=x.half())), ((x, w), dict(eps=-1.0)), ((x, w), dict(eps=float("nan"))), ((x[:, :0], w[:0]), {}), ((w[0], w), {}),
                 ((x, w), dict(residual=x.cpu()))):
        for call in (F.rms_norm, F.rms_norm_e4m3):
            with pytest.raises(ValueError):
                call(*a, **k)
    with pytest.raises(ValueError, match="no gradient"):
        F.rms_norm_e4m3(x.requires_grad_(), w)
    with torch.no_grad():
        F.rms_norm_e4m3(x, w)
    y = F.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_offsets_beyond_32_bits():
    """Rows whose elements are numbered above 2^31 (bf16, 4.5 GB a tensor)."""
    n, D = 2 ** 21 + 77, 1032
    x = torch.zeros(n, D, device="cuda", dtype=torch.bfloat16)
    g = gen(10)
    at = torch.tensor([0, 5, n // 2, n - 2, n - 1], device="cuda")
    x[at] = rows(g, 5, D)
    w = rows(g, D)
    assert torch.equal(F.rms_norm(x, w)[at], F.rms_norm(x[at], w))
    leaf, small = x.requires_grad_(), x.detach()[at].requires_grad_()
    dy = rows(g, 5, D)
    up = torch.zeros(n, D, device="cuda", dtype=torch.bfloat16)
    up[at] = dy
    (a,) = torch.autograd.grad(F.rms_norm(leaf, w), leaf, up)
    (b,) = torch.autograd.grad(F.rms_norm(small, w), small, dy)
    assert torch.equal(a[at], b) and not a[1].any()
