"""The AdamW step against its oracle in 64 bits, at the sizes, alignments and values where it can go wrong.

Tolerances.  u = 2^-24, e the rounding of the parameter's type.  m' is a product, a product and a fused sum, with coefficients that are
rounded themselves: 4 u of the magnitudes that are added; v' the same with one product more, all of one sign: 5 u.  The gradient's factor
adds 4 u where gradients are clipped.  The step that is taken from p is m' through a root (2^-22), a quotient (2^-21) and two bias
corrections (exponentials to 2^-22, a reciprocal root to 2^-22): below 2^-19 of its magnitude, taken with the magnitudes that m' is the sum
of; p' has one rounding besides, 2 u of p, and e.  8 bits: an element's place among the e4m3 numbers is known to 16 u of its place and to the
error of m', in steps of the numbers' distance; where a rounding border is not nearer than that the number is the oracle's."""
import pickle

import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200._lib import BlstmError
from oracle import adamw_oracle as A

from test_gpu_language import DT, EPS, TINY, U, gen, np64, within

pytestmark = pytest.mark.gpu

HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def model(shapes, dtype, seed, make=None):
    """Parameters with gradients; a tenth of each gradient is 0."""
    g = gen(seed)
    params = []
    for k, s in enumerate(shapes):
        p = (torch.randn(s, generator=g, device="cuda") * 0.5).to(DT[dtype])
        p = make(p) if make else p
        p.requires_grad_()
        p.grad = (torch.randn(s, generator=g, device="cuda") * (torch.rand(s, generator=g, device="cuda") < 0.9) * 10.0 ** (k % 3 - 2)).to(DT[dtype])
        params.append(p)
    return params


def snapshot(o, params):
    """What the oracle starts from, flat and in 64 bits."""
    state = []
    for p in params:
        s, n = o.state.get(p), p.numel()
        if not s:
            state.append({"p": np64(p).reshape(-1), "m": np.zeros(n), "v": np.zeros(n), "step": 0})
            continue
        d = {k: np64(v).reshape(-1) for k, v in s.items() if v.dim()}
        d["step"] = int(s["step"])
        d["p"] = d["master"] if "master" in d else np64(p).reshape(-1)
        if "exp_avg_scale" in d:
            d["m"], d["v"] = A.each(d["exp_avg_scale"], n) * d["exp_avg"], (A.each(d["exp_avg_sq_root_scale"], n) * d["exp_avg_sq_root"]) ** 2
        else:
            d["m"], d["v"] = d["exp_avg"], d["exp_avg_sq"]
        state.append(d)
    return state


def check_step(o, params, dtype, norm=True):
    before, grads = snapshot(o, params), [np64(p.grad).reshape(-1) for p in params]
    total = np.sqrt(sum((g * g).sum() for g in grads))
    factor = 1.0 if o.max_norm is None else min(1.0, o.max_norm / (total + 1e-6))
    o.step()
    F.check_status()
    if o.max_norm is not None:
        # (squares of eight neighbours are added up in 32 bits)
        assert abs(float(o.grad_norm) - total) <= 6 * U * total
    clip = 4 * U if factor < 1 else 0.0
    group = o.param_groups[0]
    (b1, b2), number = group["betas"], 0
    for p, s, g in zip(params, before, grads):
        now, n, t = o.state[p], p.numel(), s["step"] + 1
        assert int(now["step"]) == t
        m, v, size = A.moments(s["m"], s["v"], g * factor, b1, b2)
        m_err, v_err = (4 * U + clip) * size + 1e-45, (5 * U + 2 * clip) * v + 1e-44
        if o.state_bits == 32:
            within(np64(now["exp_avg"]).reshape(-1), m, m_err, "exp_avg")
            within(np64(now["exp_avg_sq"]).reshape(-1), v, v_err, "exp_avg_sq")
        else:
            draws = A.words(n, group["seed"], t, number).astype(np.int64)
            root = np.sqrt(v)
            for name, x, err, draw in (("exp_avg", m, m_err, draws & 0xFFFF), ("exp_avg_sq_root", root, 2.0 ** -21 * root, draws >> 16)):
                scales = A.scales_of(x)
                got = np64(now[name + "_scale"])
                within(got, scales, A.scales_of(err) + 4 * U * scales, name + "_scale")
                place, step = A.position(x, got, draw)
                s_each = A.each(got, n)
                slack = 16 * U * place + np.divide(err, s_each * step, out=np.zeros(n), where=s_each > 0)
                codes = np.abs(np64(now[name]).reshape(-1))
                want = np.minimum(np.floor(place) * step, 448)
                if name == "exp_avg_sq_root":
                    want = np.where((root > 0) & (s_each > 0) & (want == 0), 2.0 ** -9, want)
                border = np.abs(place - np.rint(place)) <= slack
                assert (codes[~border] == want[~border]).all(), name
                # (few of them: a hundredth, or two where that is less than an element of a small tensor)
                assert (np.abs(codes - want)[border] <= step[border]).all() and border.sum() <= 2 + 0.01 * n, name
                if name == "exp_avg":
                    sign = np64(now[name]).reshape(-1) * m >= 0
                    assert (sign | (np.abs(m) <= m_err)).all()
        new = A.update(s["p"], m, v, t, group["lr"], b1, b2, group["eps"], group["weight_decay"])
        move = group["lr"] * size / (1 - b1 ** t) / (np.sqrt(v / (1 - b2 ** t)) + group["eps"])
        err = (2.0 ** -19 + clip) * move + 2 * U * np.abs(s["p"])
        if "master" in now:
            within(np64(now["master"]).reshape(-1), new, err + U * np.abs(new), "master")
            assert torch.equal(now["master"].to(p.dtype), p.detach())
        within(np64(p).reshape(-1), new, err + EPS[dtype] * np.abs(new) + TINY[dtype], "p")
        number += 1


SHAPES = [(1,), (7,), (8,), (255,), (256,), (257,), (2047,), (2048,), (2049,), (33, 61), (5, 3, 400), (70001,)]


@pytest.mark.parametrize("dtype,master", [("fp32", False), ("fp16", True), ("fp16", False), ("bf16", True), ("bf16", False)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
def test_sizes(dtype, master, bits, max_norm):
    params = model(SHAPES, dtype, 1)
    o = F.AdamW(params, **HYPER, state_bits=bits, master_weights=master, max_norm=max_norm, seed=2 ** 63 + 12345)
    for k in range(3):
        check_step(o, params, dtype)
        for q, p in zip(model(SHAPES, dtype, 10 + k), params):
            p.grad = q.grad
    assert ("master" in o.state[params[0]]) == master


def test_norms_that_are_kept():
    """What was asked for after a step stays that step's."""
    p = torch.zeros(50, device="cuda", requires_grad=True)
    o = F.AdamW([p], max_norm=1.0)
    norms = []
    for k in range(3):
        p.grad = torch.full((50,), float(k), device="cuda")
        o.step()
        norms.append(o.grad_norm)
    assert [round(float(n) / 50 ** 0.5, 5) for n in norms] == [0, 1, 2]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_addresses_on_odd_boundaries(bits, dtype):
    """Parameters and gradients that are pieces of flat buffers, as buckets hand them out."""
    def odd(p):
        flat = torch.zeros(p.numel() + 3, device="cuda", dtype=p.dtype)
        flat[3:] = p.reshape(-1)
        return flat[3:].view(p.shape)
    params = model(SHAPES, dtype, 2, odd)
    for p in params[::2]:
        p.grad = odd(p.grad)
    o = F.AdamW(params, **HYPER, state_bits=bits, max_norm=1.0)
    check_step(o, params, dtype)
    check_step(o, params, dtype)


def test_gradients_of_other_layouts():
    """Turned and expanded gradients; what lies between the elements of a cut one counts for nothing."""
    g = gen(3)
    params = [torch.randn(40, 30, generator=g, device="cuda", requires_grad=True) for _ in range(3)]
    params[0].grad = torch.randn(30, 40, generator=g, device="cuda").t()
    params[1].grad = torch.randn(40, 1, generator=g, device="cuda").expand(40, 30)
    params[2].grad = torch.full((40, 60), float("nan"), device="cuda")[:, ::2].normal_(generator=g)
    o = F.AdamW(params, **HYPER, max_norm=1.0)
    check_step(o, params, "fp32")


@pytest.mark.parametrize("count", [32, 33, 384, 385, 900])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(count, bits):
    params = model([(5 + k % 300,) for k in range(count)], "fp32", 4)
    o = F.AdamW(params, **HYPER, state_bits=bits, max_norm=0.7)
    check_step(o, params, "fp32")
    check_step(o, params, "fp32")


def test_types_side_by_side_and_parameters_without_gradients():
    """One norm over all types and groups; a tensor counts only its own steps; groups have their own rates."""
    params = model([(300,), (41, 7)], "fp32", 5) + model([(300,)], "bf16", 6) + model([(9,), (2000,)], "fp16", 7)
    o = F.AdamW([dict(params=params[:3], lr=0.5), dict(params=params[3:], betas=(0.5, 0.6), weight_decay=0.0)], lr=0.01, max_norm=1.0)
    late = params[1].grad
    params[1].grad = None
    kept = params[1].detach().clone()
    o.step()
    assert torch.equal(params[1].detach(), kept) and params[1] not in o.state
    params[1].grad = late
    total = np.sqrt(sum((np64(p.grad) ** 2).sum() for p in params))
    before = snapshot_one(params[3], o)
    o.step()
    assert [int(o.state[p]["step"]) for p in params] == [2, 1, 2, 2, 2]
    assert abs(float(o.grad_norm) - total) <= 6 * U * total
    m, v, _ = A.moments(before[0], before[1], np64(params[3].grad) * min(1, 1 / (total + 1e-6)), 0.5, 0.6)
    want = A.update(before[2], m, v, 2, 0.01, 0.5, 0.6, 1e-8, 0.0)
    assert np.abs(np64(o.state[params[3]]["master"]) - want).max() <= 1e-6


def snapshot_one(p, o):
    s = o.state[p]
    return np64(s["exp_avg"]), np64(s["exp_avg_sq"]), np64(s["master"])


@pytest.mark.parametrize("bits", [32, 8])
def test_like_torch_over_many_steps(bits):
    """Thirty steps beside torch's in 64 bits, with a schedule: each step moves a weight by its error at most, 2^-18 of the rate in 32 bits.  In 8
    bits moments are off by up to a step of e4m3 (2^-3) each, which chance spreads: means over 20000 weights stay within 5 %."""
    g = gen(8)
    p = torch.randn(20000, generator=g, device="cuda").requires_grad_()
    q = p.detach().double().clone().requires_grad_()
    mine, ref = F.AdamW([p], lr=0.01, state_bits=bits, seed=3), torch.optim.AdamW([q], lr=0.01)
    moved = 0.0
    start = q.detach().clone()
    scale = 10 ** (torch.rand(20000, generator=g, device="cuda") * 3 - 3)
    for t in range(30):
        for o in (mine, ref):
            o.param_groups[0]["lr"] = 0.01 / (1 + t)
        moved += 0.01 / (1 + t)
        p.grad = (torch.randn(20000, generator=g, device="cuda") + 0.5) * scale
        q.grad = p.grad.double()
        mine.step()
        ref.step()
    d, far = (p.detach().double() - q.detach()).abs(), (q.detach() - start).abs()
    if bits == 32:
        assert float(d.max()) <= 2.0 ** -18 * 3.3 * moved + 30 * U * float(q.detach().abs().max())
        s = ref.state[q]
        assert float((mine.state[p]["exp_avg"].double() - s["exp_avg"]).norm() / s["exp_avg"].norm()) <= 1e-6
    else:
        a, b = p.detach().double() - start, q.detach() - start
        assert abs(float((a * b).sum() / (b * b).sum()) - 1) <= 0.05 and float(d.norm()) <= 0.25 * float(far.norm())


def test_chance_keeps_the_mean_and_follows_the_seed():
    """A second moment that changes by a thousandth of itself in a step, far less than the numbers' distance, follows its mean over
    many elements: 65536 elements, each off by at most a step (a sixteenth of itself on average of the two binades' ends, an eighth at most)
    with both signs: the mean's standard deviation is below 2^-3 / sqrt(65536) a step, and five of those over 100 steps 2^-3 / 256 * 5 * 10."""
    n = 65536
    p = torch.zeros(n, device="cuda", requires_grad=True)

    def run(seed, steps=100):
        o = F.AdamW([p], lr=0.0, state_bits=8, seed=seed)
        g = gen(9)
        p.grad = 0.5 + torch.rand(n, generator=g, device="cuda")
        o.step()
        for _ in range(steps):
            p.grad = torch.zeros(n, device="cuda")
            o.step()
        return o.state[p]
    s = run(1)
    root = (s["exp_avg_sq_root"].float().view(-1, 256) * s["exp_avg_sq_root_scale"][:, None]).double().view(-1)
    g = gen(9)
    want = (0.001 * (0.5 + torch.rand(n, generator=g, device="cuda").double()) ** 2 * 0.999 ** 100).sqrt()
    assert abs(float((root / want).mean()) - 1) <= 2.0 ** -3 / 256 * 50
    again, other = run(1), run(2)
    assert all(torch.equal(s[k].float(), again[k].float()) for k in s)
    assert not torch.equal(s["exp_avg_sq_root"].float(), other["exp_avg_sq_root"].float())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_gradients_that_are_not_finite_change_nothing(bits, bad):
    params = model([(300,), (5000,), (3,)], "fp32", 11)
    o = F.AdamW(params, **HYPER, state_bits=bits, max_norm=1.0)
    o.step()
    keep = [p.detach().clone() for p in params] + [t.clone() for p in params for t in o.state[p].values()]
    params[1].grad[4321] = bad
    o.step()
    now = [p.detach() for p in params] + [t for p in params for t in o.state[p].values()]
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(keep, now)) and not bool(o.grad_norm.isfinite())
    params[1].grad[4321] = 0.5
    check_step(o, params, "fp32")


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_and_tiny_and_huge_gradients(bits):
    """Blocks of zeros stay zeros; gradients down to 2^-60 and up to 2^60 side by side, in one block and in blocks of their own."""
    p = torch.randn(2048, generator=gen(12), device="cuda").requires_grad_()
    g = torch.randn(2048, generator=gen(13), device="cuda")
    g[:256] = 0
    g[256:512] *= 2.0 ** -60
    g[512:768] *= 2.0 ** 60
    g[768:1024] *= 2.0 ** torch.linspace(-50, 10, 256, device="cuda")
    p.grad = g
    o = F.AdamW([p], **HYPER, state_bits=bits)
    check_step(o, [p], "fp32")
    s = o.state[p]
    assert not s["exp_avg"][:256].float().any()
    if bits == 8:
        assert (s["exp_avg_sq_root"].float()[256:] > 0).all() and float(s["exp_avg_scale"][0]) == 0
    check_step(o, [p], "fp32")
    assert p.detach().isfinite().all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_saved_and_loaded(bits, dtype, tmp_path):
    """A run that is saved and loaded goes on bit by bit."""
    def grads(params, k):
        for p, q in zip(params, model([(300,), (77, 9)], dtype, 20 + k)):
            p.grad = q.grad
    params = model([(300,), (77, 9)], dtype, 14)
    o = F.AdamW(params, **HYPER, state_bits=bits, seed=7)
    for k in range(3):
        grads(params, k)
        o.step()
    torch.save({"p": params, "o": o.state_dict()}, tmp_path / "run.pt")
    kept = torch.load(tmp_path / "run.pt")
    other = [p.detach().clone().requires_grad_() for p in kept["p"]]
    n = F.AdamW(other, lr=1.0, state_bits=bits)
    n.load_state_dict(kept["o"])
    for k in range(3, 5):
        grads(params, k), grads(other, k)
        o.step(), n.step()
    for a, b in zip(params, other):
        assert torch.equal(a, b) and all(torch.equal(o.state[a][k].float(), n.state[b][k].float()) for k in o.state[a])


def test_states_of_torch():
    p = torch.randn(500, generator=gen(15), device="cuda").requires_grad_()
    p.grad = torch.randn(500, generator=gen(16), device="cuda")
    ref = torch.optim.AdamW([p], **{k: v for k, v in HYPER.items()})
    ref.step()
    q = p.detach().clone().requires_grad_()
    o = F.AdamW([q], lr=1.0)
    o.load_state_dict(ref.state_dict())
    q.grad = p.grad.clone()
    check_step(o, [q], "fp32")
    ref.step()
    assert int(o.state[q]["step"]) == 2 and float((p - q).detach().abs().max()) <= 2e-6


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(bits):
    """A captured step, replayed with new gradients and rates, does what steps one by one do; the step is noticed as a change of the
    parameters."""
    params, twin = (model([(300,), (4000,)], "bf16", 17) for _ in range(2))
    rate, seed = torch.full((), 0.01, device="cuda"), 5
    o = F.AdamW(params, lr=rate, state_bits=bits, max_norm=0.5, seed=seed)
    ref = F.AdamW(twin, lr=0.01, state_bits=bits, max_norm=0.5, seed=seed)
    fresh = F.AdamW(params, lr=rate)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o.step()
    torch.cuda.current_stream().wait_stream(s)
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before a capture"):
            fresh.step()
        o.step()
    for k in range(3):
        for p, q, new in zip(params, twin, model([(300,), (4000,)], "bf16", 30 + k)):
            p.grad.copy_(new.grad)
            q.grad = new.grad
        rate.fill_(0.01 * (k + 1))
        ref.param_groups[0]["lr"] = float(rate)
        graph.replay()
        ref.step()
    for p, q in zip(params, twin):
        assert torch.equal(p, q) and all(torch.equal(o.state[p][k].float(), ref.state[q][k].float()) for k in o.state[p])
    assert float(o.grad_norm) == float(ref.grad_norm)


def test_first_step_captured():
    """After a state was loaded the first step may be a captured one, and steps one by one go on before its replays: what launches use lies
    outside of the graph's memory, which holds something else until then."""
    params = model([(300,), (4000,)], "bf16", 18)
    twin = model([(300,), (4000,)], "bf16", 18)
    ref = F.AdamW(twin, lr=0.01, max_norm=0.5)
    ref.step()
    o = F.AdamW(params, lr=0.01, max_norm=0.5)
    o.load_state_dict(ref.state_dict())
    with torch.no_grad():
        for p, q in zip(params, twin):
            p.copy_(q)
    pool = torch.cuda.graph_pool_handle()
    other, graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(other, pool=pool):
        full = [torch.full((4,), 12345, dtype=torch.int32, device="cuda") for _ in range(64)]
        del full
    other.replay()
    with torch.cuda.graph(graph, pool=pool):
        o.step()
    for k in range(2):
        o.step() if k == 0 else graph.replay()
        ref.step()
        for p, q in zip(params, twin):
            assert torch.equal(p, q) and int(o.state[p]["step"]) == int(ref.state[q]["step"]) == k + 2
    # one that was never used has no place for it
    copy = pickle.loads(pickle.dumps(o))
    for p in copy.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        with pytest.raises(RuntimeError, match="before a capture"):
            copy.step()
    copy.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizers_at_once(bits):
    """Two optimizers on two streams side by side."""
    def run(streams):
        sides = []
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                params = model([(300,), (70001,)], "bf16", 40 + k)
                sides.append((params, F.AdamW(params, **HYPER, state_bits=bits, max_norm=0.3)))
        for _ in range(10):
            for s, (_, o) in zip(streams, sides):
                with torch.cuda.stream(s):
                    o.step()
        torch.cuda.synchronize()
        return sides
    here = torch.cuda.current_stream()
    for (p, o), (q, n) in zip(run([here, here]), run([torch.cuda.Stream(), torch.cuda.Stream()])):
        assert float(o.grad_norm) == float(n.grad_norm)
        for a, b in zip(p, q):
            assert torch.equal(a, b) and all(torch.equal(o.state[a][k].float(), n.state[b][k].float()) for k in o.state[a])


def test_a_step_is_a_change_in_place():
    w = torch.randn(8, device="cuda", requires_grad=True)
    y = (w * w).sum()
    w.grad = torch.ones(8, device="cuda")
    F.AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    w = torch.zeros(6, 4, device="cuda").t().requires_grad_()
    w.grad = torch.zeros(4, 6, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        F.AdamW([w]).step()
    table = torch.zeros(10, 4, device="cuda", requires_grad=True)
    table.grad = torch.sparse_coo_tensor(torch.tensor([[1, 3]]), torch.ones(2, 4), (10, 4)).cuda()
    for norm in (None, 1.0):
        with pytest.raises(ValueError, match="sparse"):
            F.AdamW([table], max_norm=norm).step()
    d = torch.zeros(4, device="cuda", dtype=torch.float64, requires_grad=True)
    d.grad = torch.zeros_like(d)
    with pytest.raises(ValueError, match="dtype"):
        F.AdamW([d]).step()
    p = torch.zeros(4, device="cuda", requires_grad=True)
    p.grad = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="float32"):
        F.AdamW([p], lr=torch.zeros(1, device="cuda", dtype=torch.float64)).step()
    o = F.AdamW([p])
    o.step()
    o.state[p]["exp_avg"] = torch.zeros(5, device="cuda")
    with pytest.raises(ValueError, match="shape"):
        o.step()
    empty = torch.zeros(0, 3, device="cuda", requires_grad=True)
    empty.grad = torch.zeros_like(empty)
    F.AdamW([empty], max_norm=1.0).step()


@pytest.mark.parametrize("bits", [32, 8])
def test_the_least_eps(bits):
    """2^-126: a weight whose gradient has always been 0 only decays."""
    p = torch.randn(600, generator=gen(70), device="cuda").requires_grad_()
    p.grad = torch.randn(600, generator=gen(71), device="cuda")
    p.grad[:256] = 0
    before = p.detach()[:256].clone()
    o = F.AdamW([p], lr=0.01, weight_decay=0.0, eps=2.0 ** -126, state_bits=bits)
    o.step()
    assert torch.equal(p.detach()[:256], before) and p.detach().isfinite().all()
    o.param_groups[0]["eps"] = 1e-40
    with pytest.raises(ValueError, match="eps"):
        o.step()


def test_offsets_beyond_32_bits():
    """A tensor of more than 2^31 elements (26 GB with its states): its ends are what small tensors' are."""
    n = 2 ** 31 + 2 ** 12 + 5
    g = gen(18)
    p = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    p.grad = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    at = [slice(0, 4096), slice(n - 4101, n)]
    parts = []
    for s in at:
        k = s.stop - s.start
        p[s] = torch.randn(k, generator=g, device="cuda")
        p.grad[s] = torch.randn(k, generator=g, device="cuda")
        q = p[s].clone().requires_grad_()
        q.grad = p.grad[s].clone()
        parts.append(q)
    p.requires_grad_()
    kw = dict(lr=0.1, master_weights=False, max_norm=1.0)
    o, small = F.AdamW([p], **kw), F.AdamW(parts, **kw)
    o.step(), small.step()
    assert abs(float(o.grad_norm) - float(small.grad_norm)) <= 1e-6 * float(o.grad_norm)
    for s, q in zip(at, parts):
        assert float((p.detach()[s].float() - q.detach().float()).abs().max()) <= 2.0 ** -8 * 4.5
        assert float((o.state[p]["exp_avg"][s] - small.state[q]["exp_avg"]).abs().max()) <= 1e-6
    assert not p.detach()[2 ** 20:2 ** 30].any() and int(o.state[p]["step"]) == 1


def test_a_refused_step_changes_nothing():
    """Groups and types are launched one by one, but checked before the first of them: weights, states and counts stay what they are."""
    params = model([(300,), (4000,)], "fp32", 50) + model([(77,)], "bf16", 51) + model([(300,)], "fp32", 52)
    groups = [dict(params=params[:3]), dict(params=params[3:], lr=0.5)]
    good = dict(lr=0.5, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1, seed=0)
    for max_norm in (None, 1.0):
        o = F.AdamW(groups, **HYPER, max_norm=max_norm)
        o.step()
        keep = [p.detach().clone() for p in params] + [t.clone() for p in params for t in o.state[p].values()]

        def unchanged():
            torch.cuda.synchronize()
            now = [p.detach() for p in params] + [t for p in params for t in o.state[p].values()]
            return all(torch.equal(a, b) for a, b in zip(keep, now))
        for bad in (dict(lr=torch.zeros(1, device="cuda", dtype=torch.float64)), dict(lr=float("nan")), dict(lr="fast"), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)),
                    dict(betas=0.9), dict(eps=-1.0), dict(eps=float("inf")), dict(weight_decay=float("nan")), dict(seed=2 ** 64), dict(seed=-1),
                    dict(seed=0.5)):
            o.param_groups[1].update({**good, **bad})
            with pytest.raises((ValueError, TypeError)):
                o.step()
            assert unchanged(), bad
        o.param_groups[1].update(good)
        del o.param_groups[1]["betas"]
        with pytest.raises(ValueError, match="betas"):
            o.step()
        o.param_groups[1].update(good)
        F.reorder_states(torch.zeros(1, 2, 3, device="cuda"), torch.tensor([[0, 5]], device="cuda"))      # a report that is still to be heard
        torch.cuda.synchronize()
        with pytest.raises(BlstmError):
            o.step()
        assert unchanged()
        o.step()
        assert not unchanged() and [int(o.state[p]["step"]) for p in params] == [2] * 4


def test_parameters_that_share_memory_are_refused():
    """All tensors of a launch are worked on at a time.  Neighbours in one buffer, and parameters without a gradient, are fine."""
    flat = torch.zeros(100, device="cuda")
    a, b, c = (flat[s].detach().requires_grad_() for s in (slice(0, 40), slice(40, 80), slice(79, 100)))
    o = F.AdamW([a, c, b])
    a.grad, b.grad = torch.ones(40, device="cuda"), torch.ones(40, device="cuda")
    o.step()
    before = flat.clone()
    c.grad = torch.ones(21, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        o.step()
    assert torch.equal(flat, before) and int(o.state[a]["step"]) == 1


def test_gradient_norm_is_added_up_in_64_bits():
    """Seven small squares behind a large one, each below half a step of 32 bits: summed in 32 bits the norm is 1.6 u too small, in 64 it has the
    one rounding to its own 32 bits."""
    small = (0.9 * 2.0 ** -25) ** 0.5
    for dtype, n in (("fp32", 4096), ("fp32", 70000), ("bf16", 4096)):
        g = torch.full((n,), small, device="cuda")
        g[::8] = 1
        p = torch.zeros(n, device="cuda", dtype=DT[dtype], requires_grad=True)
        p.grad = g.to(DT[dtype])
        total = np.sqrt((np64(p.grad) ** 2).sum())
        o = F.AdamW([p], max_norm=1e6)
        o.step()
        assert abs(float(o.grad_norm) - total) <= 1.001 * U * total


@pytest.mark.parametrize("dtype,master", [("fp32", False), ("bf16", True), ("fp16", False)])
@pytest.mark.parametrize("bits", [8, 32])
def test_more_chunks_than_blocks(dtype, master, bits):
    """Blocks that go on from chunk to chunk and from tensor to tensor, past chunks that are not whole and a tensor on another boundary, with
    copies of the next ones under way."""
    sizes = [700 * 8192 + 100, 3 * 8192 - 5, 8192, 50 * 8192, 300 * 8192, 17, 900 * 8192 + 8191, 40 * 8192]
    made = [0]

    def odd(p):
        made[0] += 1
        if made[0] != 4:
            return p
        flat = torch.zeros(p.numel() + 1, device="cuda", dtype=p.dtype)
        flat[1:] = p
        return flat[1:]
    params = model([(n,) for n in sizes], dtype, 60, odd)
    o = F.AdamW(params, **HYPER, state_bits=bits, master_weights=master, max_norm=100.0, seed=77)
    check_step(o, params, dtype)
    check_step(o, params, dtype)
