"""AdamW without a GPU: the oracle against torch in 64 bits, the arguments and states that are refused, and what the C entry points
refuse before anything runs on a device."""
import copy
import ctypes

import numpy as np
import pytest
import torch

import fastlstm_b200 as F
from fastlstm_b200 import _lib
from oracle import adamw_oracle as A

PTR = 0x10000     # (never touched: every check comes before the first CUDA call)


def test_oracle_matches_torch():
    g = torch.Generator().manual_seed(2)
    p = torch.randn(50, generator=g, dtype=torch.float64).requires_grad_()
    o = torch.optim.AdamW([p], lr=0.03, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.2)
    q, m, v = p.detach().numpy().copy(), np.zeros(50), np.zeros(50)
    for t in range(1, 6):
        p.grad = torch.randn(50, generator=g, dtype=torch.float64)
        o.step()
        m, v, _ = A.moments(m, v, p.grad.numpy(), 0.8, 0.95)
        q = A.update(q, m, v, t, 0.03, 0.8, 0.95, 1e-6, 0.2)
        np.testing.assert_allclose(p.detach().numpy(), q, rtol=1e-12)


def test_oracle_positions_are_those_of_e4m3():
    x = np.abs(np.random.RandomState(1).randn(4000)) * 10 ** np.random.RandomState(2).uniform(-6, 0, 4000)
    s = A.scales_of(x)
    w, step = A.position(x, s, np.zeros(x.size))
    down, up = np.floor(w + 1e-9) * step, np.ceil(w - 1e-9) * step     # (448 itself is one, give or take the division)
    for v in (down, up):
        assert (v == torch.tensor(v).to(torch.float8_e4m3fn).double().numpy()).all()
    exact = x / A.each(s, x.size)
    assert (down <= exact + 1e-9).all() and (up >= exact - 1e-9).all() and (up - down <= step).all()


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(betas=(0.9,)), dict(eps=-1e-8),
                                 dict(weight_decay=-1.0), dict(weight_decay=float("inf")), dict(state_bits=16), dict(max_norm=0.0), dict(max_norm=-1.0),
                                 dict(max_norm=float("nan")), dict(seed=-1), dict(seed=2 ** 64), dict(seed=0.5), dict(lr=torch.ones(2)),
                                 dict(lr=torch.ones(1, dtype=torch.long))])
def test_arguments_refused(bad):
    with pytest.raises(ValueError):
        F.AdamW([torch.zeros(3, requires_grad=True)], **bad)
    if not set(bad) & {"state_bits", "max_norm", "seed"}:
        with pytest.raises(ValueError):
            F.AdamW([dict(params=[torch.zeros(3, requires_grad=True)], **bad)])


@pytest.mark.parametrize("bad", [dict(seed=-1), dict(seed=2 ** 64), dict(seed=0.5), dict(lr=1e39), dict(lr=-1.0), dict(eps=1e39), dict(weight_decay=1e39),
                                 dict(betas=(0.9, 1.0)), dict(betas=(0.9,))])
def test_groups_are_refused_when_they_come(bad):
    """A group's own values, and those of a loaded state: what is there stays."""
    a, b = torch.zeros(3, requires_grad=True), torch.zeros(4, requires_grad=True)
    o = F.AdamW([a], lr=0.5, seed=3)
    with pytest.raises(ValueError):
        o.add_param_group(dict(params=[b], **bad))
    assert len(o.param_groups) == 1
    saved = o.state_dict()
    state = {"step": 3, "exp_avg": torch.zeros(3), "exp_avg_sq": torch.zeros(3)}
    with pytest.raises(ValueError):
        o.load_state_dict({"state": {0: state}, "param_groups": [{**saved["param_groups"][0], **bad}]})
    assert not o.state and o.param_groups[0]["lr"] == 0.5 and o.param_groups[0]["seed"] == 3
    o.add_param_group(dict(params=[b], seed=4.0))
    assert [repr(g["seed"]) for g in o.param_groups] == ["3", "4"]
    with pytest.raises(ValueError, match="max_norm"):
        F.AdamW([a], max_norm=1e-50)


def test_eps_whose_reciprocal_is_infinite_is_refused():
    """Below 2^-126 a weight without a gradient would move by 0 times infinity."""
    p = torch.zeros(3, requires_grad=True)
    for eps in (1e-40, 1e-300, 2.0 ** -126 * 0.999):
        with pytest.raises(ValueError, match="eps"):
            F.AdamW([p], eps=eps)
        d, _ = _desc(eps=eps)
        assert _lib.load().blstm_adamw(d, None) == 1
    F.AdamW([p], eps=2.0 ** -126)
    F.AdamW([p], eps=0)


def test_states_of_coupled_weight_decay_are_refused():
    """torch's Adam adds weight decay to the gradient: its state does not go on here, unless there is none."""
    p = torch.zeros(3, requires_grad=True)
    o = F.AdamW([p], lr=0.5)
    with pytest.raises(ValueError, match="decay"):
        o.load_state_dict(torch.optim.Adam([p], weight_decay=0.1).state_dict())
    assert o.param_groups[0]["lr"] == 0.5
    o.load_state_dict(torch.optim.Adam([p], lr=0.25).state_dict())
    o.load_state_dict(torch.optim.AdamW([p], lr=0.125, weight_decay=0.1).state_dict())
    assert o.param_groups[0]["lr"] == 0.125 and o.param_groups[0]["weight_decay"] == 0.1


def test_load_hooks_see_and_change_the_whole_state():
    """What a hook in front returns is what is checked and loaded; a hook behind sees the final state."""
    p = torch.zeros(5, requires_grad=True)
    o = F.AdamW([p])
    groups = o.state_dict()["param_groups"]
    old = {"m": torch.full((5,), 7.0), "exp_avg_sq": torch.ones(5), "step": 2}
    seen = []

    def convert(optimizer, d):
        assert optimizer is o and list(d["state"]) == [0]
        return {**d, "state": {k: {"exp_avg": s["m"], "exp_avg_sq": s["exp_avg_sq"], "step": 9} for k, s in d["state"].items()}}
    first = o.register_load_state_dict_pre_hook(convert)
    o.register_load_state_dict_pre_hook(lambda optimizer, d: seen.append(d["state"][0]["step"]))
    o.register_load_state_dict_post_hook(lambda optimizer: seen.append((int(o.state[p]["step"]), float(o.state[p]["exp_avg"][0]))))
    given = {"state": {0: old}, "param_groups": groups}
    o.load_state_dict(given)
    assert seen == [9, (9, 7.0)] and list(given["state"][0]) == ["m", "exp_avg_sq", "step"]
    first.remove()
    with pytest.raises(ValueError, match="exp_avg"):
        o.load_state_dict(given)
    assert len(seen) == 3 and int(o.state[p]["step"]) == 9       # (refused: no hook behind)
    o.load_state_dict(o.state_dict())                            # (hooks are still there)
    assert seen[3:] == [9, (9, 7.0)]


def test_cpu_parameters_are_refused_and_none_is_fine():
    p = torch.zeros(3, requires_grad=True)
    o = F.AdamW([p])
    assert o.step() is None and o.step(lambda: 7) == 7 and not o.state and o.grad_norm is None
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="CUDA"):
        o.step()


def test_states_are_checked_when_they_are_loaded():
    p = torch.zeros(300, requires_grad=True)
    state = {"step": 3, "exp_avg": torch.zeros(300), "exp_avg_sq": torch.zeros(300)}
    o = F.AdamW([p])
    groups = o.state_dict()["param_groups"]
    o.load_state_dict({"state": {0: state}, "param_groups": groups})
    assert int(o.state[p]["step"]) == 3 and o.state[p]["step"].dtype == torch.int64
    assert list(o.state_dict()["state"][0]) == ["exp_avg", "exp_avg_sq", "step"]
    for bad in ({**state, "exp_avg": torch.zeros(301)}, {k: v for k, v in state.items() if k != "exp_avg_sq"}, {**state, "step": torch.zeros(2)},
                {**state, "exp_avg": torch.zeros(300).to(torch.float8_e4m3fn)}):
        with pytest.raises(ValueError):
            o.load_state_dict({"state": {0: bad}, "param_groups": groups})
    with pytest.raises(ValueError):
        o.load_state_dict({"state": {1: state}, "param_groups": groups})
    assert int(o.state[p]["step"]) == 3                     # (what was there stays)
    eight = F.AdamW([p], state_bits=8)
    with pytest.raises(ValueError, match="state_bits"):
        eight.load_state_dict({"state": {0: state}, "param_groups": groups})
    theirs = torch.optim.AdamW([p], lr=0.5, weight_decay=0.3).state_dict()
    o.load_state_dict(theirs)
    assert o.param_groups[0]["lr"] == 0.5 and o.param_groups[0]["weight_decay"] == 0.3 and o.param_groups[0]["seed"] == 0 and not o.state
    theirs["param_groups"][0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        o.load_state_dict(theirs)
    half = torch.full((300,), 0.1, dtype=torch.bfloat16, requires_grad=True)
    h = F.AdamW([half])
    h.load_state_dict({"state": {0: state}, "param_groups": groups})     # (of torch's AdamW: no masters)
    assert torch.equal(h.state[half]["master"], half.detach().float())


def test_copies_and_groups():
    a, b = torch.zeros(3, requires_grad=True), torch.zeros(4, requires_grad=True)
    o = F.AdamW([dict(params=[a], lr=0.5), dict(params=[b], weight_decay=0.0)], lr=0.1, state_bits=8, max_norm=2.0, seed=2 ** 64 - 1)
    assert [g["lr"] for g in o.param_groups] == [0.5, 0.1] and [g["weight_decay"] for g in o.param_groups] == [0.01, 0.0]
    c = copy.deepcopy(o)
    assert c.state_bits == 8 and c.max_norm == 2.0 and c.master_weights and c.param_groups[0]["seed"] == 2 ** 64 - 1
    torch.optim.lr_scheduler.StepLR(o, 1)


def test_hooks_and_profilers_are_heard():
    p = torch.zeros(3, requires_grad=True)
    o = F.AdamW([p])
    seen = []
    handles = [o.register_step_pre_hook(lambda *a: seen.append("before")), o.register_step_post_hook(lambda *a: seen.append("behind"))]
    assert o.step(lambda: seen.append("closure") or 3) == 3 and seen == ["before", "closure", "behind"]
    for h in handles:
        h.remove()
    assert o.step(lambda: 4) == 4 and len(seen) == 3
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        o.step()
    assert any("AdamW.step" in e.key for e in prof.key_averages())
    scheduler = torch.optim.lr_scheduler.StepLR(o, 1, gamma=0.5)
    o.step()
    scheduler.step()
    assert o.param_groups[0]["lr"] == 5e-4


def test_descriptor_layouts_match_the_library():
    assert [ctypes.sizeof(c) for c in (_lib.AdamWItem, _lib.AdamWDesc, _lib.GradItem, _lib.GradNormDesc)] == [80, 96, 24, 48]


def _desc(items=1, bits=32, master=False, **given):
    item = (_lib.AdamWItem * max(items, 1))()
    for i in item:
        for f in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step"):
            setattr(i, f, PTR)
        i.master, i.n = PTR if master else None, 5
    d = _lib.AdamWDesc(dtype=_lib.BF16, bits=bits, items=items, item=item, lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, ticket=PTR)
    for k, v in given.items():
        setattr(d, k, v)
    return d, item


@pytest.mark.parametrize("change", [dict(dtype=3), dict(bits=16), dict(items=-1), dict(item=None), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0),
                                    dict(lr=float("nan")), dict(weight_decay=float("inf")), dict(ticket=None), dict(ticket=PTR + 2), dict(lr_at=PTR + 1),
                                    dict(factor=PTR + 2), dict(dtype=_lib.F32)])
def test_descriptors_refused(change):
    d, item = _desc(master="dtype" in change, **change)
    assert _lib.load().blstm_adamw(d, None) == 1


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("change", [dict(n=0), dict(n=-3), dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(step=None),
                                    dict(param=PTR + 1), dict(grad=PTR + 1), dict(step=PTR + 4), dict(master=PTR), dict(exp_avg_scale=PTR + 2)])
def test_items_refused(bits, change):
    d, item = _desc(items=2, bits=bits)
    for k, v in change.items():
        setattr(item[1], k, v)
    assert _lib.load().blstm_adamw(d, None) == 1
    if bits == 8:
        d, item = _desc(items=2, bits=bits)
        item[0].exp_avg_sq_scale = None
        assert _lib.load().blstm_adamw(d, None) == 1
    else:
        d, item = _desc(items=2, bits=bits)
        item[0].exp_avg = PTR + 2
        assert _lib.load().blstm_adamw(d, None) == 1


def test_gradient_norm_refused():
    lib = _lib.load()
    need = lib.blstm_grad_norm_workspace(1)
    assert need > 0 and need % 256 == 0 and lib.blstm_grad_norm_workspace(1000) > need

    def call(**given):
        item = (_lib.GradItem * 1)(_lib.GradItem(PTR, 5, _lib.BF16, 0))
        for k in ("grad", "n", "dtype"):
            if k in given:
                setattr(item[0], k, given.pop(k))
        d = _lib.GradNormDesc(**{**dict(item=item, items=1, max_norm=1.0, out=PTR, ticket=PTR, workspace=PTR, workspace_bytes=need), **given})
        return lib.blstm_grad_norm(d, None)
    for bad in (dict(grad=None), dict(grad=PTR + 1), dict(n=0), dict(dtype=9), dict(items=-1), dict(item=None), dict(max_norm=0.0), dict(max_norm=float("nan")),
                dict(out=None), dict(out=PTR + 2), dict(ticket=None)):
        assert call(**bad) == 1, bad
    for bad in (dict(workspace=None), dict(workspace=PTR + 16), dict(workspace_bytes=need - 1)):
        assert call(**bad) == 3
    assert call(items=0) == 0
    empty, _ = _desc(items=0)
    assert lib.blstm_adamw(empty, None) == 0
