"""Operators around an LSTM language model that is trained deep and asked for whole sequences, as cases that can be timed and
compared: the root-mean-square norm between residual layers, the AdamW step over all of a model's tensors, and a step of
beam search with the reordering of the layers' states.

A case is one pass through one operator as a program makes it.  `run` is the operators' plain form in elementary torch
operations where `own` is false, and the framework's own operators where it is true."""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 256                    # elements that share a scale in 8-bit optimiser states


def _norm(name=None, **given):
    c = dict({"op": "norm", "dtype": "bf16", "steps": 1, "batch": 1, "width": 512, "residual": True, "train": True,
              "eight_bits": False, "batch_first": False}, **given)
    return c if name is None else dict(c, name=name)


def _adam(name=None, **given):
    c = dict({"op": "adamw", "dtype": "fp32", "vocab": 0, "width": 512, "layers": 2, "bits": 32, "master": False, "max_norm": 0.0,
              "decay": 0.01, "step": 100}, **given)
    return c if name is None else dict(c, name=name)


def _beam(name=None, **given):
    c = dict({"op": "beam", "dtype": "bf16", "batch": 1, "beams": 4, "width": 4, "vocab": 50000, "layers": 2, "hidden": 512, "written": 16,
              "finished": 0.0, "masked": 0.0, "penalty": 0.0}, **given)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # Generation: eight streams between two layers, one step each.  Latency of one launch.
        _norm("norm_step", batch=8, train=False),
        # A small fp32 training step at sizes that are multiples of nothing.
        _norm("norm_train_ragged", dtype="fp32", steps=33, batch=19, width=301),
        # Between the layers of the two-layer benchmark stack, one GPU's shard of eight.
        _norm("norm_train", steps=256, batch=512),
        # Scoring a corpus: what goes into a product of 8-bit operands, the mid-size benchmark shape.
        _norm("norm_eight_bits", dtype="fp16", steps=512, batch=256, width=1024, train=False, eight_bits=True),
        # A small layer in fp32 with its biases, odd sizes, no clipping: latency.
        _adam("adamw_layer", width=301, layers=1),
        # The two-layer benchmark stack with a vocabulary of words: bf16 weights with masters, gradients clipped.
        _adam("adamw_words", dtype="bf16", vocab=50000, master=True, max_norm=1.0),
        # The same sizes made odd, states in 8 bits.
        _adam("adamw_eight_bits_ragged", vocab=10007, width=301, bits=8, max_norm=0.5),
        # The largest: a vocabulary of sub-words, as little memory as there can be for it.
        _adam("adamw_eight_bits", dtype="bf16", vocab=131072, width=1024, bits=8),
        # One sentence, four hypotheses: latency.
        _beam("beam_sentence"),
        # Characters in fp32: short rows, many sentences, some of whose hypotheses have ended.
        _beam("beam_characters", dtype="fp32", batch=256, beams=10, width=10, vocab=205, hidden=301, written=100, finished=0.2, penalty=1.0),
        # Translation: words that cannot follow ruled out, long hypotheses favoured.
        _beam("beam_words", batch=16, beams=8, width=8, hidden=1024, written=40, finished=0.1, masked=0.5, penalty=0.6),
        # The largest: wide beams over sub-words.
        _beam("beam_subwords", dtype="fp16", batch=64, beams=16, width=16, vocab=131072, layers=4, hidden=1024, written=64, finished=0.1),
    ]


def _spread(rng, low, high):
    """A whole number between the two, its logarithm evenly spread."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    op = rng.choice(["norm", "adamw", "beam"])
    most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        if op == "norm":
            train = rng.random() < 0.6
            c = _norm(dtype=dtype, steps=_spread(rng, 1, 1024), batch=_spread(rng, 1, 512), width=_spread(rng, 32, 8192), residual=rng.random() < 0.7,
                      train=train, eight_bits=not train and rng.random() < 0.5, batch_first=rng.random() < 0.3)
        elif op == "adamw":
            c = _adam(dtype=dtype, vocab=rng.choice([0, _spread(rng, 64, 131072)]), width=_spread(rng, 32, 2048), layers=rng.choice([1, 2]),
                      bits=rng.choice([32, 8]), master=dtype != "fp32" and rng.random() < 0.6, max_norm=rng.choice([0.0, 0.5, 5.0]),
                      decay=rng.choice([0.0, 0.01, 0.1]), step=_spread(rng, 1, 100000))
        else:
            width, first = rng.randint(2, 24), rng.random() < 0.15
            c = _beam(dtype=dtype, batch=_spread(rng, 1, 256), beams=1 if first else width, width=width, vocab=_spread(rng, 64, 131072),
                      layers=rng.choice([1, 2, 4]), hidden=_spread(rng, 32, 2048), written=_spread(rng, 1, 256),
                      finished=0.0 if first else rng.choice([0.0, 0.2]), masked=rng.choice([0.0, 0.5]), penalty=rng.choice([0.0, 0.6, 1.0]))
        if work(c)["bytes"] <= most:
            return c


def _tensors(case):
    """The shapes of a model's parameters: the table, and each layer's two weights and two biases."""
    H = case["width"]
    return ([(case["vocab"], H)] if case["vocab"] else []) + [(4 * H, H), (4 * H, H), (4 * H,), (4 * H,)] * case["layers"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype or dt)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": case}
    if case["op"] == "norm":
        T, B, D = case["steps"], case["batch"], case["width"]
        # [T,B,D], laid out as a loader's or a layer's [B,T,D] where batch_first
        rows = (lambda std: normal(B, T, D, std=std).transpose(0, 1)) if case["batch_first"] else (lambda std: normal(T, B, D, std=std))
        s["x"] = rows(0.3)                    # what a layer gives: between -1 and 1
        s["residual"] = rows(1.5) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
        if case["train"]:
            for k in ("x", "residual", "weight"):
                if s[k] is not None:
                    s[k].requires_grad_()
            s["grads"] = [normal(T, B, D)] + ([normal(T, B, D)] if case["residual"] else [])
        return s
    if case["op"] == "adamw":
        # a model in the middle of its training; most words were not in this batch
        s["seed"], s["lr"], s["step"] = seed, 1e-3, case["step"] + seed % 7
        s["params"], s["state"] = [], []
        for shape in _tensors(case):
            n, word = math.prod(shape), len(shape) == 2 and shape[0] == case["vocab"]
            live = uniform(shape[0], 1) < 0.1 if word else None
            p = normal(*shape, std=0.05)
            p.requires_grad_()
            p.grad = normal(*shape, std=2e-3)
            if word:
                p.grad *= live
            st = {"step": torch.tensor(s["step"], device="cuda")}
            if case["bits"] == 32:
                st["exp_avg"] = normal(*shape, std=1e-3, dtype=torch.float32)
                st["exp_avg_sq"] = normal(*shape, std=2e-3, dtype=torch.float32).square_()
            else:
                blocks = -(-n // BLOCK)
                st["exp_avg"] = (normal(*shape, std=100.0, dtype=torch.float32).clamp_(-448, 448)).to(torch.float8_e4m3fn)
                st["exp_avg_scale"] = 5e-6 * (0.5 + uniform(blocks))
                st["exp_avg_sq_root"] = (normal(*shape, std=120.0, dtype=torch.float32).abs_().clamp_(0, 448)).to(torch.float8_e4m3fn)
                st["exp_avg_sq_root_scale"] = 1e-5 * (0.5 + uniform(blocks))
            if case["master"]:
                st["master"] = p.detach().float() * (1 + 2.0 ** -10 * (uniform(*shape) - 0.5))
            s["params"].append(p)
            s["state"].append(st)
        return s
    B, n, V, W = case["batch"], case["beams"], case["vocab"], case["width"]
    # predictions of a model that has learnt something: noise, and a few words of each well above it
    z = torch.randn(B, n, V, generator=g, device="cuda", dtype=torch.float32).mul_(2.0)
    z.scatter_add_(2, torch.randint(0, V, (B, n, 6), generator=g, device="cuda"), uniform(B, n, 6) * 9 + 4)
    if case["masked"] > 0:
        z.masked_fill_(torch.rand(B, n, V, generator=g, device="cuda") < case["masked"], -math.inf)
    s["end"] = V - 1
    s["logits"] = z.to(dt)
    s["scores"] = -(1 + uniform(B, n) * 8).sort(dim=1).values if n > 1 else torch.zeros(B, 1, device="cuda")
    written = case["written"]
    s["lengths"] = torch.full((B, n), written, device="cuda")
    s["finished"] = uniform(B, n) < case["finished"]
    s["lengths"] -= s["finished"] * torch.randint(0, written, (B, n), generator=g, device="cuda")
    s["states"] = [normal(case["layers"], B * n, case["hidden"], std=0.5), normal(case["layers"], B * n, case["hidden"])]
    s["history"] = torch.randint(0, V, (written, B * n), generator=g, device="cuda")
    return s


# ---------------------------------------------------------------- the framework's operators
def _own(s):
    import fastlstm_b200 as F
    case = s["case"]
    if case["op"] == "norm":
        if case["eight_bits"]:
            r = F.rms_norm_e4m3(s["x"], s["weight"], residual=s["residual"])
            return [r.values, r.scales] + ([r.sum] if case["residual"] else [])
        out = F.rms_norm(s["x"], s["weight"], residual=s["residual"])
        outs = list(out) if case["residual"] else [out]
        if not case["train"]:
            return outs
        inputs = [s["x"]] + ([s["residual"]] if case["residual"] else []) + [s["weight"]]
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, inputs, s["grads"]))
    if case["op"] == "adamw":
        if "optimizer" not in s:
            o = s["optimizer"] = F.AdamW(s["params"], lr=s["lr"], weight_decay=case["decay"], state_bits=case["bits"], master_weights=case["master"],
                                         max_norm=case["max_norm"] or None, seed=s["seed"])
            o.load_state_dict({"state": dict(enumerate(s["state"])), "param_groups": o.state_dict()["param_groups"]})
        s["optimizer"].step()
        return [[p.detach()] + [t for k, t in sorted(s["optimizer"].state[p].items()) if k != "step"] for p in s["params"]]
    r = F.beam_step(s["logits"], s["scores"], width=case["width"], end_token=s["end"], finished=s["finished"], lengths=s["lengths"],
                    length_penalty=case["penalty"])
    return [r.scores, r.parents, r.tokens, r.finished, r.lengths, *F.reorder_states([*s["states"], s["history"]], r.parents)]


# ---------------------------------------------------------------- their plain forms
def _plain_norm(s):
    case, x, r, w = s["case"], s["x"].detach(), s["residual"], s["weight"].detach()
    dt = x.dtype
    h = x if r is None else (x.float() + r.detach().float()).to(dt)
    f = h.float()
    i = torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)
    y = f * i * w.float()
    if case["eight_bits"]:
        scales = y.abs().amax(-1) / 448
        q = torch.where(scales[..., None] > 0, y / scales[..., None], 0.0).clamp(-448, 448).to(torch.float8_e4m3fn)
        return [q.contiguous(), scales.contiguous()] + ([h.contiguous()] if r is not None else [])
    res = [y.to(dt).contiguous()] + ([h.contiguous()] if r is not None else [])
    if not case["train"]:
        return res
    dy = s["grads"][0].float()
    n = dy * w.float()
    d = i * (n - f * (i * i * (n * f).mean(-1, keepdim=True)))
    if r is not None:
        d += s["grads"][1].float()
    d = d.to(dt).contiguous()
    dw = (dy * f * i).flatten(0, 1).sum(0, dtype=torch.float64).to(dt)
    return res + [d] + ([d] if r is not None else []) + [dw]


def _plain_words(n, seed, step, tensor, device):
    """n 32-bit words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) with the
    seed as the key and (block, step, tensor) as the counter, in whole numbers of 64 bits."""
    low = 0xFFFFFFFF
    block = torch.arange(-(-n // 4), device=device)
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, step & low), torch.full_like(block, tensor)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]


def _plain_blocks(x):
    """x flat in blocks, the last one filled up with zeros."""
    full = x.new_zeros(-(-x.numel() // BLOCK) * BLOCK)
    full[: x.numel()] = x.reshape(-1)
    return full.view(-1, BLOCK)


def _plain_encode(x, draw):
    """x [blocks, 256] as e4m3 numbers times a scale: cut off or rounded up with the probability of the part that is cut off, which 16
    random bits decide.  A number times 2^-120 has the e4m3 number's bits at the top of a 32-bit float's, its subnormal numbers too."""
    most = x.abs().amax(1, keepdim=True)
    fine = most > 2.0 ** -110
    bits = (x.abs() * torch.where(fine, 448 / most, 0.0) * 2.0 ** -120).view(torch.int32)
    code = ((bits + (draw.int() << 4)) >> 20).clamp(max=126)
    code = torch.where(x < 0, code + 128, code).to(torch.uint8)
    return code.view(torch.float8_e4m3fn), torch.where(fine, most / 448, 0.0)[:, 0]


def _plain_adamw(s):
    case, t = s["case"], s["step"]
    b1, b2, lr = 0.9, 0.999, s["lr"]
    clip = 1.0
    if case["max_norm"]:
        norm = torch.stack([p.grad.double().square().sum() for p in s["params"]]).sum().sqrt()
        clip = torch.clamp(case["max_norm"] / (norm + 1e-6), max=1.0).float()
    t = s["step"] = t + 1
    c1, c2 = lr / (1 - b1 ** t), 1 / math.sqrt(1 - b2 ** t)
    for k, (p, st) in enumerate(zip(s["params"], s["state"])):
        n, shape = p.numel(), p.shape
        grad = p.grad.float() * clip
        if case["bits"] == 32:
            m, v = st["exp_avg"], st["exp_avg_sq"]
            m.mul_(b1).add_(grad, alpha=1 - b1)
            v.mul_(b2).add_(grad * grad, alpha=1 - b2)
            u = v.sqrt()
        else:
            m = _plain_blocks(st["exp_avg"].float()) * st["exp_avg_scale"][:, None]
            v = (_plain_blocks(st["exp_avg_sq_root"].float()) * st["exp_avg_sq_root_scale"][:, None]).square()
            grad = _plain_blocks(grad)
            m = b1 * m + (1 - b1) * grad
            u = (b2 * v + (1 - b2) * (grad * grad)).sqrt()
            del v, grad
            words = _plain_blocks(_plain_words(n, s["seed"], t, k, p.device))
            q, st["exp_avg_scale"][:] = _plain_encode(m, words & 0xFFFF)
            st["exp_avg"].copy_(q.view(-1)[:n].view(shape))
            q, st["exp_avg_sq_root_scale"][:] = _plain_encode(u, words >> 16)
            least = torch.tensor(2.0 ** -9, device=p.device).to(torch.float8_e4m3fn)
            q = torch.where((u > 0) & (q.view(torch.uint8) == 0), least.view(torch.uint8), q.view(torch.uint8)).view(torch.float8_e4m3fn)
            st["exp_avg_sq_root"].copy_(q.view(-1)[:n].view(shape))
            del words, q
            m, u = m.view(-1)[:n].view(shape), u.view(-1)[:n].view(shape)
        x = st["master"] if case["master"] else p.detach().float()
        x = x * (1 - lr * case["decay"]) - c1 * m / (u * c2 + 1e-8)
        p.detach().copy_(x)
        if case["master"]:
            st["master"].copy_(x)
    return [[p.detach()] + [v for k, v in sorted(st.items()) if k != "step"] for p, st in zip(s["params"], s["state"])]


def _reordered(s, parents):
    B, n, W = s["case"]["batch"], s["case"]["beams"], s["case"]["width"]
    rows = (torch.arange(B, device=parents.device)[:, None] * n + parents).view(-1)
    return [t[:, rows] for t in (*s["states"], s["history"])]


def _plain_beam(s):
    case = s["case"]
    B, n, V, W = case["batch"], case["beams"], case["vocab"], case["width"]
    z = s["logits"].double()                # which hypothesis wins goes by differences that are small next to the scores
    high = z.amax(-1, keepdim=True)
    total = z - (high + torch.log(torch.exp(z - high).sum(-1, keepdim=True))) + s["scores"].double()[..., None]
    over = s["finished"][..., None]
    total = torch.where(over, -math.inf, total)
    total[..., s["end"]] = torch.where(s["finished"], s["scores"].double(), total[..., s["end"]])
    del z
    lengths = s["lengths"] + ~s["finished"]
    rank = total / (lengths.double() ** case["penalty"])[..., None]
    best = torch.sort(rank.view(B, n * V), dim=1, descending=True, stable=True).indices[:, :W]
    parents, tokens = best // V, best % V
    scores = total.view(B, n * V).gather(1, best).float()
    ended = s["finished"].gather(1, parents) | (tokens == s["end"])
    return [scores, parents, tokens, ended, lengths.gather(1, parents), *_reordered(s, parents)]


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "adamw": _plain_adamw, "beam": _plain_beam}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_norm(s):
    case, x, r, w = s["case"], s["x"].detach(), s["residual"], s["weight"].detach().double()
    h = x.double() if r is None else (x.double() + r.detach().double()).to(x.dtype).double()
    root = (h.square().sum(-1, keepdim=True) / case["width"] + 1e-6).sqrt()
    unit = h / root
    y = unit * w
    more = [] if r is None else [h]
    if case["eight_bits"]:
        scales = y.abs().amax(-1, keepdim=True) / 448
        v = torch.where(scales > 0, y / scales, 0.0).abs()
        step = torch.exp2(torch.floor(torch.log2(v.clamp_min(2.0 ** -6))) - 3)       # between e4m3 numbers, subnormal ones too
        return [torch.round(v / step) * step * torch.sign(y), scales[..., 0], *more]
    if not case["train"]:
        return [y, *more]
    dy = s["grads"][0].double()
    through = dy * w
    d = (through - unit * (through * unit).sum(-1, keepdim=True) / case["width"]) / root
    if r is not None:
        d = d + s["grads"][1].double()
    return [y, *more, d] + ([d] if r is not None else []) + [(dy * unit).sum((0, 1))]


def _exact_words(n, seed, step, tensor, device):
    """Philox again, each 32-bit product from 16-bit halves."""
    half, low = 0xFFFF, 0xFFFFFFFF

    def high_low(x, m):
        m1, m0, x1, x0 = m >> 16, m & half, x >> 16, x & half
        mid = m1 * x0 + ((m0 * x0) >> 16)
        side = m0 * x1 + (mid & half)
        return m1 * x1 + (mid >> 16) + (side >> 16), ((side & half) << 16) | (m0 * x0 & half)

    v = [torch.arange((n + 3) // 4, device=device)]
    v = [v[0] % 2 ** 32, v[0] // 2 ** 32, torch.full_like(v[0], step), torch.full_like(v[0], tensor)]
    for r in range(10):
        (h0, l0), (h1, l1) = high_low(v[0], 0xD2511F53), high_low(v[2], 0xCD9E8D57)
        key = [(seed % 2 ** 32 + r * 0x9E3779B9) & low, (seed // 2 ** 32 + r * 0xBB67AE85) & low]
        v = [h1 ^ v[1] ^ key[0], l1, h0 ^ v[3] ^ key[1], l0]
    return torch.stack(v, 1).flatten()[:n]


def _exact_encode(x, draws):
    """(e4m3 numbers as 64-bit ones, scales) of x, flat: a number between two of them goes up where what it is above the lower one, in
    65536ths of their distance, and the draw make a whole."""
    n = x.numel()
    blocks = torch.zeros(-(-n // BLOCK), BLOCK, device=x.device, dtype=x.dtype)
    blocks.view(-1)[:n] = x.abs()
    most = blocks.amax(1)
    scales = torch.where(most > 2.0 ** -110, most / 448, 0.0)
    each = scales.repeat_interleave(BLOCK)[:n]
    v = torch.where(each > 0, x.abs() / each, 0.0)
    step = torch.exp2(torch.floor(torch.log2(v.clamp_min(2.0 ** -6))) - 3)
    v = torch.floor(v / step + draws.double() / 65536) * step
    return v.clamp_max(448) * torch.sign(x), scales


def _exact_adamw(s):
    case, t = s["case"], s["step"] + 1
    grads = [p.grad.double() for p in s["params"]]
    factor = 1.0
    if case["max_norm"]:
        factor = min(1.0, case["max_norm"] / (math.sqrt(sum(float((g * g).sum()) for g in grads)) + 1e-6))
    res = []
    for k, (p, st, g) in enumerate(zip(s["params"], s["state"], grads)):
        g, new = g.flatten() * factor, {}
        if case["bits"] == 32:
            m, v = st["exp_avg"].double().flatten(), st["exp_avg_sq"].double().flatten()
        else:
            spread = lambda name: st[name + "_scale"].double().repeat_interleave(BLOCK)[: p.numel()] * st[name].double().flatten()
            m, v = spread("exp_avg"), spread("exp_avg_sq_root").square()
        m, v = m + 0.1 * (g - m), 0.999 * v + 0.001 * g * g
        if case["bits"] == 32:
            new["exp_avg"], new["exp_avg_sq"] = m.view(p.shape), v.view(p.shape)
        else:
            words = _exact_words(p.numel(), s["seed"], t, k, p.device)
            q, new["exp_avg_scale"] = _exact_encode(m, words % 65536)
            new["exp_avg"] = q.view(p.shape)
            q, new["exp_avg_sq_root_scale"] = _exact_encode(v.sqrt(), words // 65536)
            new["exp_avg_sq_root"] = torch.where((v > 0) & (q == 0), 2.0 ** -9, q).view(p.shape)
            del words, q
        x = (st["master"] if case["master"] else p.detach()).double().flatten()
        x = x - s["lr"] * (case["decay"] * x + m / (1 - 0.9 ** t) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8))
        if case["master"]:
            new["master"] = x.view(p.shape)
        res.append([x.view(p.shape)] + [new[name] for name in sorted(new)])
    return res


def _exact_beam(s):
    case = s["case"]
    B, n, V, W = case["batch"], case["beams"], case["vocab"], case["width"]
    scores, found = torch.empty(B, W, device="cuda", dtype=torch.float64), torch.empty(B, W, 2, device="cuda", dtype=torch.int64)
    lengths = torch.where(s["finished"], s["lengths"], s["lengths"] + 1)
    for b in range(B):
        total = s["scores"][b, :, None].double() + torch.log_softmax(s["logits"][b].double(), -1)
        over = s["finished"][b].nonzero()[:, 0]
        total[over] = -math.inf
        total[over, s["end"]] = s["scores"][b, over].double()
        rank = total * lengths[b, :, None].double().pow(-case["penalty"])
        # the best of each hypothesis, then of those
        first = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, : min(W, V)]
        flat = (first + torch.arange(n, device="cuda")[:, None] * V).flatten()
        flat = flat[torch.sort(rank.flatten()[flat], descending=True, stable=True).indices[:W]]
        scores[b], found[b] = total.flatten()[flat], torch.stack([flat // V, flat % V], 1)
    parents, tokens = found.unbind(-1)
    moved = [t.double() if t.is_floating_point() else t for t in _reordered(s, parents)]
    return [scores, parents, tokens, s["finished"].gather(1, parents) | (tokens == s["end"]), lengths.gather(1, parents), *moved]


def exact(case, seed):
    return {"norm": _exact_norm, "adamw": _exact_adamw, "beam": _exact_beam}[case["op"]](prepare(case, seed))


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Bytes: each input read once and each output written once (of logits the rows of hypotheses that go on; of states the rows that
    winners go on from).  Flops: the additions, products and roots of the formulas; a random word counts none."""
    e = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, D, r = case["steps"] * case["batch"] * case["width"], case["width"], case["residual"]
        b = e * (n * (3 if r else 1) + D) + (n + 4 * n // D if case["eight_bits"] else e * n)
        f = n * (6 if case["eight_bits"] else 5)
        if case["train"]:
            b += e * (n * (3 if r else 2) + D)      # (dx and the residual's gradient are one tensor; the sum is at hand from forward)
            f += 10 * n
        return {"bytes": b, "flops": f}
    if case["op"] == "adamw":
        n = sum(math.prod(t) for t in _tensors(case))
        state = 8 if case["bits"] == 32 else 2 + 8 / BLOCK
        return {"bytes": n * (e + 2 * state + (8 + e if case["master"] else 2 * e)), "flops": n * (15 if case["bits"] == 32 else 23)}
    B, W, H, L = case["batch"], case["width"], case["hidden"], case["layers"]
    live = B * case["beams"] * (1 - case["finished"])
    rows = B * W * (2 * L * H * e + 8 * case["written"])
    return {"bytes": live * case["vocab"] * e + B * case["beams"] * 13 + B * W * 29 + 2 * rows, "flops": 4 * live * case["vocab"]}
