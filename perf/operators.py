"""The operators around an LSTM language model as cases that can be timed and compared: the lookup of its tokens'
embeddings with the gradient of the table, dropout between its layers with a mask that is never stored, and the log
probabilities of given tokens with the entropy of the prediction and the likeliest alternatives.

A case is one pass through one operator as a program makes it: a call without gradients (serving, scoring), or forward
and backward (training).  `run` is the operators' plain form in elementary torch operations where `own` is false, and the
framework's own operators where it is true."""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def _embed(name=None, **given):
    c = dict({"op": "embedding", "dtype": "bf16", "steps": 1, "batch": 1, "width": 512, "vocab": 10000, "scale": 1.0,
              "train": True, "padded": 0.0, "batch_first": False}, **given)
    return c if name is None else dict(c, name=name)


def _drop(name=None, **given):
    c = dict({"op": "dropout", "dtype": "bf16", "steps": 1, "batch": 1, "width": 512, "p": 0.5, "shared": False,
              "batch_first": False}, **given)
    return c if name is None else dict(c, name=name)


def _score(name=None, **given):
    c = dict({"op": "log_probs", "dtype": "bf16", "steps": 1, "batch": 1, "vocab": 50000, "top": 0, "temperature": 1.0,
              "train": True, "ignored": 0.0, "masked": 0.0}, **given)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # Generation: the last token of eight streams becomes the next step's input.  Latency of one launch.
        _embed("embed_step", train=False, batch=8),
        # A small fp32 training step at sizes that are multiples of nothing; the table is larger than the batch.
        _embed("embed_train_ragged", dtype="fp32", steps=33, batch=19, width=301, vocab=10007, scale=301 ** 0.5),
        # An ordinary training step: ragged sequences padded with a token that gets no gradient, the loader's [B,T] tokens
        # read as [T,B].
        _embed("embed_train", steps=256, batch=64, vocab=50000, padded=0.25, batch_first=True),
        # The largest: a vocabulary of sub-words, T and B of the mid-size benchmark shape.
        _embed("embed_train_large", dtype="fp16", steps=512, batch=256, width=1024, vocab=131072, scale=32.0),
        # Between two small fp32 layers; latency.
        _drop("dropout_train_ragged", dtype="fp32", steps=33, batch=19, width=301),
        # Between the layers of the two-layer benchmark stack, one GPU's shard of eight.
        _drop("dropout_train", steps=256, batch=512, p=0.2),
        # One mask for all steps of a sequence (variational dropout), the mid-size benchmark shape.
        _drop("dropout_train_shared", dtype="fp16", steps=512, batch=256, width=1024, p=0.3, shared=True),
        # Generation: four streams, the log probability of the token taken and five alternatives.
        _score("score_step", train=False, batch=4, top=5),
        # Constrained generation of a larger batch: half of the vocabulary ruled out, as many alternatives as servers report.
        _score("score_masked", train=False, dtype="fp16", batch=64, vocab=131072, top=20, masked=0.5, temperature=0.7),
        # A character model in fp32: many rows, short ones.
        _score("train_characters", dtype="fp32", steps=512, batch=32, vocab=205),
        # A word model in fp32, odd sizes, some padding, gradients through the alternatives too.
        _score("train_words_ragged", dtype="fp32", steps=33, batch=19, vocab=10007, top=3, ignored=0.2, temperature=0.8),
        # The training step of a sub-word model: 8192 predictions.
        _score("train_subwords", steps=128, batch=64, vocab=50000, ignored=0.1),
    ]


def _spread(rng, low, high):
    """A whole number between the two, its logarithm evenly spread."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    op = rng.choice(["embedding", "dropout", "log_probs"])
    most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        rows = {"dtype": dtype, "steps": _spread(rng, 1, 1024), "batch": _spread(rng, 1, 512)}
        if op == "embedding":
            c = _embed(**rows, width=_spread(rng, 32, 2048), vocab=_spread(rng, 64, 131072), scale=rng.choice([1.0, 11.3, 32.0]),
                       train=rng.random() < 0.75, padded=rng.choice([0.0, 0.25]), batch_first=rng.random() < 0.5)
        elif op == "dropout":
            c = _drop(**rows, width=_spread(rng, 32, 2048), p=rng.choice([0.1, 0.2, 0.3, 0.5, 0.65]),
                      shared=rng.random() < 0.3, batch_first=rng.random() < 0.3)
        else:
            c = _score(**rows, vocab=_spread(rng, 64, 131072), top=rng.choice([0, 0, 1, 5, 20]), train=rng.random() < 0.6,
                       temperature=rng.choice([1.0, 0.7, 1.3]), ignored=rng.choice([0.0, 0.2]),
                       masked=rng.choice([0.0, 0.0, 0.5]))
        if work(c)["bytes"] <= most and c["steps"] * c["batch"] * c.get("vocab", 1) <= 2 ** 35:
            return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, T, B = TYPES[case["dtype"]], case["steps"], case["batch"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dt)

    def rows(*shape):
        # [T,B,...], laid out as the loader's or the layer's [B,T,...] where batch_first
        return normal(B, T, *shape).transpose(0, 1) if case["batch_first"] else normal(T, B, *shape)

    def words(n):
        # frequent words first, as vocabularies are numbered: the probability falls with the number
        u = torch.rand(B, T, generator=g, device="cuda", dtype=torch.float64)
        return ((n + 1.0) ** u).long().sub_(1).clamp_(0, n - 1)

    if case["op"] == "embedding":
        tokens = words(case["vocab"])
        if case["padded"] > 0:       # sequences of different lengths, token 0 behind their ends
            length = T - (2 * case["padded"] * T * torch.rand(B, generator=g, device="cuda")).long()
            tokens = torch.where(torch.arange(T, device="cuda")[None] < length[:, None], tokens, 0)
        tokens = tokens.t() if case["batch_first"] else tokens.t().contiguous()
        s = {"case": case, "tokens": tokens, "weight": normal(case["vocab"], case["width"], std=1 / case["scale"])}
        if case["train"]:
            s["weight"].requires_grad_()
            s["grad"] = normal(T, B, case["width"])
        return s
    if case["op"] == "dropout":
        # the seed of the training step, the layer as the offset
        s = {"case": case, "x": rows(case["width"]), "grad": normal(T, B, case["width"]),
             "seed": (seed * 0x9E3779B97F4A7C15 + 12345) % 2 ** 63, "offset": 1 + seed % 3}
        s["x"].requires_grad_()
        return s
    # logits of a model that has learnt something: noise, and most of the targets well above it
    V = case["vocab"]
    tokens = words(V).t().contiguous()
    logits = torch.randn(T, B, V, generator=g, device="cuda", dtype=torch.float32).mul_(2.5)
    sure = torch.rand(T, B, 1, generator=g, device="cuda") * 14 - 3
    logits.scatter_add_(2, tokens[..., None], sure)
    if case["masked"] > 0:           # words that a grammar rules out, never the token itself
        out = torch.rand(T, B, V, generator=g, device="cuda") < case["masked"]
        out.scatter_(2, tokens[..., None], False)
        logits.masked_fill_(out, -math.inf)
    logits = logits.to(dt)
    if case["ignored"] > 0:
        tokens[torch.rand(T, B, generator=g, device="cuda") < case["ignored"]] = -100
    s = {"case": case, "logits": logits, "tokens": tokens}
    if case["train"]:
        logits.requires_grad_()
        # a weighted likelihood, a little entropy, and the alternatives' share where there are any (16-bit users scale losses)
        s["grads"] = [-0.5 - torch.rand(T, B, generator=g, device="cuda"), 0.05 * torch.randn(T, B, generator=g, device="cuda")]
        if case["top"]:
            s["grads"].append(0.1 * torch.randn(T, B, case["top"], generator=g, device="cuda"))
    return s


# ---------------------------------------------------------------- the framework's operators
def _own(s):
    import fastlstm_b200 as F
    case = s["case"]
    if case["op"] == "embedding":
        out = F.embedding(s["tokens"], s["weight"], scale=case["scale"], padding_idx=0 if case["padded"] > 0 else None)
        if not case["train"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, s["weight"], s["grad"])]
    if case["op"] == "dropout":
        out = F.dropout(s["x"], case["p"], s["seed"], offset=s["offset"], shared_dim=0 if case["shared"] else None)
        return [out.detach(), *torch.autograd.grad(out, s["x"], s["grad"])]
    r = F.token_log_probs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"])
    outs = [r.log_probs, r.entropy] + ([r.top_log_probs] if case["top"] else [])
    res = [t.detach() for t in outs] + ([r.top_tokens] if case["top"] else [])
    if case["train"]:
        res += torch.autograd.grad(outs, s["logits"], s["grads"])
    return res


# ---------------------------------------------------------------- their plain forms
def _plain_embedding(s):
    case, tokens, weight = s["case"], s["tokens"], s["weight"].detach()
    out = (weight[tokens].float() * case["scale"]).to(weight.dtype)
    if not case["train"]:
        return [out]
    rows = s["grad"].float().reshape(-1, case["width"])
    dW = torch.zeros(weight.shape, device=weight.device).index_add_(0, tokens.reshape(-1), rows)
    dW *= case["scale"]
    if case["padded"] > 0:
        dW[0] = 0
    return [out, dW.to(weight.dtype)]


def _plain_words(n, seed, offset, device):
    """n 32-bit words of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) with the
    seed as the key and (block, offset) as the counter, in whole numbers of 64 bits."""
    low = 0xFFFFFFFF
    block = torch.arange(-(-n // 4), device=device)
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]


def _plain_dropout(s):
    case, x, grad = s["case"], s["x"].detach(), s["grad"]
    shape = x.shape[1:] if case["shared"] else x.shape
    kept = (_plain_words(math.prod(shape), s["seed"], s["offset"], x.device) >= round(case["p"] * 2 ** 32)).view(shape)
    scale = 1 / (1 - case["p"])
    return [torch.where(kept, t.float() * scale, 0.0).to(t.dtype).contiguous() for t in (x, grad)]


def _plain_log_probs(s):
    case, tokens, logits, k = s["case"], s["tokens"], s["logits"].detach(), s["case"]["top"]
    z = logits.float() / case["temperature"]
    high = z.amax(-1, keepdim=True)
    e = torch.exp(z - high)
    total = e.sum(-1, keepdim=True)
    lp = z - (high + torch.log(total))
    p = e / total
    del z, e
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    valid = tokens >= 0
    at = torch.where(valid, tokens, 0)[..., None]
    res = [torch.where(valid, lp.gather(-1, at)[..., 0], 0.0), torch.where(valid, entropy, 0.0)]
    if k:
        # the largest logits, the lowest number first among equal ones: both in one whole number
        bits = (logits.float() + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * 2 ** 32 + (2 ** 32 - 1 - torch.arange(lp.shape[-1], device=lp.device))
        best = 2 ** 32 - 1 - (key.topk(k, -1).values & 0xFFFFFFFF)
        del bits, key
        res += [torch.where(valid[..., None], lp.gather(-1, best), -math.inf), torch.where(valid[..., None], best, -1)]
    if case["train"]:
        g_lp, g_h = s["grads"][0][..., None], s["grads"][1][..., None]
        g_sum = g_lp + s["grads"][2].sum(-1, keepdim=True) if k else g_lp
        d = -p * (g_sum + g_h * torch.where(p > 0, lp + entropy[..., None], 0.0))
        d.scatter_add_(-1, at, g_lp)
        if k:
            d.scatter_add_(-1, best, s["grads"][2])
        res.append(torch.where(valid[..., None], d / case["temperature"], 0.0).to(logits.dtype))
    return res


def run(state):
    if own:
        return _own(state)
    return {"embedding": _plain_embedding, "dropout": _plain_dropout, "log_probs": _plain_log_probs}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_kept(n, seed, offset, p, device):
    """Philox again, each 32-bit product from 16-bit halves; which of n elements stay."""
    kept = torch.empty(n, dtype=torch.bool, device=device)
    half, low = 0xFFFF, 0xFFFFFFFF

    def high_low(x, m):
        m1, m0, x1, x0 = m >> 16, m & half, x >> 16, x & half
        mid = m1 * x0 + ((m0 * x0) >> 16)
        side = m0 * x1 + (mid & half)
        return m1 * x1 + (mid >> 16) + (side >> 16), ((side & half) << 16) | (m0 * x0 & half)

    for begin in range(0, n, 1 << 26):
        end = min(n, begin + (1 << 26))
        v = [torch.arange(begin // 4, -(-end // 4), device=device)]
        v = [v[0] % 2 ** 32, v[0] // 2 ** 32, torch.full_like(v[0], offset % 2 ** 32), torch.full_like(v[0], offset // 2 ** 32)]
        for r in range(10):
            (h0, l0), (h1, l1) = high_low(v[0], 0xD2511F53), high_low(v[2], 0xCD9E8D57)
            key = [(seed % 2 ** 32 + r * 0x9E3779B9) & low, (seed // 2 ** 32 + r * 0xBB67AE85) & low]
            v = [h1 ^ v[1] ^ key[0], l1, h0 ^ v[3] ^ key[1], l0]
        w = torch.stack(v, 1).flatten()[: end - begin]
        kept[begin:end] = w.double() >= math.floor(p * 2.0 ** 32 + 0.5)
    return kept


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        W, tokens = s["weight"].detach().double(), s["tokens"]
        res = [torch.nn.functional.embedding(tokens, W) * case["scale"]]
        if case["train"]:
            g = s["grad"].double() * case["scale"]
            if case["padded"] > 0:
                g = g * (tokens != 0)[..., None]
            res.append(torch.zeros_like(W).index_add_(0, tokens.flatten(), g.flatten(0, 1)))
        return res
    if case["op"] == "dropout":
        x = s["x"].detach()
        shape = x.shape[1:] if case["shared"] else x.shape
        kept = _exact_kept(math.prod(shape), s["seed"], s["offset"], case["p"], x.device).view(shape)
        return [(t.double() / (1 - case["p"])).mul_(kept).contiguous() for t in (x, s["grad"])]
    logits, tokens, k, V = s["logits"].detach().flatten(0, 1), s["tokens"].flatten(), case["top"], case["vocab"]
    N = tokens.numel()
    f64 = dict(device=logits.device, dtype=torch.float64)
    lp, ent = torch.zeros(N, **f64), torch.zeros(N, **f64)
    tops, ids = torch.full((N, k), -math.inf, **f64), torch.full((N, k), -1, device=logits.device)
    d = torch.zeros(N, V, **f64) if case["train"] else None
    step = max(1, (1 << 27) // V)
    for begin in range(0, N, step):
        rows = torch.arange(begin, min(N, begin + step), device=logits.device)
        rows = rows[tokens[rows] != -100]
        z = logits[rows].double() / case["temperature"]
        at = tokens[rows, None]
        logp = torch.log_softmax(z, -1)
        p = logp.exp()
        weighed = torch.nan_to_num(logp, neginf=0.0)
        lp[rows], ent[rows] = logp.gather(1, at)[:, 0], -(p * weighed).sum(1)
        if k:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
            tops[rows], ids[rows] = logp.gather(1, order), order
        if d is not None:
            gs = [t.flatten(0, 1)[rows].double() for t in s["grads"]]
            # through the log-softmax: what reaches every log probability, less p times its sum
            up = -gs[1][:, None] * p * (weighed + 1)
            up.scatter_add_(1, at, gs[0][:, None])
            if k:
                up.scatter_add_(1, order, gs[2])
            d[rows] = (up - p * up.sum(1, keepdim=True)) / case["temperature"]
    shape = s["tokens"].shape
    res = [lp.view(shape), ent.view(shape)] + ([tops.view(*shape, k), ids.view(*shape, k)] if k else [])
    return res + ([d.view(*shape, V)] if case["train"] else [])


# ---------------------------------------------------------------- what a pass cannot do without
def _different(n, vocab):
    """How many different words n draws are expected to meet (word v with probability log(1 + 1/(v+1)) / log(vocab+1))."""
    v = torch.arange(1, vocab + 1, dtype=torch.float64)
    p = torch.log1p(1 / v) / math.log(vocab + 1)
    return float((1 - torch.exp(n * torch.log1p(-p))).sum())


def work(case):
    """Bytes: each input read once and each output written once (of a table the rows that are met; of a table's gradient all;
    rows of logits that are ignored are not read).  Flops: the additions and products of the formulas; a random word counts none."""
    e, N = SIZE[case["dtype"]], case["steps"] * case["batch"]
    if case["op"] == "embedding":
        D, V = case["width"], case["vocab"]
        live = N * (1 - case["padded"])
        b = 8 * N + e * D * (N + _different(live, V))
        f = N * D
        if case["train"]:
            b += e * D * (live + V)
            f += 2 * live * D
        return {"bytes": b, "flops": f}
    if case["op"] == "dropout":
        n = N * case["width"]
        return {"bytes": 4 * e * n, "flops": 2 * n}
    V, k, live = case["vocab"], case["top"], N * (1 - case["ignored"])
    b = e * live * V + N * (8 + 8 + 12 * k)
    f = 6 * live * V
    if case["train"]:
        b += e * N * V + N * (8 + 4 * k)
        f += 6 * live * V
    return {"bytes": b, "flops": f}
