"""The operators around a language model in numpy, 64 bits, straight from their formulas (no torch, no kernels)."""
import numpy as np


# ---------------------------------------------------------------- embedding
def embedding(tokens, weight, scale=1.0):
    return weight.astype(np.float64)[tokens] * scale


def embedding_grad(tokens, dout, vocab, scale=1.0, padding_idx=None):
    """(dW, sum of the terms' magnitudes, terms) per row of the table; the last two bound what rounding may do."""
    flat, rows = tokens.reshape(-1), dout.astype(np.float64).reshape(tokens.size, -1)
    dW, size, terms = np.zeros((vocab, rows.shape[1])), np.zeros((vocab, rows.shape[1])), np.zeros(vocab)
    counted = np.ones(flat.shape, bool) if padding_idx is None else flat != padding_idx
    np.add.at(dW, flat[counted], rows[counted] * scale)
    np.add.at(size, flat[counted], np.abs(rows[counted] * scale))
    np.add.at(terms, flat[counted], 1)
    return dW, size, terms


# ---------------------------------------------------------------- dropout
def philox4x32(counter, key, rounds=10):
    """counter [..., 4], key [..., 2] of 32-bit words -> [..., 4] (Salmon, Moraes, Dror, Shaw 2011)."""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [np.asarray(key)[..., i].astype(np.uint64) for i in range(2)]
    low, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ k[0], b & low, (a >> s32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return np.stack(c, -1).astype(np.uint32)


def kept(count, p, seed, offset=0, first=0):
    """Which of the elements first .. first + count - 1 stay (first a multiple of 4)."""
    block = np.arange(first // 4, -(-(first + count) // 4), dtype=np.uint64)
    low, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    counter = np.stack([block & low, block >> s32, np.full_like(block, offset % 2 ** 32), np.full_like(block, offset // 2 ** 32)], -1)
    words = philox4x32(counter, np.array([seed % 2 ** 32, seed // 2 ** 32], np.uint64)).reshape(-1)[:count]
    return words.astype(np.float64) >= np.floor(p * 2.0 ** 32 + 0.5)


def dropout(x, p, seed, offset=0, shared_dim=None):
    """The mask applied to x (float64; the mask and the values are exact, the division is by 1 - p in 64 bits)."""
    shape = list(x.shape)
    if shared_dim is not None:
        shape[shared_dim] = 1
    mask = kept(int(np.prod(shape)), p, seed, offset).reshape(shape)
    return np.where(mask, x.astype(np.float64) / (1 - p if p < 1 else 1), 0.0)


# ---------------------------------------------------------------- log probabilities
def token_log_probs(logits, tokens, top=0, temperature=1.0, ignore_index=-100):
    """Rows of [N, V] -> dict of log_probs, entropy, top_log_probs, top_tokens and lp (all log probabilities)."""
    raw = logits.astype(np.float64)
    z = raw / temperature
    N, V = z.shape
    with np.errstate(all="ignore"):
        m = z.max(1, keepdims=True)
        none = np.isneginf(m)
        lp = z - np.where(none, 0, m)
        lp = np.where(none, -np.inf, lp - np.log(np.exp(lp).sum(1, keepdims=True)))
        ent = -np.where(np.isneginf(lp), 0.0, np.exp(lp) * lp).sum(1)
    live = tokens != ignore_index
    out = {"lp": lp, "log_probs": np.where(live, lp[np.arange(N), np.where(live, tokens, 0)], 0.0), "entropy": np.where(live, ent, 0.0)}
    if top:
        order = np.argsort(-raw, axis=1, kind="stable")[:, :top]
        out["top_tokens"] = np.where(live[:, None], order, -1)
        out["top_log_probs"] = np.where(live[:, None], np.take_along_axis(lp, order, 1), -np.inf)
    return out


def token_log_probs_grad(logits, tokens, g_lp=None, g_h=None, g_top=None, temperature=1.0, ignore_index=-100):
    """(dlogits, magnitude of the terms that the softmax multiplies) for rows of [N, V]."""
    top = 0 if g_top is None else g_top.shape[1]
    r = token_log_probs(logits, tokens, top, temperature, ignore_index)
    N, V = logits.shape
    zero = np.zeros(N)
    g_lp, g_h = (zero if g is None else g.astype(np.float64) for g in (g_lp, g_h))
    p, H, lp = np.exp(r["lp"]), r["entropy"][:, None], np.where(np.isneginf(r["lp"]), 0.0, r["lp"])
    g = g_lp + (0 if g_top is None else g_top.astype(np.float64).sum(1))
    d = -p * (g[:, None] + g_h[:, None] * (lp + H))
    size = p * (np.abs(g_lp)[:, None] + (0 if g_top is None else np.abs(g_top).sum(1)[:, None]) + np.abs(g_h)[:, None] * (np.abs(lp) + H))
    live = (tokens != ignore_index) & ~np.isneginf(r["lp"]).all(1)
    rows = np.arange(N)
    np.add.at(d, (rows[live], tokens[live]), g_lp[live])
    for k in range(top):
        np.add.at(d, (rows[live], r["top_tokens"][live, k]), g_top[live, k].astype(np.float64))
    return np.where(live[:, None], d / temperature, 0.0), np.where(live[:, None], size / temperature, 0.0)
