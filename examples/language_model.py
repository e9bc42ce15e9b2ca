"""A language model of LSTM layers on the package's operators: trained on sequences of different lengths, then asked to go on.

    python -m examples.language_model [--steps 200] [--vocab 1000] [--width 256] [--layers 2] [--dtype fp32]

One table serves both ends (tokens in, predictions out); dropout uses one mask for all steps of a sequence; padding counts
neither in the loss nor in the table's gradient.  The sequences count upwards in steps of one to four, modulo the vocabulary."""
import argparse
import math

import torch
import torch.nn as nn

import fastlstm_b200 as F

PADDING = 0


class LanguageModel(nn.Module):
    def __init__(self, vocab, width, layers=2, dropout=0.2, device="cuda", dtype=torch.bfloat16, seed=1):
        super().__init__()
        self.table = nn.Parameter(torch.randn(vocab, width, device=device, dtype=torch.float32).mul_(width ** -0.5).to(dtype))
        self.layers = nn.ModuleList(F.FastLSTM(width, width, device=device, dtype=dtype) for _ in range(layers))
        self.dropout, self.seed = dropout, seed

    def forward(self, tokens, states=None, step=0):
        """tokens [T,B] -> (logits [T,B,vocab], states).  step: the training step's number, for masks of its own."""
        n = len(self.layers)
        x = F.embedding(tokens, self.table, scale=math.sqrt(self.table.shape[1]), padding_idx=PADDING)
        out = []
        for i, layer in enumerate(self.layers):
            x = F.dropout(x, self.dropout, self.seed, offset=step * (n + 1) + i, shared_dim=0, training=self.training)
            x, state = layer(x, None if states is None else states[i])
            out.append(state)
        x = F.dropout(x, self.dropout, self.seed, offset=step * (n + 1) + n, shared_dim=0, training=self.training)
        return x @ self.table.t(), out

    def loss(self, tokens, targets, step=0, entropy_weight=0.0):
        """Mean negative log likelihood of the targets that are no padding (less entropy_weight times the mean entropy)."""
        logits, _ = self(tokens, step=step)
        r = F.token_log_probs(logits, targets, ignore_index=PADDING)
        return -(r.log_probs + entropy_weight * r.entropy).sum() / (targets != PADDING).sum()

    @torch.no_grad()
    def go_on(self, tokens, steps, top=5, temperature=1.0):
        """The likeliest continuation of tokens [T,B]: (its tokens [steps,B], their log probabilities, the `top` alternatives
        of every step and theirs [steps,B,top])."""
        logits, states = self(tokens)
        picked = []
        for _ in range(steps):
            # (asked about a token that is known already; the alternatives are what matters here)
            r = F.token_log_probs(logits[-1], tokens[-1], top=top, temperature=temperature, ignore_index=-1)
            tokens = r.top_tokens[None, :, 0]
            picked.append((tokens[0], r.top_log_probs[:, 0], r.top_tokens, r.top_log_probs))
            logits, states = self(tokens, states)
        return tuple(torch.stack(t) for t in zip(*picked))


def batch(vocab, T, B, generator):
    """Tokens and targets [T,B]: counting modulo the vocabulary (without the padding token), padded behind each one's end."""
    g = dict(generator=generator, device="cuda")
    first, pace = torch.randint(0, vocab - 1, (B,), **g), torch.randint(1, 5, (B,), **g)
    length = torch.randint(T // 2, T + 1, (B,), **g)
    t = torch.arange(T + 1, device="cuda")[:, None]
    s = torch.where(t <= length, 1 + (first + pace * t) % (vocab - 1), PADDING)
    return s[:-1], torch.where(t[1:] <= length, s[1:], PADDING)


def train(model, steps, T=48, B=64, lr=3e-3, report=None):
    vocab = model.table.shape[0]
    generator = torch.Generator(device="cuda").manual_seed(7)
    optimiser = torch.optim.Adam(model.parameters(), lr=lr)
    losses = []
    for step in range(steps):
        tokens, targets = batch(vocab, T, B, generator)
        loss = model.loss(tokens, targets, step)
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
        if report and step % report == 0:
            print("step %4d  loss %.4f" % (step, float(losses[-1])))
    F.check_status()
    return torch.stack(losses).float().tolist()


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--vocab", type=int, default=1000)
    p.add_argument("--width", type=int, default=256)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--dtype", choices=("fp32", "fp16", "bf16"), default="fp32")
    a = p.parse_args()
    torch.manual_seed(0)
    dtype = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    model = LanguageModel(a.vocab, a.width, a.layers, dtype=dtype)
    train(model, a.steps, report=20)
    model.eval()
    start = 1 + torch.arange(10, device="cuda")[:, None] * torch.tensor([1, 2, 3], device="cuda")
    tokens, log_probs, top_tokens, top_log_probs = model.go_on(start, 8)
    for b in range(start.shape[1]):
        print(start[:, b].tolist(), "->", tokens[:, b].tolist(), "log probability %.3f" % float(log_probs[:, b].sum()))
        print("    alternatives of the first:", [(t, round(lp, 2)) for t, lp in zip(top_tokens[0, b].tolist(), top_log_probs[0, b].tolist())])


if __name__ == "__main__":
    main()
