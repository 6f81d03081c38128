"""A small gated recurrence language model on the package's operators: its embedding scaled and tied to the head, trained by truncated backpropagation through
time with the states carried from segment to segment, then served in a batch of prompts of different lengths, token by token.

    python examples/gated_recurrence_lm.py [--steps 60] [--tokens 32]

The text is synthetic: every token determines the next (next = 5 token + 3 modulo the vocabulary)."""
import argparse
import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rwkv-infctx-trainer_amd"))
from rwkv_wkv_hip import gated, sampling, ssm  # noqa: E402

VOCABULARY, WIDTH, INNER, TAPS, HIDDEN, EPS = 256, 256, 320, 4, 640, 1e-6


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        ones = lambda n: torch.nn.Parameter(torch.ones(n).bfloat16())
        linear = lambda i, o: torch.nn.Linear(i, o, bias=False, dtype=torch.bfloat16)
        weight = lambda *s: torch.nn.Parameter((torch.randn(*s) * s[-1] ** -0.5).bfloat16())
        self.eps, self.activation = EPS, "gelu"
        self.norm_weight, self.ff_norm_weight = ones(WIDTH), ones(WIDTH)
        self.in_proj, self.gate_proj, self.out_proj, self.ff_down = linear(WIDTH, 2 * INNER), linear(INNER, 2 * INNER), linear(INNER, WIDTH), linear(HIDDEN, WIDTH)
        self.conv_weight, self.conv_bias = weight(INNER, TAPS), torch.nn.Parameter(torch.zeros(INNER).bfloat16())
        # an open gate of scale 8 leaves a between 0.9 and 0.999 of the state: softplus(decay) = -log(a) / 8
        self.decay = torch.nn.Parameter(torch.log(torch.expm1(-torch.log(torch.empty(INNER).uniform_(0.9, 0.999)) / 8.0)))
        self.ff_gate, self.ff_up = weight(HIDDEN, WIDTH), weight(HIDDEN, WIDTH)

    def forward(self, x, residual, state, lengths=None):
        return gated.block_forward(self, x, residual, state, lengths)


class Model(torch.nn.Module):
    def __init__(self, layers=2):
        super().__init__()
        self.table = torch.nn.Parameter((torch.randn(VOCABULARY, WIDTH) * WIDTH ** -0.5).bfloat16())
        self.blocks = torch.nn.ModuleList(Block() for _ in range(layers))
        self.norm_weight = torch.nn.Parameter(torch.ones(WIDTH).bfloat16())

    def states(self, batch):
        return [gated.block_state(b, batch, torch.bfloat16) for b in self.blocks]

    def body(self, tokens, states, lengths=None):
        """(what the last block adds to the stream, the stream, the new states); the stream is kept in fp32"""
        x, new = gated.embedding(tokens, self.table, math.sqrt(WIDTH)), []
        residual = torch.zeros(x.shape, device=x.device)
        for block, state in zip(self.blocks, states):
            x, residual, state = block(x, residual, state, lengths)
            new.append(state)
        return x, residual, new

    def forward(self, tokens, states):
        x, residual, states = self.body(tokens, states)
        return ssm.rms_norm(x, self.norm_weight, EPS, residual)[0] @ self.table.t(), states


def text(batch, length, generator):
    rows = [torch.randint(0, VOCABULARY, (batch, 1), generator=generator, device="cuda")]
    for _ in range(length):
        rows.append((5 * rows[-1] + 3) % VOCABULARY)
    return torch.cat(rows, 1)


def train(model, steps, batch=16, segments=2, length=96, generator=None, report=print):
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3, weight_decay=0.0)
    losses = []
    for step in range(steps):
        tokens, states = text(batch, segments * length, generator), model.states(batch)
        for s in range(segments):
            part = tokens[:, s * length:(s + 1) * length + 1]
            logits, states = model(part[:, :-1], states)
            loss = F.cross_entropy(logits.flatten(0, 1).float(), part[:, 1:].flatten())
            optimizer.zero_grad(set_to_none=True)
            loss.backward()
            optimizer.step()
            states = [(w.detach(), h.detach()) for w, h in states]          # the next segment goes on from here
        losses.append(loss.detach())
        if report and step % 20 == 0:
            report(f"step {step}: loss {losses[-1].item():.3f}", flush=True)
    return [v.item() for v in losses]


@torch.no_grad()
def serve(model, prompts, tokens, temperature=0.7, top_k=20, top_p=0.95, generator=None):
    """prompts: token lists of any lengths -> (batch, tokens) sampled continuations and their log probabilities"""
    B, lengths = len(prompts), torch.tensor([len(p) for p in prompts], device="cuda", dtype=torch.int32)
    padded = torch.full((B, max(map(len, prompts))), -1)          # (padding is no token: its row is zeros)
    for i, p in enumerate(prompts):
        padded[i, :len(p)] = torch.tensor(p)
    x, residual, states = model.body(padded.cuda(), model.states(B), lengths)
    last = (lengths.long() - 1)[:, None, None].expand(B, 1, WIDTH)
    x, residual = x.gather(1, last), residual.gather(1, last)
    out, logprobs = [], []
    for _ in range(tokens):
        logits = ssm.rms_norm(x[:, 0], model.norm_weight, EPS, residual[:, 0])[0] @ model.table.t()
        token, logprob = sampling.sample(logits, torch.rand(B, device="cuda", generator=generator), temperature, top_k, top_p)
        out.append(token)
        logprobs.append(logprob)
        x, residual, states = model.body(token[:, None], states)
    return torch.stack(out, 1), torch.stack(logprobs, 1)


def main():
    a = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    a.add_argument("--steps", type=int, default=60)
    a.add_argument("--tokens", type=int, default=32)
    a = a.parse_args()
    torch.manual_seed(0)
    generator = torch.Generator(device="cuda").manual_seed(0)
    model = Model().cuda()
    losses = train(model, a.steps, generator=generator)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}")
    prompts = [text(1, n, generator)[0].tolist() for n in (1, 7, 30, 95)]
    written, logprobs = serve(model, prompts, a.tokens, generator=generator)
    for p, w, l in zip(prompts, written.tolist(), logprobs):
        right = sum(b == (5 * x + 3) % VOCABULARY for x, b in zip([p[-1]] + w, w))
        print(f"prompt of {len(p)} tokens: {right} of {len(w)} tokens follow the rule, mean log probability {l.mean().item():.3f}")


if __name__ == "__main__":
    main()
