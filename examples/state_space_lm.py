"""A small state space language model on the package's operators: trained by truncated backpropagation through time, its states carried
from segment to segment, then served in a batch of prompts of different lengths, token by token, with the last norm in 8 bits in front of
an 8-bit head product and a sampling setting per user.

    python examples/state_space_lm.py [--steps 60] [--tokens 32]

The text is synthetic: every token determines the next (next = 5 token + 3 modulo the vocabulary), so what the model has
learned shows in what it writes."""
import argparse
import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rwkv-infctx-trainer_amd"))
from rwkv_wkv_hip import sampling, ssm  # noqa: E402

VOCABULARY, WIDTH, INNER, STATES, TAPS, RANK, EPS = 256, 256, 512, 16, 4, 16, 1e-5


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        p = lambda *s, std: torch.nn.Parameter((torch.randn(*s) * std).bfloat16())
        self.eps = EPS
        self.norm_weight = torch.nn.Parameter(torch.ones(WIDTH).bfloat16())
        self.in_proj = torch.nn.Linear(WIDTH, 2 * INNER, bias=False, dtype=torch.bfloat16)
        self.conv_weight, self.conv_bias = p(INNER, TAPS, std=TAPS ** -0.5), torch.nn.Parameter(torch.zeros(INNER).bfloat16())
        self.x_proj = torch.nn.Linear(INNER, RANK + 2 * STATES, bias=False, dtype=torch.bfloat16)
        self.dt_proj_weight = p(INNER, RANK, std=RANK ** -0.5)
        step = torch.exp(torch.empty(INNER).uniform_(math.log(1e-3), math.log(0.1)))
        self.dt_bias = torch.nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = torch.nn.Parameter(torch.log(torch.arange(1, STATES + 1).float()).expand(INNER, STATES).clone())
        self.D = torch.nn.Parameter(torch.ones(INNER))
        self.out_proj = torch.nn.Linear(INNER, WIDTH, bias=False, dtype=torch.bfloat16)

    def forward(self, x, residual, state, lengths=None):
        return ssm.block_forward(self, x, residual, state, lengths)


class Model(torch.nn.Module):
    def __init__(self, layers=2):
        super().__init__()
        self.embedding = torch.nn.Embedding(VOCABULARY, WIDTH, dtype=torch.bfloat16)
        self.blocks = torch.nn.ModuleList(Block() for _ in range(layers))
        self.norm_weight = torch.nn.Parameter(torch.ones(WIDTH).bfloat16())
        self.head = torch.nn.Linear(WIDTH, VOCABULARY, bias=False, dtype=torch.bfloat16)

    def states(self, batch):
        return [ssm.block_state(b, batch, torch.bfloat16) for b in self.blocks]

    def body(self, tokens, states, lengths=None):
        """(what the last block adds to the stream, the stream, the new states); the stream is kept in fp32"""
        x, new = self.embedding(tokens), []
        residual = torch.zeros(x.shape, device=x.device)
        for block, state in zip(self.blocks, states):
            x, residual, state = block(x, residual, state, lengths)
            new.append(state)
        return x, residual, new

    def forward(self, tokens, states):
        x, residual, states = self.body(tokens, states)
        y, _ = ssm.rms_norm(x, self.norm_weight, EPS, residual)
        return self.head(y), states


def text(batch, length, generator):
    t = torch.randint(0, VOCABULARY, (batch, 1), generator=generator, device="cuda")
    rows = [t]
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
def serve(model, prompts, tokens, temperature=0.7, top_k=20, top_p=0.95, min_p=0.0, generator=None):
    """prompts: token lists of any lengths -> (batch, tokens) sampled continuations and their log probabilities.  The settings are numbers
    or tensors with one per prompt."""
    B, lengths = len(prompts), torch.tensor([len(p) for p in prompts], device="cuda", dtype=torch.int32)
    padded = torch.zeros(B, max(map(len, prompts)), dtype=torch.long)
    for i, p in enumerate(prompts):
        padded[i, :len(p)] = torch.tensor(p)
    # the head in 8 bits, a scale per word
    head = model.head.weight.float()
    head_scale = head.abs().amax(1, keepdim=True) / 448.0
    head8 = (head / head_scale).to(torch.float8_e4m3fn)
    x, residual, states = model.body(padded.cuda(), model.states(B), lengths)
    last = (lengths.long() - 1)[:, None, None].expand(B, 1, WIDTH)
    x, residual = x.gather(1, last), residual.gather(1, last)
    out, logprobs = [], []
    for _ in range(tokens):
        q, scale, _ = ssm.rms_norm_fp8(x[:, 0], model.norm_weight, EPS, residual[:, 0])
        logits = torch._scaled_mm(q, head8.t(), scale_a=scale, scale_b=head_scale.t(), out_dtype=torch.bfloat16)
        u = torch.rand(B, device="cuda", generator=generator)
        token, logprob = sampling.sample(logits, u, temperature, top_k, top_p, min_p)
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
    written, logprobs = serve(model, prompts, a.tokens, temperature=torch.tensor([0.0, 0.5, 0.7, 1.0], device="cuda"), generator=generator)
    for p, w, l in zip(prompts, written.tolist(), logprobs):
        right = sum(b == (5 * x + 3) % VOCABULARY for x, b in zip([p[-1]] + w, w))
        print(f"prompt of {len(p)} tokens: {right} of {len(w)} tokens follow the rule, mean log probability {l.mean().item():.3f}")


if __name__ == "__main__":
    main()
