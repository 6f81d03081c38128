"""CPU oracle for the operators of a gated recurrence model (test infrastructure only), written from the definitions, token by token, in the type of its inputs (the
tests hand in fp64), so that autograd through it is the gradient of the definition.

Pinned by (tests/test_oracle_gated.py): the recurrence with constant gates against the geometric series, and against two halves chained through the
state; the activations against torch's; the lookup against a one-hot product; every gradient against differences."""
from __future__ import annotations

import math

import torch


def gated_recurrence(x, r, i, decay, z=None, state=None, lengths=None, scale=8.0):
    B, T, D = x.shape
    ends = torch.full((B,), T) if lengths is None else torch.as_tensor(lengths).cpu().long()
    soft = torch.logaddexp(decay, torch.zeros_like(decay))
    h = torch.zeros(B, D, dtype=x.dtype) if state is None else state
    ys = []
    for t in range(T):
        live = (t < ends)[:, None]
        # (what is not there is replaced before it is used: a NaN in it must not reach a gradient)
        at = lambda v: torch.where(live, v[:, t], torch.zeros_like(v[:, t]))
        log_a = -scale * soft * torch.sigmoid(at(r))
        one = -torch.expm1(2 * log_a)
        some = one > 0
        beta = torch.where(some, torch.where(some, one, torch.ones_like(one)).sqrt(), torch.zeros_like(one))
        h = torch.where(live, torch.exp(log_a) * h + beta * torch.sigmoid(at(i)) * at(x), h)
        y = h if z is None else h * at(z) * torch.sigmoid(at(z))
        ys.append(torch.where(live, y, torch.zeros_like(y)))
    return torch.stack(ys, 1), h


def activation(name, g):
    if name == "relu":
        return torch.where(g > 0, g, torch.zeros_like(g))
    if name == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def gated_feed_forward(x, w_gate, w_up, name="silu"):
    return activation(name, x @ w_gate.t()) * (x @ w_up.t())


def embedding(tokens, weight, scale=1.0):
    rows = [scale * weight[t] if 0 <= t < len(weight) else torch.zeros_like(weight[0]) for t in tokens.flatten().tolist()]
    return torch.stack(rows).view(*tokens.shape, weight.shape[1])
