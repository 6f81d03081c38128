"""CPU oracle for the state space operators and for sampling (test infrastructure only), written token by token and row by row from the
definitions, in the type of its inputs (the tests hand in fp64), so that autograd through it is the gradient of the definition.

Pinned by (tests/test_oracle_ssm.py): the scan with one state and constant inputs against the geometric series, and against two halves
chained through the state; the convolution against torch's conv1d; the norm against a row of equal elements; sampling against
the cuts counted by hand, and its frequencies against the weights."""
from __future__ import annotations

import math

import torch


def _ends(lengths, B, T):
    return [T] * B if lengths is None else [int(n) for n in lengths]


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True):
    B, T, D = x.shape
    W = weight.shape[1]
    ys, states = [], []
    for b, end in enumerate(_ends(lengths, B, T)):
        window = [state[b, i] if state is not None else torch.zeros_like(x[b, 0]) for i in range(W - 1)]
        rows = []
        for t in range(T):
            if t >= end:
                rows.append(torch.zeros_like(x[b, 0]))
                continue
            window.append(x[b, t])
            p = sum(weight[:, k] * window[k] for k in range(W))
            p = p if bias is None else p + bias
            rows.append(p * torch.sigmoid(p) if silu else p)
            window.pop(0)
        ys.append(torch.stack(rows))
        states.append(torch.stack(window))
    return torch.stack(ys), torch.stack(states)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None):
    Bn, T, Dn = x.shape
    N = A.shape[1]
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    G = B.shape[2]
    ys, states = [], []
    for b, end in enumerate(_ends(lengths, Bn, T)):
        h = state[b] if state is not None else torch.zeros(Dn, N, dtype=x.dtype)
        rows = []
        for t in range(T):
            if t >= end:
                rows.append(torch.zeros_like(x[b, 0]))
                continue
            step = torch.nn.functional.softplus(dt[b, t] if dt_bias is None else dt[b, t] + dt_bias, threshold=50)
            vb, vc = (v[b, t].repeat_interleave(Dn // G, 0) for v in (B, C))             # (D, N)
            h = torch.exp(step[:, None] * A) * h + (step * x[b, t])[:, None] * vb
            y = (h * vc).sum(1)
            y = y if D is None else y + D * x[b, t]
            rows.append(y if z is None else y * z[b, t] * torch.sigmoid(z[b, t]))
        ys.append(torch.stack(rows))
        states.append(h)
    return torch.stack(ys), torch.stack(states)


def rms_norm(x, weight, eps, residual=None):
    r = x if residual is None else x + residual
    return r / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + eps) * weight, r


def sample(logits, u, temperature, top_k, top_p, min_p):
    """One row: (token, log of its probability, the kept tokens).  The weights are those of fp32 arithmetic, as the definition
    has them: exponents in octaves and their powers rounded to fp32, whole 2^-31ths."""
    l = [-math.inf if math.isnan(v) else v for v in logits.double().tolist()]
    top = max(l)
    if top == -math.inf:
        return -1, -math.inf, []
    f32 = lambda v: torch.tensor(v, dtype=torch.float32)
    warm = temperature >= 1e-6
    scale = f32(1.4426950408889634) / f32(temperature if warm else 1.0)
    s = torch.where(logits.float() == top, f32(0.0), (f32(top) - f32(l)) * scale).tolist()
    s = [math.inf if v == -math.inf else o for v, o in zip(l, s)]
    w = [int(round(float(f32(2.0 ** -v).double()) * 2 ** 31)) if v < 40 else 0 for v in s]
    order = sorted(range(len(l)), key=lambda i: (s[i], i))
    if not warm:
        order = order[:1]
    elif top_k > 0:
        order = order[:top_k]
    least = min(max(math.ceil(float(f32(min_p).double()) * 2 ** 31), 1), 2 ** 31)
    order = [i for i in order if w[i] >= least]
    p = float(f32(top_p).double())
    if p < 1:
        total = sum(w[i] for i in order)
        need, run, n = max(1, math.ceil(p * float(total))), 0, 0
        while run < need:
            run += w[order[n]]
            n += 1
        order = order[:n]
    kept = sorted(order)
    total = sum(w[i] for i in kept)
    target = min(math.floor(float(f32(u).double()) * float(total)), total - 1)
    run = 0
    for i in kept:
        run += w[i]
        if run > target:
            return i, math.log(w[i] / total), kept
