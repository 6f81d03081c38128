"""The operators of a gated recurrence model on the HIP kernels of csrc/gated_*.hip and csrc/embedding.hip, and a block's forward on them.

  gated_recurrence     the gated linear recurrence over the tokens, a state per channel carried in and out, with its output gate
  gated_feed_forward   both input projections of a gated feed-forward, the activation and the product
  embedding            rows of a table by token, scaled; the table's gradient from the places sorted by token

  block_forward        norm, projections, convolution, recurrence, projection, norm, gated feed-forward of a module that holds the parameters

All are differentiable in every floating-point input, states included; a call that no gradient is recorded for keeps nothing for a backward.  Sums, states and
norms are held in fp32 whatever the inputs' type.  Results and gradients repeat to the bit.  Every function needs GPU tensors and the built
library; there is no CPU path.

The reference has no such models; the operators follow the conventions of its time mix (states in and out, truncated backpropagation through
time) and those of the state space operators beside them, with the layouts (B, T, channels)."""
from __future__ import annotations

import torch

from .ssm import _call, causal_conv, rms_norm

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}


def gated_recurrence(x, r, i, decay, z=None, state=None, lengths=None, scale=8.0, out_state=None):
    """x, r, i (B,T,D), decay (D) -> (y (B,T,D), new_state (B,D) fp32):

        a[t] = exp(-scale softplus(decay) sigmoid(r[t]))
        h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) sigmoid(i[t]) x[t]
        y[t] = h[t] silu(z[t]),  or h[t] without z

    r and i are the gates before their sigmoids.  x, r, i and z (B,T,D) share one type and may be slices of wider tensors (any strides but the last); decay and the
    incoming ``state`` (B,D; None: zeros) are read in fp32 whatever their type, and the new state is fp32.  ``lengths`` (B, integers): where each
    sequence ends; later tokens are not read, their y is zero, and the new state is the one after the sequence's last token.  ``out_state``: a buffer the
    new state is written to, without autograd, as by an operation in place; for a single token it may be ``state`` itself.

    A recorded call keeps an fp32 state per 64 tokens, a sixteenth of a byte per token and channel, beside its inputs."""
    return _call("gated_recurrence", x, r, i, decay, z, state, lengths, float(scale), out_state)


def gated_feed_forward(x, w_gate, w_up, activation="silu"):
    """x (..., C), w_gate and w_up (F, C) as torch.nn.Linear keeps them -> act(x w_gate') * (x w_up') (..., F), act "silu", "gelu" (its tanh
    form) or "relu".  All of one type (under torch.autocast different ones are cast to
    its type, as torch's own projections cast them); sums in fp32, the result rounded once.  The second projection stays the caller's matrix product.

    A recorded call keeps both projections' results in fp32 (2 F numbers per row) for its backward, whose workspace is their slopes, 2 F elements of x's type per row
    (twice that up to 32 rows), and the sums of a small product's shares.  Where C is not whole pieces of 16 bytes the backward copies x and the weights, the forward where
    there are many rows.  The slopes are rounded to x's type, up to 32 rows to twice its digits; in fp16 they are scaled by a
    power of two first, to the largest of the call, so that they have fp32's range: what is below 2^-29 of the largest loses digits."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r} is none of {', '.join(ACTIVATIONS)}")
    return _call("gated_product", x, w_gate, w_up, ACTIVATIONS[activation])


def embedding(tokens, weight, scale=1.0):
    """tokens (...) int64 or int32, weight (V, C) -> scale * weight[tokens] (..., C) in weight's type, rounded once.

    A token below zero or from V on is a place without one, as padding has it: its row is zeros, and its gradient goes nowhere.  The gradient of ``weight`` is dense,
    each row the fp32 sum of its places' gradients: by runs of up to 64 of the places sorted by token, each run in the places' order, then over the runs in order.  Where the
    runs begin depends on the other places too, so a row's last bits do; the same call gives the same bits."""
    return _call("embedding", tokens, weight, float(scale))


def block_state(module, batch, dtype, device="cuda"):
    """The state before the first token: the convolution's window and the recurrence's state."""
    D, W = module.conv_weight.shape
    return torch.zeros(batch, W - 1, D, dtype=dtype, device=device), torch.zeros(batch, D, dtype=torch.float32, device=device)


def block_forward(self, x, residual, state, lengths=None):
    """One gated recurrence block on a residual stream: x (B,T,C) is the block before's output, ``residual`` (B,T,C) the stream it is added to (None: x
    begins it), ``state`` as ``block_state`` gives it.  Returns (out (B,T,C), residual, new_state).

    ``self`` holds norm_weight (C), eps, in_proj (C -> 2D, the stream and its gate), conv_weight (D,W), conv_bias (D), gate_proj (D -> 2D: r and i), decay (D),
    out_proj (D -> C), ff_norm_weight (C), ff_gate and ff_up (F,C), ff_down (F -> C) and activation; the other projections stay torch
    matmuls (hipBLASLt)."""
    h, residual = rms_norm(x, self.norm_weight, self.eps, residual)
    u, z = self.in_proj(h).chunk(2, dim=-1)
    u, window = causal_conv(u, self.conv_weight, self.conv_bias, state[0], lengths, silu=False)
    r, i = self.gate_proj(u).chunk(2, dim=-1)
    y, h = gated_recurrence(u, r, i, self.decay, z=z, state=state[1], lengths=lengths)
    n, residual = rms_norm(self.out_proj(y), self.ff_norm_weight, self.eps, residual)
    return self.ff_down(gated_feed_forward(n, self.ff_gate, self.ff_up, self.activation)), residual, (window, h)
