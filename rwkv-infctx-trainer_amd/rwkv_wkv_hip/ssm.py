"""The operators of a state space block on the HIP kernels of csrc/ssm_*.hip, and the block's forward on them.

  causal_conv       the short causal convolution over the tokens, a filter per channel, its window carried as a state
  selective_scan    the selective state space scan with its gate, the state carried in and out
  rms_norm          the residual's addition and the root-mean-square norm
  rms_norm_fp8      the same with the normalised rows in 8 bits and a scale per row, for an 8-bit projection

  block_forward     norm, projection, convolution, projections, scan, projection of a module that holds the parameters

All but rms_norm_fp8 are differentiable in every floating-point input, the states included; a call that no gradient is recorded for keeps
nothing for a backward, and the scan of a single token has a kernel of its own.  Sums, states and norms are held in fp32 whatever
the inputs' type.  Results and gradients repeat to the bit.  Every function needs GPU tensors and the built library; there is no CPU path.

A recorded scan keeps fp32 states from its forward to its backward, one in 16 tokens: 4 bytes per token and channel up to 16 states, 8 up to 32, 16 above.
While it runs its backward takes N / 4 bytes per token and channel (N / 2 above 32 states) for the gradients of B and C: 268 MB kept and 268 MB taken for 16384 tokens
of 4096 channels with 16 states, 8.6 GB and 17 GB for 65536 tokens of 8192 channels with 64.

The reference has no state space models; the operators follow the conventions of its time mix (states in and out, truncated
backpropagation through time) with the layouts (B, T, channels)."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _lib
from .ops import _Traced


def _call(name, *args):
    out = getattr(_lib.host(), name)(*args)
    if out is not None:
        return out
    # torch.jit.trace records: the call is one node of the graph, over its tensors
    at = [i for i, a in enumerate(args) if torch.is_tensor(a)]

    def again(*tensors):
        full = list(args)
        for i, t in zip(at, tensors):
            full[i] = t
        return _call(name, *full)

    return _Traced.apply(again, None, *[args[i] for i in at])


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True, out_state=None):
    """x (B,T,D), weight (D,W) with W = 2 to 4 taps, bias (D) -> (y (B,T,D), new_state (B,W-1,D)):

        y[t] = act(bias + sum_k weight[:, k] xx[t - (W-1) + k]),   xx = x continued to the left by ``state``

    with act the SiLU, or nothing with ``silu=False``.  ``state`` (B,W-1,D), the W-1 inputs before x (None: zeros), and the
    new state have x's type; weight and bias are read in x's type if both have it, else both in fp32.  x may be a slice of a wider
    tensor (any strides but the last).  ``lengths`` (B, integers): where each sequence ends; later tokens are not read, their y is
    zero, and the new state is the one after the sequence's last token.  ``out_state``: a buffer the new state is written
    to, without autograd, as by an operation in place; for a single token it may be ``state`` itself."""
    return _call("causal_conv", x, weight, bias, state, lengths, bool(silu), out_state)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, state=None, lengths=None, out_state=None):
    """x, dt (B,T,D), A (D,N), B, C (B,T,N) or (B,T,G,N) -> (y (B,T,D), new_state (B,D,N) fp32), with N up to 64:

        step = softplus(dt + dt_bias)
        h[t] = exp(step A) h[t-1] + step x[t] B[t]
        y[t] = (C[t] . h[t] + D x[t]) silu(z[t])

    G groups of D/G consecutive channels have a B and C of their own.  D, dt_bias (D), the gate z (B,T,D) and the incoming ``state``
    may be left out.  x, dt, z, B and C share one type and may be slices of wider tensors (any strides but the last); A, D,
    dt_bias and the state are read in fp32 whatever their type, and the new state is fp32.  ``lengths`` and ``out_state`` as in ``causal_conv``."""
    return _call("selective_scan", x, dt, A, B, C, D, z, dt_bias, state, lengths, out_state)


def rms_norm(x, weight, eps=1e-5, residual=None):
    """x (..., C), weight (C), residual (..., C) in x's type or fp32 -> (y in x's type, the sum x + residual in the residual's type):
    y = r / sqrt(mean(r^2) + eps) * weight of r = x + residual.  Without a residual the second result is x."""
    return _call("rms_norm", x, weight, float(eps), residual)


def rms_norm_fp8(x, weight, eps=1e-5, residual=None):
    """As ``rms_norm``, its y in 8 bits: (q (..., C) float8_e4m3fn, scale (..., 1) fp32, sum) with y = q * scale,
    scale = max |y| / 448 of the row (1 for a row of zeros, NaN for a row with one), as ``torch._scaled_mm`` takes them.  Without autograd only."""
    return _call("rms_norm_fp8", x, weight, float(eps), residual)


def block_state(module, batch, dtype, device="cuda"):
    """The state before the first token: the convolution's window and the scan's state."""
    D, W = module.conv_weight.shape
    return (torch.zeros(batch, W - 1, D, dtype=dtype, device=device),
            torch.zeros(batch, D, module.A_log.shape[1], dtype=torch.float32, device=device))


def block_forward(self, x, residual, state, lengths=None):
    """One state space block on a residual stream: x (B,T,C) is the block before's output, ``residual`` (B,T,C) the stream it is added to (None: x
    begins it), ``state`` as ``block_state`` gives it.  Returns (out (B,T,C), residual, new_state).

    ``self`` holds norm_weight (C), eps, in_proj (C -> 2D, the stream and its gate), conv_weight (D,W), conv_bias (D), x_proj
    (D -> R + 2N: the time step's low-rank input, B, C), dt_proj_weight (D,R), dt_bias (D), A_log (D,N), D (D), out_proj (D -> C); the
    projections stay torch matmuls (hipBLASLt)."""
    h, residual = rms_norm(x, self.norm_weight, self.eps, residual)
    u, z = self.in_proj(h).chunk(2, dim=-1)
    u, window = causal_conv(u, self.conv_weight, self.conv_bias, state[0], lengths)
    N, R = self.A_log.shape[1], self.dt_proj_weight.shape[1]
    low, b, c = self.x_proj(u).split([R, N, N], dim=-1)
    y, h = selective_scan(u, F.linear(low, self.dt_proj_weight), -torch.exp(self.A_log.float()), b, c, D=self.D, z=z, dt_bias=self.dt_bias,
                          state=state[1], lengths=lengths)
    return self.out_proj(y), residual, (window, h)
