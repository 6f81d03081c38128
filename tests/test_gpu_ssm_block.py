"""The state space block on the package's operators against the same block on the oracle's, and the example that trains and serves it."""
import os
import sys

import pytest
import torch

from oracle import ssm as O
from tests.util import assert_close

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


class Block(torch.nn.Module):
    def __init__(self, C=24, D=40, N=16, R=3, W=4, eps=1e-5):
        super().__init__()
        g = torch.Generator().manual_seed(1)
        p = lambda *s, std=0.3: torch.nn.Parameter(torch.randn(*s, generator=g) * std)
        self.eps, self.norm_weight, self.conv_weight, self.conv_bias = eps, p(C, std=1.0), p(D, W), p(D)
        self.in_proj, self.x_proj, self.out_proj = (torch.nn.Linear(i, o, bias=False) for i, o in ((C, 2 * D), (D, R + 2 * N), (D, C)))
        self.dt_proj_weight, self.dt_bias, self.A_log, self.D = p(D, R), p(D), p(D, N), p(D)


def oracle_block(m, x, residual, state, lengths=None):
    h, residual = O.rms_norm(x, m.norm_weight, m.eps, residual)
    u, z = m.in_proj(h).chunk(2, -1)
    u, window = O.causal_conv(u, m.conv_weight, m.conv_bias, state[0], lengths)
    N, R = m.A_log.shape[1], m.dt_proj_weight.shape[1]
    low, b, c = m.x_proj(u).split([R, N, N], -1)
    y, h = O.selective_scan(u, low @ m.dt_proj_weight.t(), -torch.exp(m.A_log), b, c, m.D, z, m.dt_bias, state[1], lengths)
    return m.out_proj(y), residual, (window, h)


@pytest.mark.parametrize("T,lengths", [(1, None), (33, None), (33, [33, 0, 20])])
def test_block_and_its_gradients(T, lengths):
    """fp32, 3 sequences; the projections are torch's on both sides.  1e-3 of |ref| + rms: the products' and kernels' fp32 rounding through
    the block's six steps, a few 2^-23 each times sums of up to 100 terms, taken generously."""
    from rwkv_wkv_hip import ssm as K
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g)
    ref, got = Block().double(), Block().cuda()
    got.load_state_dict(ref.state_dict())
    x, residual, state = r(3, T, 24), r(3, T, 24), (r(3, 3, 40), r(3, 40, 16))
    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)

    def run(f, m, to):
        leaves = [to(t).requires_grad_(True) for t in (x, residual, *state)]
        out, res, new = f(m, leaves[0], leaves[1], (leaves[2], leaves[3]), L if L is None else L.to(leaves[0].device))
        w = torch.Generator().manual_seed(3)
        loss = sum((o * to(torch.randn(o.shape, generator=w))).sum() for o in (out, res, *new))
        loss.backward()
        return [out, res, *new, *(t.grad for t in leaves), *(p.grad for p in m.parameters())]

    for a, b in zip(run(K.block_forward, got, lambda t: t.cuda()), run(oracle_block, ref, lambda t: t.double())):
        assert_close(a, b, 1e-3)


def test_block_token_by_token_is_the_prompt():
    from rwkv_wkv_hip import ssm as K
    m = Block().cuda()
    x, residual = torch.randn(2, 9, 24, device="cuda"), torch.randn(2, 9, 24, device="cuda")
    with torch.no_grad():
        start = K.block_state(m, 2, torch.float32)
        whole, sums, end = K.block_forward(m, x, residual, start)
        state, rows = start, []
        for t in range(9):
            out, _, state = K.block_forward(m, x[:, t:t + 1], residual[:, t:t + 1], state)
            rows.append(out)
    assert_close(torch.cat(rows, 1), whole, 1e-3)
    assert_close(sums, x + residual, 1e-6)
    for a, b in zip(state, end):
        assert_close(a, b, 1e-3)


def test_example_learns_and_serves():
    import state_space_lm as E
    torch.manual_seed(0)
    g = torch.Generator(device="cuda").manual_seed(0)
    model = E.Model().cuda()
    losses = E.train(model, 40, generator=g, report=None)
    assert losses[-1] < 0.5 * losses[0]
    written, logprobs = E.serve(model, [[1], [5, 28, 143], list(range(20))], 6, temperature=torch.tensor([0.0, 0.8, 1.0], device="cuda"), generator=g)
    assert written.shape == (3, 6) and bool(((written >= 0) & (written < E.VOCABULARY)).all())
    assert bool((logprobs <= 0).all()) and bool((logprobs[0] == 0).all())


def test_traced():
    """torch.jit.trace records the operators as nodes that run again on the inputs the graph is given."""
    from rwkv_wkv_hip import ssm as K
    class Part(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.m = Block()

        def forward(self, x, dt, b, c):
            u, _ = K.causal_conv(x, self.m.conv_weight, self.m.conv_bias)
            y, s = K.selective_scan(u, dt, -torch.exp(self.m.A_log), b, c, D=self.m.D)
            return K.rms_norm(y, self.m.D)[0], s

    f = Part().cuda()
    r = lambda *s: torch.randn(*s, device="cuda")
    inputs, other = ((r(2, 7, 40), r(2, 7, 40), r(2, 7, 16), r(2, 7, 16)) for _ in range(2))
    with torch.no_grad():
        traced = torch.jit.trace(f, inputs, check_trace=False)
        for got, want in zip(traced(*other), f(*other)):
            assert torch.equal(got, want)
