"""The gated recurrence block on the package's operators against the same block on the oracle's, and the example that trains and serves it."""
import os
import sys

import pytest
import torch

from oracle import gated as O
from oracle import ssm as OS
from tests.util import assert_close

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
VOCABULARY = 17


class Block(torch.nn.Module):
    def __init__(self, C=24, D=40, F=56, W=4, eps=1e-5):
        super().__init__()
        g = torch.Generator().manual_seed(1)
        p = lambda *s, std=0.3: torch.nn.Parameter(torch.randn(*s, generator=g) * std)
        self.eps, self.activation, self.norm_weight, self.ff_norm_weight = eps, "gelu", p(C, std=1.0), p(C, std=1.0)
        self.conv_weight, self.conv_bias, self.decay = p(D, W), p(D), p(D, std=1.0)
        self.in_proj, self.gate_proj, self.out_proj, self.ff_down = (torch.nn.Linear(i, o, bias=False) for i, o in ((C, 2 * D), (D, 2 * D), (D, C), (F, C)))
        self.ff_gate, self.ff_up, self.table = p(F, C), p(F, C), p(VOCABULARY, C, std=1.0)


def oracle_block(m, x, residual, state, lengths=None):
    h, residual = OS.rms_norm(x, m.norm_weight, m.eps, residual)
    u, z = m.in_proj(h).chunk(2, -1)
    u, window = OS.causal_conv(u, m.conv_weight, m.conv_bias, state[0], lengths, silu=False)
    r, i = m.gate_proj(u).chunk(2, -1)
    y, h = O.gated_recurrence(u, r, i, m.decay, z, state[1], lengths)
    n, residual = OS.rms_norm(m.out_proj(y), m.ff_norm_weight, m.eps, residual)
    return m.ff_down(O.gated_feed_forward(n, m.ff_gate, m.ff_up, m.activation)), residual, (window, h)


@pytest.mark.parametrize("T,lengths", [(1, None), (33, None), (70, [70, 0, 20])])
def test_block_and_its_gradients(T, lengths):
    """fp32, 3 sequences, from tokens (some of them padding) through the lookup and the block; the projections are torch's on both sides.  1e-3 of |ref| + rms: the
    products' and kernels' fp32 rounding through the block's eight steps, a few 2^-23 each times sums of up to 100 terms, taken generously."""
    from rwkv_wkv_hip import gated as K
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g)
    ref, got = Block().double(), Block().cuda()
    got.load_state_dict(ref.state_dict())
    tokens = torch.randint(-1, VOCABULARY, (3, T), generator=g)
    residual, state = r(3, T, 24), (r(3, 3, 40), r(3, 40))
    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)

    def run(lookup, f, m, to):
        leaves = [to(t).requires_grad_(True) for t in (residual, *state)]
        there = leaves[0].device
        x = lookup(tokens.to(there), m.table, 24 ** 0.5)
        out, res, new = f(m, x, leaves[0], (leaves[1], leaves[2]), L if L is None else L.to(there))
        w = torch.Generator().manual_seed(3)
        loss = sum((o * to(torch.randn(o.shape, generator=w))).sum() for o in (out, res, *new))
        loss.backward()
        return [out, res, *new, *(t.grad for t in leaves), *(p.grad for p in m.parameters())]

    for a, b in zip(run(K.embedding, K.block_forward, got, lambda t: t.cuda()), run(O.embedding, oracle_block, ref, lambda t: t.double())):
        assert_close(a, b, 1e-3)


def test_block_token_by_token_is_the_prompt():
    from rwkv_wkv_hip import gated as K
    m = Block().cuda()
    tokens, residual = torch.randint(-1, VOCABULARY, (2, 9), device="cuda"), torch.randn(2, 9, 24, device="cuda")
    with torch.no_grad():
        x = K.embedding(tokens, m.table)
        start = K.block_state(m, 2, torch.float32)
        whole, sums, end = K.block_forward(m, x, residual, start)
        state, rows = start, []
        for t in range(9):
            out, s, state = K.block_forward(m, K.embedding(tokens[:, t:t + 1], m.table), residual[:, t:t + 1], state)
            assert_close(s, sums[:, t:t + 1], 1e-3)
            rows.append(out)
    assert_close(torch.cat(rows, 1), whole, 1e-3)
    for a, b in zip(state, end):
        assert_close(a, b, 1e-3)


def test_example_trains_and_serves():
    """It runs, every parameter has a finite gradient, and what it writes are tokens."""
    import gated_recurrence_lm as E
    torch.manual_seed(0)
    g = torch.Generator(device="cuda").manual_seed(0)
    model = E.Model().cuda()
    losses = E.train(model, 3, generator=g, report=None)
    assert len(losses) == 3 and all(map(torch.isfinite, map(torch.tensor, losses)))
    for n, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any(), n
    written, logprobs = E.serve(model, [[1], [5, 28, 143], list(range(20))], 6, temperature=torch.tensor([0.0, 0.8, 1.0], device="cuda"), generator=g)
    assert written.shape == (3, 6) and bool(((written >= 0) & (written < E.VOCABULARY)).all())
    assert bool((logprobs <= 0).all()) and bool((logprobs[0] == 0).all())


def test_traced():
    """torch.jit.trace records the operators as nodes that run again on the inputs the graph is given."""
    from rwkv_wkv_hip import gated as K

    class Part(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.m = Block()

        def forward(self, tokens, r, i):
            y, s = K.gated_recurrence(K.embedding(tokens, self.m.table, 2.0), r, i, self.m.norm_weight)
            return K.gated_feed_forward(y, self.m.ff_gate, self.m.ff_up, "relu"), s

    f = Part().cuda()
    r = lambda *s: torch.randn(*s, device="cuda")
    t = lambda: torch.randint(0, VOCABULARY, (2, 7), device="cuda")
    inputs, other = ((t(), r(2, 7, 24), r(2, 7, 24)) for _ in range(2))
    with torch.no_grad():
        traced = torch.jit.trace(f, inputs, check_trace=False)
        for got, want in zip(traced(*other), f(*other)):
            assert torch.equal(got, want)
