"""The oracle of a gated recurrence model's operators against forms that are written down independently of it."""
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import gated as O

D64 = torch.float64


def test_recurrence_is_the_geometric_series():
    """Constant inputs: h[t] = beta sigmoid(i) x (1 - a^(t+1)) / (1 - a)."""
    T, x, r, i, decay, scale = 9, 1.5, 0.3, -0.2, -0.7, 2.0
    one = lambda v, *s: torch.full(s, v, dtype=D64)
    y, h = O.gated_recurrence(one(x, 1, T, 1), one(r, 1, T, 1), one(i, 1, T, 1), one(decay, 1), scale=scale)
    sig = lambda v: 1 / (1 + math.exp(-v))
    a = math.exp(-scale * math.log1p(math.exp(decay)) * sig(r))
    want = [math.sqrt(1 - a * a) * sig(i) * x * (1 - a ** (t + 1)) / (1 - a) for t in range(T)]
    assert torch.allclose(y[0, :, 0], torch.tensor(want, dtype=D64), rtol=1e-12) and math.isclose(float(h), want[-1], rel_tol=1e-12)


def test_recurrence_chains_through_its_state():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=D64)
    B, T, D = 2, 7, 5
    x, a, i, z, decay, s0 = r(B, T, D), r(B, T, D), r(B, T, D), r(B, T, D), r(D), r(B, D)
    whole = O.gated_recurrence(x, a, i, decay, z, s0)
    cut = lambda s: [v[:, s] for v in (x, a, i)]
    first = O.gated_recurrence(*cut(slice(0, 3)), decay, z[:, :3], s0)
    second = O.gated_recurrence(*cut(slice(3, T)), decay, z[:, 3:], first[1])
    assert torch.allclose(whole[0], torch.cat([first[0], second[0]], 1)) and torch.allclose(whole[1], second[1])
    short = O.gated_recurrence(x, a, i, decay, z, s0, lengths=[3, 0])
    assert torch.equal(short[1][0], first[1][0]) and torch.equal(short[1][1], s0[1]) and not short[0][1].any()
    assert torch.allclose(O.gated_recurrence(x, a, i, decay, None, s0)[0] * F.silu(z), whole[0])
    # a shut gate keeps the state, an infinite decay forgets it
    assert torch.equal(O.gated_recurrence(x, torch.full_like(a, -math.inf), i, decay, None, s0)[1], s0)
    assert torch.allclose(O.gated_recurrence(x, a, i, torch.full_like(decay, 1e4), None, s0)[1], torch.sigmoid(i[:, -1]) * x[:, -1])


def test_activations_and_lookup():
    g = torch.linspace(-6, 6, 101, dtype=D64)
    assert torch.allclose(O.activation("silu", g), F.silu(g)) and torch.allclose(O.activation("gelu", g), F.gelu(g, approximate="tanh"))
    assert torch.equal(O.activation("relu", g), F.relu(g))
    w, t = torch.randn(6, 4, dtype=D64, generator=torch.Generator().manual_seed(2)), torch.tensor([[0, 5, 5], [-1, 6, 2]])
    one_hot = F.one_hot(t.clamp(0, 5), 6).double() * ((t >= 0) & (t < 6))[..., None]
    assert torch.allclose(O.embedding(t, w, 3.0), 3.0 * one_hot @ w)


@pytest.mark.parametrize("lengths", [None, [4, 1, 0]])
def test_gradients_are_differences(lengths):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=D64).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x, a, i, d, z, s: O.gated_recurrence(x, a, i, d, z, s, lengths), (r(3, 4, 2), r(3, 4, 2), r(3, 4, 2), r(2), r(3, 4, 2), r(3, 2)))
    assert torch.autograd.gradcheck(lambda x, a, b: O.gated_feed_forward(x, a, b, "gelu"), (r(3, 4), r(5, 4), r(5, 4)))
    assert torch.autograd.gradcheck(lambda w: O.embedding(torch.tensor([1, 1, -1, 0]), w, 0.5), (r(3, 2),))
