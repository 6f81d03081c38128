"""The oracle of the state space operators and of sampling against forms that are written down independently of it."""
import math

import pytest
import torch

from oracle import ssm as O


def test_scan_is_the_geometric_series():
    """One state, constant inputs: h[t] = step x B (1 - a^t) / (1 - a)."""
    T, x, raw, A, b, c = 9, 1.5, 0.3, -0.7, 0.4, 2.0
    one = lambda v, *s: torch.full(s, v, dtype=torch.float64)
    y, h = O.selective_scan(one(x, 1, T, 1), one(raw, 1, T, 1), one(A, 1, 1), one(b, 1, T, 1), one(c, 1, T, 1))
    step = math.log1p(math.exp(raw))
    a = math.exp(step * A)
    want = [step * x * b * (1 - a ** (t + 1)) / (1 - a) for t in range(T)]
    assert torch.allclose(y[0, :, 0], c * torch.tensor(want, dtype=torch.float64), rtol=1e-12)
    assert math.isclose(float(h), want[-1], rel_tol=1e-12)


def test_scan_and_convolution_chain_through_their_states():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    B, T, D, N, G, W = 2, 7, 6, 3, 2, 4
    x, dt, z, A, b, c, s0 = r(B, T, D), r(B, T, D), r(B, T, D), -r(D, N).abs(), r(B, T, G, N), r(B, T, G, N), r(B, D, N)
    whole = O.selective_scan(x, dt, A, b, c, z=z, state=s0)
    first = O.selective_scan(x[:, :3], dt[:, :3], A, b[:, :3], c[:, :3], z=z[:, :3], state=s0)
    second = O.selective_scan(x[:, 3:], dt[:, 3:], A, b[:, 3:], c[:, 3:], z=z[:, 3:], state=first[1])
    assert torch.allclose(whole[0], torch.cat([first[0], second[0]], 1)) and torch.allclose(whole[1], second[1])
    short = O.selective_scan(x, dt, A, b, c, z=z, state=s0, lengths=[3, 0])
    assert torch.equal(short[1][0], first[1][0]) and torch.equal(short[1][1], s0[1]) and not short[0][1].any()
    w, w0 = r(D, W), r(B, W - 1, D)
    y, s = O.causal_conv(x, w, None, w0, silu=False)
    padded = torch.cat([w0, x], 1).transpose(1, 2)
    assert torch.allclose(y, torch.nn.functional.conv1d(padded, w.unsqueeze(1), groups=D).transpose(1, 2))
    assert torch.equal(s, x[:, -(W - 1):]) and torch.equal(O.causal_conv(x, w, None, w0, lengths=[1, 0])[1][1], w0[1])


def test_norm_of_equal_elements():
    y, r = O.rms_norm(torch.full((2, 8), 3.0, dtype=torch.float64), torch.arange(8.0, dtype=torch.float64), 0.0, torch.full((2, 8), -1.0, dtype=torch.float64))
    assert torch.equal(r, torch.full((2, 8), 2.0, dtype=torch.float64)) and torch.allclose(y, torch.arange(8.0, dtype=torch.float64).expand(2, 8))


def test_sampling_cuts_by_hand():
    l = torch.log(torch.tensor([0.1, 0.4, 0.2, 0.2, 0.1]))
    assert O.sample(l, 0.0, 1.0, 0, 1.0, 0.0)[2] == [0, 1, 2, 3, 4]
    assert O.sample(l, 0.0, 1.0, 2, 1.0, 0.0)[2] == [1, 2]                # the tie goes to the lower index
    assert O.sample(l, 0.0, 1.0, 0, 0.61, 0.0)[2] == [1, 2, 3]
    assert O.sample(l, 0.0, 1.0, 0, 1.0, 0.4)[2] == [1, 2, 3]
    assert O.sample(l, 0.9, 0.0, 0, 1.0, 0.0)[:2] == (1, 0.0)
    assert O.sample(torch.full((3,), -math.inf), 0.5, 1.0, 0, 1.0, 0.0)[0] == -1


@pytest.mark.parametrize("temperature", [0.7, 1.0])
def test_sampling_frequencies(temperature):
    l = torch.tensor([0.3, -1.0, 2.0, 0.0])
    n = 2000
    tokens = [O.sample(l, (i + 0.5) / n, temperature, 0, 1.0, 0.0)[0] for i in range(n)]
    p = torch.softmax(l.double() / temperature, 0)
    for i in range(4):
        assert abs(tokens.count(i) / n - float(p[i])) < 1.5 / n
