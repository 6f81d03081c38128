"""Sampling on the HIP kernel against the oracle (oracle/ssm.py).  Tokens are compared as they are: the sums are of whole numbers.  (The one thing
that may differ is the last bit of a weight, one part in 2^24 of it; a token moves by that only if u lies as near to a boundary.)"""
import math

import pytest
import torch

from oracle import ssm as O

pytestmark = pytest.mark.gpu


def _check(logits, u, **k):
    from rwkv_wkv_hip.sampling import sample
    B = logits.shape[0]
    rows = {n: k.get(n, d) for n, d in dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0).items()}
    token, logprob = sample(logits.cuda(), u.cuda(), **{n: v.cuda() if torch.is_tensor(v) else v for n, v in rows.items()})
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32
    at = lambda v, b: v[b].item() if torch.is_tensor(v) else v
    for b in range(B):
        t, p, kept = O.sample(logits[b].float(), float(u[b]), *(at(rows[n], b) for n in ("temperature", "top_k", "top_p", "min_p")))
        assert int(token[b]) == t, (b, int(token[b]), t, len(kept))
        assert (float(logprob[b]) == p) if math.isinf(p) else abs(float(logprob[b]) - p) <= 1e-6 + 1e-6 * abs(p)


def _logits(dtype, B, V, seed, scale=2.0):
    return (torch.randn(B, V, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 7, 1000, 8192, 8193, 20001])
@pytest.mark.parametrize("k", [dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
                               dict(temperature=0.7, top_k=50, top_p=0.8, min_p=0.02), dict(top_k=1), dict(top_p=0.0)])
def test_settings(dtype, V, k):
    _check(_logits(dtype, 3, V, V), torch.tensor([0.0, 0.37, 0.99999]), **k)


def test_settings_per_row():
    B, V = 24, 5003
    g = torch.Generator().manual_seed(4)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (B,), generator=g)]
    for dtype in (torch.float32, torch.bfloat16):
        _check(_logits(dtype, B, V, 5), torch.rand(B, generator=g), temperature=pick(0.0, 0.5, 1.0, 1.7), top_k=pick(0, 1, 40, 3000), top_p=pick(1.0, 0.3, 0.95), min_p=pick(0.0, 0.05))


@pytest.mark.parametrize("V", [65536, 50277, 131072, 300001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_whole_vocabularies(dtype, V):
    _check(_logits(dtype, 2, V, V), torch.tensor([0.21, 0.83]), temperature=0.8, top_k=200, top_p=0.9)
    _check(_logits(dtype, 2, V, V + 1), torch.tensor([0.55, 0.02]), top_p=0.97)


@pytest.mark.parametrize("V", [100, 10000, 70000])
def test_ties_go_to_the_lowest_index(V):
    """All equal, and a few values over many tokens: the cuts fall among equals."""
    same = torch.full((3, V), 1.25)
    u = torch.tensor([0.0, 0.5, 0.999])
    _check(same, u, top_k=17)
    _check(same, u, top_p=0.31)
    _check(same, u, temperature=0.0)
    few = torch.randint(0, 4, (3, V), generator=torch.Generator().manual_seed(V)).float()
    _check(few, u, top_k=V // 3)
    _check(few, u, top_p=0.4)
    _check(few, u, top_k=V // 2, top_p=0.77)


@pytest.mark.parametrize("V", [1000, 9000])
def test_nearly_equal_logits(V):
    """Thousands of different values within one bin of the search."""
    l = 1.0 + torch.randperm(V, generator=torch.Generator().manual_seed(V))[None].float() * 2.0 ** -23
    _check(l, torch.tensor([0.4]), top_k=V // 3)
    _check(l, torch.tensor([0.4]), top_p=0.6)


def test_masked_and_non_finite_logits():
    inf, nan = math.inf, math.nan
    l = torch.tensor([[-inf, 1.0, -inf, 2.0, nan], [-inf] * 5, [nan] * 5, [-inf, -inf, 3.0, -inf, -inf], [inf, 0.0, inf, 1.0, -inf],
                      [torch.finfo(torch.float32).min] * 5, [torch.finfo(torch.float32).min, 0.0, 0.0, -100.0, nan]])
    u = torch.tensor([0.9, 0.5, 0.5, 0.0, 0.7, 0.5, 0.6])
    for k in (dict(), dict(top_k=2), dict(top_p=0.5), dict(temperature=0.0), dict(min_p=1.0)):
        _check(l, u, **k)
    _check(-l.abs().nan_to_num(0.0) * 0.0, u, top_k=2)          # zeros of both signs


def test_strided_rows_and_broadcast_logits():
    wide = _logits(torch.bfloat16, 4, 3001, 9)
    from rwkv_wkv_hip.sampling import sample
    u = torch.tensor([0.1, 0.4, 0.6, 0.9])
    part = wide.cuda()[:, 1:2000]
    want = sample(part.contiguous(), u.cuda(), top_p=0.9)
    got = sample(part, u.cuda(), top_p=0.9)
    turned = sample(part.t().contiguous().t(), u.cuda(), top_p=0.9)
    one = sample(part[:1].expand(4, -1), u.cuda(), top_p=0.9)
    assert torch.equal(want[0], got[0]) and torch.equal(want[0], turned[0]) and torch.equal(one[0][0], want[0][0])
    _check(wide[:1, 1:2000].expand(4, -1), u, top_p=0.9)


def test_frequencies():
    """20000 random numbers in even steps give every token its share to within a step or two."""
    from rwkv_wkv_hip.sampling import sample
    n = 20000
    l = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.0])
    token, _ = sample(l.expand(n, -1).cuda(), ((torch.arange(n) + 0.5) / n).cuda(), temperature=0.9)
    share = torch.bincount(token.cpu(), minlength=5).double() / n
    assert (share - torch.softmax(l.double() / 0.9, 0)).abs().max() < 2 / n


def test_refusals():
    import rwkv_wkv_hip as W
    z = lambda *s: torch.zeros(*s, device="cuda")
    S = W.sampling.sample
    with pytest.raises(AssertionError):
        S(z(3), z(3))
    with pytest.raises(AssertionError):
        S(z(2, 5), z(3))
    with pytest.raises(AssertionError):
        S(z(2, 5), z(2), top_k=z(3))
    with pytest.raises(W.WKVError):
        S(z(2, 5), z(2).cpu())
    with pytest.raises(AssertionError):
        S(z(2, 5), z(2), temperature=torch.ones(2))
    with pytest.raises(ValueError):
        S(z(2, 5).double(), z(2))
    with pytest.raises(ValueError):
        S(z(1, 1).expand(1, (1 << 20) + 1), z(1))
    with pytest.raises(ValueError):
        S(z(0, 5), z(0))
