"""The operators of a gated recurrence model where fp32 arithmetic or a 16-bit type's range could lose what a result is made of: every element by the size of its own terms, not by the
tensor's.  The oracle is that of test_gpu_gated.py, in 64 bits."""
import pytest
import torch

from tests import test_gpu_gated as S

pytestmark = pytest.mark.gpu


def _kernels():
    from rwkv_wkv_hip import gated
    return gated


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 65, 300])
@pytest.mark.parametrize("decay", [0.0, 1.0, 2.0, 3.0])
@pytest.mark.parametrize("gate", [False, True])
def test_gradients_of_what_forgets_at_once(dtype, T, decay, gate):
    """A sequence of one token without a state: all of log a's slope comes by way of sqrt(1 - a^2), as a^2 / (1 - a^2) times the input, however small a is.

    Every element of gr and gdecay is one product, so it is right to the sum of its factors' errors.  In fp32 a sigmoid or a decay's rate is off by 4 x 2^-23 (the
    exponential, the sum, the reciprocal or logarithm, the product); log a by both, 2^-20 of its size; a^2 by twice that times |log a|.  1 - sigmoid(r) is off by
    2^-21 / (1 - sigmoid(r)).  The other eight factors and products: 8 x 2^-20 at most.  bf16 inputs are those of the 64-bit formula too; its gr is rounded once more (2^-8).

    The values are the formula's, written out: autograd through the oracle forms exp(2 log a) as expm1(2 log a) + 1, and that has as few digits in 64 bits."""
    D, scale = 257, 8.0
    g = S._g(T, int(decay * 10), gate)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    v = dict(x=r(1, T, D), r=r(1, T, D).clamp(-4, 4), i=r(1, T, D), decay=decay + torch.randn(D, generator=g) * 0.1)
    if gate:
        v["z"] = r(1, T, D)
    if T > 1:
        v["lengths"] = torch.ones(1, dtype=torch.int32)
    gy = r(1, T, D)
    got = S._cuda(v)
    out, _ = _kernels().gated_recurrence(scale=scale, **got)
    out.backward(gy.cuda())
    first = lambda t: t.double()[0, 0]
    s, soft, through = torch.sigmoid(first(v["r"])), torch.nn.functional.softplus(v["decay"].double()), torch.sigmoid(first(v["i"])) * first(v["x"])
    log_a = -scale * soft * s
    beta = torch.sqrt(-torch.expm1(2 * log_a))
    glog = -first(gy) * torch.exp(2 * log_a) / beta * through          # by log a: d beta / d log a = -a^2 / beta
    if gate:
        glog = glog * first(v["z"]) * torch.sigmoid(first(v["z"]))
    want = dict(r=glog * log_a * (1 - s), decay=glog * s * -scale * torch.sigmoid(v["decay"].double()))
    log_a = log_a.abs()
    off = 2.0 ** -20 * (2 * log_a + 8 + 1 / (1 - s))
    for n, more in (("r", S._step(dtype)), ("decay", 0.0)):
        a, b = got[n].grad.cpu().double(), want[n]
        if n == "r":
            assert not a[0, 1:].any()
            a = a[0, 0]
        worst = ((a - b).abs() / ((off + more) * b.abs() * (1 + off))).max().item()
        assert worst <= 1, f"gradient of {n}: {worst:.3g} of the bound"
