"""The operators of a gated recurrence model on the HIP kernels against the oracle in 64 bits (oracle/gated.py, gradients by autograd through it).

Tolerances.  The oracle has the same (rounded) inputs in 64 bits.  The recurrence, of |ref| + rms(ref) per element: an output's rounding, half a step (bf16 2^-8,
fp16 2^-11, taken twice), and fp32 arithmetic: a decay is right to a few 2^-23, a state over the few hundred tokens that it remembers to
at most their sum, some 5e-5, taken twice.  The products and the lookup by bounds of their own, written at each."""
import math

import pytest
import torch

from oracle import gated as O
from tests.util import assert_close

pytestmark = pytest.mark.gpu
RTOL = {torch.float32: 1e-4, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _g(*seed):
    n = 23
    for s in seed:
        n = n * 1009 + int(s)
    return torch.Generator().manual_seed(n % (1 << 31))


def _double(v):
    return {n: t.double().requires_grad_(True) if torch.is_tensor(t) and t.is_floating_point() else t for n, t in v.items()}


def _cuda(v, leaf=True):
    return {n: t.cuda().requires_grad_(leaf and t.is_floating_point()) if torch.is_tensor(t) else t for n, t in v.items()}


def compare(kernel, oracle, v, grads, names):
    """Outputs and gradients of both, each within its type's tolerance."""
    want, got = _double(v), _cuda(v)
    ref, out = oracle(**want), kernel(**got)
    for a, b, n in zip(out, ref, names):
        assert torch.isfinite(a).all()
        assert_close(a, b, RTOL[a.dtype], n)
    torch.autograd.backward(list(ref), [g.double() for g in grads])
    torch.autograd.backward(list(out), [g.cuda() for g in grads])
    torch.cuda.synchronize()
    for n, t in got.items():
        if torch.is_tensor(t) and t.requires_grad:
            assert t.grad.dtype == t.dtype and t.grad.shape == t.shape
            assert_close(t.grad, want[n].grad, RTOL[t.dtype], "gradient of " + n)


# ---- the recurrence
def recurrence_inputs(dtype, B, T, D, gate=True, state=True, lengths=None):
    g = _g(B, T, D)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    v = dict(x=r(B, T, D), r=r(B, T, D), i=r(B, T, D), decay=torch.randn(D, generator=g) * 2 - 4)
    if gate:
        v["z"] = r(B, T, D)
    if state:
        v["state"] = torch.randn(B, D, generator=g)
    if lengths is not None:
        v["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    return v, [r(B, T, D), torch.randn(B, D, generator=g)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1, 64), (2, 2, 5), (1, 8, 130), (3, 9, 1), (1, 63, 128), (2, 64, 33), (1, 65, 256), (2, 128, 40), (1, 129, 127), (1, 300, 64), (2, 777, 18)])
def test_recurrence(dtype, B, T, D):
    from rwkv_wkv_hip import gated as K
    v, grads = recurrence_inputs(dtype, B, T, D)
    compare(K.gated_recurrence, O.gated_recurrence, v, grads, ("y", "state"))


@pytest.mark.parametrize("options", [dict(gate=False), dict(state=False), dict(gate=False, state=False)])
@pytest.mark.parametrize("T,D", [(1, 24), (37, 24), (270, 24), (270, 23)])
def test_recurrence_options(options, T, D):
    from rwkv_wkv_hip import gated as K
    v, grads = recurrence_inputs(torch.float32, 2, T, D, **options)
    compare(lambda **k: K.gated_recurrence(scale=3.0, **k), lambda **k: O.gated_recurrence(scale=3.0, **k), v, grads, ("y", "state"))


@pytest.mark.parametrize("T,lengths", [(300, [0, 1, 300]), (300, [64, 129, 255]), (1400, [1399, 0, 600]), (40, [39, 0, 20]), (1, [0, 1, 1])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_recurrence_lengths(T, lengths, dtype):
    """What lies behind a sequence's end is not read: there it is NaN on the GPU, zero in the oracle."""
    from rwkv_wkv_hip import gated as K
    v, grads = recurrence_inputs(dtype, 3, T, 18, lengths=lengths)
    behind = (torch.arange(T)[None, :, None] >= v["lengths"][:, None, None]).cuda()

    def kernel(x, r, i, z, **k):
        spoil = lambda t: torch.where(behind, torch.nan, t)
        return K.gated_recurrence(spoil(x), spoil(r), spoil(i), z=spoil(z), **k)

    compare(kernel, O.gated_recurrence, v, grads, ("y", "state"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D", [(1, 8), (3, 37), (64, 200)])
@pytest.mark.parametrize("lengths", [False, True])
def test_recurrence_of_a_single_token(dtype, B, D, lengths):
    """The kernel of its own, also with the state updated in place."""
    from rwkv_wkv_hip import gated as K
    v, _ = recurrence_inputs(dtype, B, 1, D, lengths=[b % 2 for b in range(B)] if lengths else None)
    ref = O.gated_recurrence(**{n: t.double() if t.is_floating_point() else t for n, t in v.items()})
    c = _cuda(v, leaf=False)
    before = c["state"].clone()
    for out in K.gated_recurrence(**c), K.gated_recurrence(**c, out_state=c["state"]):
        for a, b in zip(out, ref):
            assert_close(a, b, RTOL[a.dtype])
    assert out[1] is c["state"] and (lengths or not torch.equal(before, c["state"]))


# ---- the gated feed-forward
def _step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0


def check_feed_forward(x, wg, wu, gy, name, out, grads):
    """Per element.  With e the half step of the type (0 in fp32: it is in c) and c = (terms + 32) 2^-23 for fp32 sums of that many terms and a few operations
    after them, a sum is off by c times its terms' sizes G, U; the activations' slopes and the slopes' slopes are below 1.2.  A gradient's sum takes
    dg and du rounded (e) and off by what g and u were off; relu's slope is anything where g may be zero."""
    d = lambda t: t.detach().double()          # (on the GPU: the library's products in 64 bits)
    x, wg, wu, gy = d(x), d(wg), d(wu), d(gy)
    e = _step(out.dtype)
    leaf = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
    ref = O.gated_feed_forward(*leaf, name)
    want = torch.autograd.grad(ref, leaf, gy)
    c = (x.shape[1] + 32) * 2.0 ** -23
    g, u = (x @ wg.t()).requires_grad_(True), x @ wu.t()
    G, U, act = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t(), O.activation(name, g)
    (slope,) = torch.autograd.grad(act.sum(), g)
    act, g = act.detach(), g.detach()
    off = 1.2 * c * (G * u.abs() + U * act.abs()) + 1.5 * c * c * G * U
    assert bool(((d(out) - ref).abs() <= (e + 2.0 ** -20) * ref.abs() + (1 + e) * off + 2.0 ** -24).all())
    # dg, du: their sizes and what they may be off
    sg, su = (gy * u * slope).abs(), (gy * act).abs()
    og = gy.abs() * 1.2 * c * (U + G * u.abs() + c * G * U) + 2.0 ** -20 * (gy * u).abs()
    if name == "relu":
        og = og + torch.where(g.abs() <= c * G, (gy * u).abs(), 0.0)
    ou = gy.abs() * 1.2 * c * G + 2.0 ** -20 * (gy * G).abs() * 0.1
    for got, ref_, size, wrong, terms in ((grads[0], want[0], sg @ wg.abs() + su @ wu.abs(), og @ wg.abs() + ou @ wu.abs(), 2 * wg.shape[0]),
                                          (grads[1], want[1], sg.t() @ x.abs(), og.t() @ x.abs(), len(x)), (grads[2], want[2], su.t() @ x.abs(), ou.t() @ x.abs(), len(x))):
        bound = e * ref_.abs() + (1 + e) * ((e + (terms + 32) * 2.0 ** -23) * size + (1 + e) * wrong) + 2.0 ** -24
        assert got.shape == ref_.shape and bool(((d(got) - ref_).abs() <= bound).all()), ((d(got) - ref_).abs() / bound).max()


def feed_forward(dtype, R, C, F, name, shape=None):
    from rwkv_wkv_hip import gated as K
    g = _g(R, C, F)
    x = torch.randn(R, C, generator=g).to(dtype).cuda().view(*(shape or (R,)), C)
    wg, wu = (torch.randn(F, C, generator=g).mul(C ** -0.5).to(dtype).cuda() for _ in range(2))
    gy = torch.randn(R, F, generator=g).to(dtype).cuda()
    leaf = [t.requires_grad_(True) for t in (x, wg, wu)]
    out = K.gated_feed_forward(*leaf, name)
    grads = torch.autograd.grad(out, leaf, gy.view_as(out))
    with torch.no_grad():
        assert torch.equal(out, K.gated_feed_forward(*leaf, name))
    assert out.shape == (*x.shape[:-1], F) and all(a.shape == b.shape and a.dtype == dtype for a, b in zip(grads, leaf))
    check_feed_forward(x.reshape(R, C), wg, wu, gy, name, out.view(R, F), (grads[0].view(R, C), *grads[1:]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C,F,name", [(1, 64, 16, "silu"), (3, 104, 40, "gelu"), (16, 256, 200, "relu"), (17, 72, 130, "silu"), (33, 1000, 333, "silu"), (64, 40, 65, "gelu"),
                                        (65, 64, 64, "silu"), (130, 104, 131, "gelu"), (257, 520, 640, "silu"), (300, 1001, 271, "relu"), (5, 33, 7, "gelu"),
                                        (70, 1, 1, "silu"), (1, 1, 1, "gelu"), (513, 136, 900, "relu")])
def test_feed_forward(dtype, R, C, F, name):
    feed_forward(dtype, R, C, F, name)


def test_feed_forward_of_more_dimensions():
    feed_forward(torch.bfloat16, 2 * 3 * 7, 48, 33, "silu", shape=(2, 3, 7))


# ---- the lookup
def check_lookup(tokens, weight, scale, gy, out, grad):
    """An output: one rounding of a fp32 product.  A gradient of n places: n fp32 sums and a product, and its rounding.  Below a type's smallest normal number
    steps no longer shrink with the value: half a step there is smallest_normal eps / 2 (fp16 2^-14 2^-11 = 2^-25)."""
    V, e = len(weight), max(_step(out.dtype), 2.0 ** -24)
    least = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps / 2
    t = tokens.cpu().flatten()
    ok = (t >= 0) & (t < V)
    w, g = weight.detach().cpu().double(), torch.where(ok[:, None], gy.cpu().double().reshape(len(t), -1), 0.0)
    ref = torch.where(ok[:, None], scale * w[t.clamp(0, V - 1)], 0.0)
    assert bool(((out.detach().cpu().double().reshape_as(ref) - ref).abs() <= (e + 2.0 ** -23) * ref.abs() + least).all())
    at = t.clamp(0, V - 1).long()
    total, size = torch.zeros_like(w).index_add_(0, at, g) * scale, torch.zeros_like(w).index_add_(0, at, g.abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64).index_add_(0, at, ok.double())[:, None]
    bound = e * total.abs() + (1 + e) * (n + 2) * 2.0 ** -24 * size + least
    assert bool(((grad.cpu().double() - total).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("n,V,C", [(1, 1, 1), (7, 3, 8), (64, 1000, 64), (200, 50, 33), (4096, 70, 24), (4097, 1023, 16), (9000, 1024, 40), (5000, 70001, 8), (12300, 5, 130)])
def test_embedding(dtype, index, n, V, C):
    from rwkv_wkv_hip import gated as K
    g = _g(n, V, C)
    tokens = torch.randint(-1, V + 1, (n,), generator=g).to(index)
    tokens[n // 3: n // 2] = V - 1                 # many of one
    w, gy = torch.randn(V, C, generator=g).to(dtype).cuda().requires_grad_(True), torch.randn(n, C, generator=g).to(dtype).cuda()
    out = K.embedding(tokens.cuda(), w, 1.7)
    (grad,) = torch.autograd.grad(out, w, gy)
    assert out.shape == (n, C) and grad.shape == w.shape and grad.dtype == dtype
    check_lookup(tokens, w, torch.tensor(1.7, dtype=torch.float32).item(), gy, out, grad)


def test_embedding_of_more_dimensions_and_strides():
    from rwkv_wkv_hip import gated as K
    g = _g(5)
    tokens = torch.randint(0, 11, (3, 8), generator=g).cuda().t()          # not contiguous
    w = torch.randn(11, 40, generator=g).cuda()[:, :24].requires_grad_(True)
    gy = torch.randn(8, 3, 48, generator=g).cuda()[..., 5:29]
    out = K.embedding(tokens, w, 2.0)
    (grad,) = torch.autograd.grad(out, w, gy)
    assert out.shape == (8, 3, 24)
    check_lookup(tokens, w, 2.0, gy, out, grad)
