"""The operators of a gated recurrence model at their edges: what is not finite, shut and wide open gates, strides and addresses, offsets beyond 32 bits, streams and
captured graphs, buffers that autograd holds, calls that are refused.  Oracle and tolerances as in test_gpu_gated.py unless a test says otherwise."""
import math

import pytest
import torch

from oracle import gated as O
from tests import test_gpu_gated as S
from tests.util import assert_close

pytestmark = pytest.mark.gpu
RTOL, TYPES = S.RTOL, S.TYPES


def _kernels():
    from rwkv_wkv_hip import gated
    return gated


# ---- the recurrence
@pytest.mark.parametrize("T", [1, 9, 300])
@pytest.mark.parametrize("grad", [False, True])
def test_decays_and_gates_at_their_ends(T, grad):
    """A decay of minus infinity or a shut gate keeps the state, one of plus infinity forgets it, whatever the other is; gradients are the formula's limits."""
    K = _kernels()
    v, grads = S.recurrence_inputs(torch.float32, 2, T, 12)
    v["decay"][:6] = torch.tensor([-math.inf, -200.0, -30.0, 60.0, 1e30, math.inf])
    v["r"][0, ::3] = -math.inf
    v["r"][1, ::4] = 200.0
    v["r"][1, 1::4] = -200.0
    v["i"][0, 1::3] = math.inf
    v["i"][1, 1::3] = -math.inf
    want, got = S._double(v), S._cuda(v, leaf=grad)
    # (infinity times a gate of zero is zero there, in the kernel as in the limit: a decay that is large enough stands for it)
    want["decay"] = want["decay"].detach().clamp(max=1e36).requires_grad_(True)
    ref, out = O.gated_recurrence(**want), K.gated_recurrence(**got)
    for a, b in zip(out, ref):
        assert_close(a, b, RTOL[torch.float32])
    if grad:
        torch.autograd.backward(list(ref), [g.double() for g in grads])
        torch.autograd.backward(list(out), [g.cuda() for g in grads])
        for n in ("x", "i", "z", "state"):
            assert_close(got[n].grad, want[n].grad, RTOL[torch.float32], n)
        # where a decay is past what a step can hold its slope is none: the others'
        for n in ("r", "decay"):
            live = torch.isfinite(want[n].grad)
            assert torch.isfinite(got[n].grad).all()
            assert_close(got[n].grad.cpu()[live], want[n].grad[live], RTOL[torch.float32], n)


@pytest.mark.parametrize("T", [1, 70, 600])
def test_what_is_not_finite_stays_in_its_channel(T):
    """A NaN in one channel's stream, decay or state: the other channels are what they are without it, to the bit."""
    K = _kernels()
    v, grads = S.recurrence_inputs(torch.bfloat16, 2, T, 64)

    def run(spoil):
        c = S._cuda(v)
        with torch.no_grad():
            if spoil:
                c["x"][0, T // 2, 3] = math.nan
                c["r"][0, T // 3, 5] = math.nan
                c["i"][1, T // 3, 7] = math.inf
                c["z"][1, 0, 9] = math.nan
                c["decay"][11] = math.nan
                c["state"][0, 13] = math.inf
        out = K.gated_recurrence(**c)
        names = ("x", "r", "i", "decay", "z", "state")
        return [*out, *torch.autograd.grad(out, [c[n] for n in names], [g.cuda() for g in grads])]

    rest = [c for c in range(64) if c not in (3, 5, 7, 9, 11, 13)]
    for a, b in zip(run(False), run(True)):
        assert torch.equal(a[..., rest], b[..., rest])
    y, state = run(True)[:2]
    assert y[0, T // 2:, 3].isnan().all() and not y[0, :T // 2, 3].isnan().any() and y[:, :, 11].isnan().all() and state[:, 11].isnan().all()


@pytest.mark.parametrize("B,T,D", [(1, 9000, 6), (2, 4100, 3), (1, 16500, 2)])
def test_long_sequences(B, T, D):
    """Cut in time into many segments.  Tolerances as for a few hundred tokens: what a state is off by is forgotten with what it was off in."""
    K = _kernels()
    v, grads = S.recurrence_inputs(torch.float32, B, T, D)
    S.compare(K.gated_recurrence, O.gated_recurrence, v, grads, ("y", "state"))


@pytest.mark.parametrize("B,T,D", [(3, 300, 4096), (1, 2100, 4096), (9, 130, 1000), (70, 40, 1026)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sequences_are_what_they_are_alone(B, T, D, dtype):
    """Whatever the batch, its cut in time and the channels to a lane: within the tolerances of a sequence's own call."""
    K = _kernels()
    v, grads = S.recurrence_inputs(dtype, B, T, D)

    def run(rows):
        c = {n: (t[rows] if n != "decay" else t).cuda().requires_grad_(True) for n, t in v.items()}
        out = K.gated_recurrence(**c)
        return [*out, *torch.autograd.grad(out, [c[n] for n in ("x", "r", "i", "z", "state")], [g[rows].cuda() for g in grads])]

    whole = run(slice(None))
    for b in (0, B - 1):
        for a, one in zip(whole, run(slice(b, b + 1))):
            assert_close(a[b:b + 1], one, RTOL[dtype])


def test_a_state_chains_two_calls():
    K = _kernels()
    v, grads = S.recurrence_inputs(torch.float32, 2, 500, 40)
    c = S._cuda(v)
    cut = 201
    part = lambda s: {n: (t[:, s] if t.dim() == 3 else t) for n, t in c.items()}
    names = ("x", "r", "i", "decay", "z", "state")
    leaf, g = [c[n] for n in names], [t.cuda() for t in grads]
    whole = K.gated_recurrence(**c)
    first = K.gated_recurrence(**part(slice(0, cut)))
    second = K.gated_recurrence(**{**part(slice(cut, None)), "state": first[1]})
    two = torch.cat([first[0], second[0]], 1), second[1]
    for a, b in zip([*whole, *torch.autograd.grad(whole, leaf, g)], [*two, *torch.autograd.grad(two, leaf, g)]):
        assert_close(a, b, RTOL[torch.float32])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_addresses(dtype):
    """Slices that begin anywhere, streams shared by the sequences or the tokens: what their copies give."""
    K = _kernels()
    B, T, D = 3, 150, 64
    wide = torch.randn(B, T, 5 * D + 9, generator=S._g(1)).to(dtype).cuda()
    decay, gy = torch.randn(D, generator=S._g(2)).cuda() - 4, torch.randn(B, T, D, generator=S._g(3)).to(dtype).cuda()
    part = lambda i: wide[..., i:i + D]
    for views in ([part(0), part(64), part(128), part(192)], [part(1), part(66), part(131), part(200)], [part(2), part(66), part(130), part(194)],
                  [part(0)[:1].expand(B, T, D), part(64), part(128)[:, :1].expand(B, T, D), part(192)], [t.transpose(0, 1).contiguous().transpose(0, 1) for t in map(part, (0, 5, 10, 15))],
                  [wide[:, ::2, 0:D].repeat_interleave(2, 1)[:, :T] for _ in range(4)]):
        def run(t):
            leaf = [v.detach().requires_grad_(True) for v in t]
            out = K.gated_recurrence(leaf[0], leaf[1], leaf[2], decay, z=leaf[3])
            return [*out, *torch.autograd.grad(out[0], leaf, gy)]
        for a, b in zip(run(views), run([v.contiguous() for v in views])):
            assert_close(a, b, RTOL[dtype])          # (one or two channels to a lane, another cut)


def test_gradients_against_differences():
    """The kernels' own fp32 forward, along a random direction: (f(v + h d) - f(v - h d)) / 2h against gradient . d.  With h = 2^-7 the third derivative leaves h^2 / 6 of the
    order of the value, 1e-5, and rounding 2^-24 |f| / h per term; f is weighted and summed in 64 bits over N values, so both stay below 1e-3 of the norms' product / sqrt(N)."""
    K = _kernels()
    g = S._g(4)
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    tokens = torch.randint(-1, 9, (50,), generator=g).cuda()
    cases = [(lambda x, a, i, d, z, s: torch.cat([t.flatten() for t in K.gated_recurrence(x, a, i, d, z, s)]), [r(2, 90, 8), r(2, 90, 8), r(2, 90, 8), r(8) - 3, r(2, 90, 8), r(2, 8)]),
             (lambda x, a, b: K.gated_feed_forward(x, a, b, "gelu").flatten(), [r(70, 40), r(30, 40) / 6, r(30, 40) / 6]),
             (lambda w: K.embedding(tokens, w, 2.0).flatten(), [r(9, 12)])]
    for f, v in cases:
        for i in range(len(v)):
            leaf = [t.clone().requires_grad_(j == i) for j, t in enumerate(v)]
            out = f(*leaf)
            weight, d, h = r(*out.shape), r(*v[i].shape), 2.0 ** -7
            (grad,) = torch.autograd.grad(out, leaf[i], weight)
            with torch.no_grad():
                at = lambda s: (f(*[t + s * d if j == i else t for j, t in enumerate(v)]).double() * weight.double()).sum()
                slope = (at(h) - at(-h)) / (2 * h)
            want = (grad.double() * d.double()).sum()
            assert abs(slope - want) <= 1e-3 * grad.double().norm() * d.double().norm() / math.sqrt(d.numel()) + 1e-3 * abs(want)


# ---- the gated feed-forward
@pytest.mark.parametrize("dtype,R,C,F", [(torch.bfloat16, 1500, 520, 4608), (torch.float16, 1100, 1024, 2816), (torch.bfloat16, 2048, 264, 8192), (torch.float32, 600, 520, 1500),
                                         (torch.bfloat16, 40, 2048, 5000), (torch.bfloat16, 17, 2056, 4100), (torch.float32, 64, 512, 2000), (torch.bfloat16, 60, 1999, 700),
                                         # rows that are not whole pieces of 16 bytes, as they lie and copied, by tiles of 64, 128 and 256
                                         (torch.bfloat16, 300, 1001, 2731), (torch.float16, 1024, 99, 2731), (torch.bfloat16, 400, 519, 14335), (torch.bfloat16, 100, 1999, 300),
                                         (torch.float16, 6000, 99, 1500), (torch.bfloat16, 16000, 261, 1500), (torch.float32, 100, 99, 300), (torch.float32, 8192, 99, 300),
                                         (torch.float32, 4096, 99, 8200), (torch.float32, 16000, 519, 1500), (torch.float16, 130, 1002, 700), (torch.bfloat16, 33, 4094, 3000),
                                         # one row of tiles whose columns are shared out evenly
                                         (torch.bfloat16, 50, 104, 9001), (torch.float16, 64, 99, 8960), (torch.bfloat16, 17, 128, 16384), (torch.bfloat16, 64, 72, 8193), (torch.float32, 64, 72, 8961),
                                         # single rows and few, by every alignment of rows
                                         (torch.bfloat16, 1, 4096, 5000), (torch.bfloat16, 3, 1002, 500), (torch.float16, 20, 1001, 500), (torch.bfloat16, 40, 1006, 300), (torch.float32, 9, 1001, 500),
                                         (torch.float32, 30, 1002, 500), (torch.float32, 64, 1004, 500), (torch.float16, 1, 9, 1), (torch.float32, 2, 3, 5)])
def test_feed_forward_by_every_size_of_tile(dtype, R, C, F):
    S.feed_forward(dtype, R, C, F, "silu")


def test_feed_forward_reads_rows_as_they_lie():
    """Slices of wider tensors, rows that begin anywhere, one row for all, weights that are not contiguous."""
    K = _kernels()
    g = S._g(6)
    wide = torch.randn(70, 200, generator=g).bfloat16().cuda()
    w = torch.randn(2, 96, 64, generator=g).bfloat16().cuda() / 8
    gy = torch.randn(70, 96, generator=g).bfloat16().cuda()
    for x in (wide[:, :64], wide[:, 8:72], wide[:, 3:67], wide[:1, :64].expand(70, 64), wide[::2, :64].repeat(2, 1), wide[:, :128:2], wide[:1, 3:67], wide[:1, :1].expand(1, 64)):
        for a, b in ((w[0], w[1]), (w.transpose(1, 2).contiguous().transpose(1, 2)[0], w[1])):
            def run(*t):
                leaf = [v.detach().requires_grad_(True) for v in t]
                out = K.gated_feed_forward(*leaf)
                return [out, *torch.autograd.grad(out, leaf, gy[:len(out)])]
            for p, q in zip(run(x, a, b), run(x.contiguous(), a.contiguous(), b.contiguous())):
                assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C,F", [(1, 99, 40), (12, 99, 40), (40, 90, 40), (200, 99, 40), (200, 35, 40), (5000, 99, 1500)])
def test_feed_forward_reads_nothing_beside_its_rows(dtype, R, C, F):
    """x's rows between NaNs, weights behind and before NaNs: what their copies give."""
    K = _kernels()
    g = S._g(R, C)
    for shift in range(0, 9, 1 if R < 300 else 4):
        wide = torch.full((R, C + 13), math.nan, dtype=dtype, device="cuda")
        x = wide[:, shift:shift + C]
        x.copy_(torch.randn(R, C, generator=g))
        flat = torch.full((F * C + 2 * 8,), math.nan, dtype=dtype, device="cuda")
        w = flat[8:8 + F * C].view(F, C)
        w.copy_(torch.randn(F, C, generator=g) / 10)
        leaf, copies = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)], [t.clone().requires_grad_(True) for t in (x, w)]
        a, b = K.gated_feed_forward(leaf[0], leaf[1], leaf[1]), K.gated_feed_forward(copies[0], copies[1], copies[1])
        assert torch.isfinite(a).all() and torch.equal(a, b)
        for p, q in zip(torch.autograd.grad(a, leaf, torch.ones_like(a)), torch.autograd.grad(b, copies, torch.ones_like(b))):
            assert torch.isfinite(p).all() and torch.equal(p, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C,F", [(20, 100, 70), (200, 104, 130), (200, 99, 130), (1500, 520, 4608)])
def test_feed_forward_not_finite_stays_in_its_row_and_column(dtype, R, C, F):
    K = _kernels()
    g = S._g(R, C)
    x, a, b = torch.randn(R, C, generator=g).to(dtype).cuda(), *((torch.randn(F, C, generator=g) / 10).to(dtype).cuda() for _ in range(2))
    clean = K.gated_feed_forward(x, a, b)
    x2, a2, b2 = x.clone(), a.clone(), b.clone()
    x2[R // 2, C - 1], a2[F // 3, 0], b2[F - 1, C - 1] = math.nan, math.inf, math.nan
    out = K.gated_feed_forward(x2, a2, b2)
    rows, columns = [r for r in range(R) if r != R // 2], [f for f in range(F) if f not in (F // 3, F - 1)]
    assert torch.equal(out[rows][:, columns], clean[rows][:, columns]) and out[R // 2].isnan().all() and out[:, F - 1].isnan().all()
    # backward: a row of x that is not finite stays in its row of gx (and reaches both weights' gradients, where it belongs)
    leaf = [t.clone().requires_grad_(True) for t in (x2, a, b)]
    y = K.gated_feed_forward(*leaf)
    gx, _, _ = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.isfinite(gx[rows].float()).all() and gx[R // 2].isnan().all()


@pytest.mark.parametrize("name", ["silu", "gelu", "relu"])
def test_activations_far_out(name):
    """One column in, weights of one: g = u = x.  Values and slopes where the exponentials are zero or infinite."""
    K = _kernels()
    x = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20.0, -20.0, 88.0, -88.0, 200.0, -200.0, 1e4, -1e4, 1e18, -1e18], device="cuda")[:, None].requires_grad_(True)
    one = torch.ones(1, 1, device="cuda")
    y = K.gated_feed_forward(x, one, one, name)
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    d = x.detach().cpu().double().requires_grad_(True)
    act = {"silu": torch.nn.functional.silu, "gelu": lambda t: torch.nn.functional.gelu(t, approximate="tanh"), "relu": torch.nn.functional.relu}[name]
    ref = act(d) * d
    (want,) = torch.autograd.grad(ref, d, torch.ones_like(ref))
    # a sigmoid of v is right to (|v| + 8) 2^-23 of itself (v's own rounding inside the exponential), zero below 2^-126
    tol = (x.detach().cpu().double().abs().clamp(max=200) * 4 + 32) * 2.0 ** -23
    for a, b in ((y, ref), (g, want)):
        assert torch.isfinite(a).all() and bool(((a.detach().cpu().double() - b).abs() <= tol * b.abs() + 1e-30).all()), (a.flatten(), b.flatten())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,C,F", [(1, 64, 96), (3, 68, 205), (16, 520, 300), (17, 99, 130), (32, 256, 1024), (32, 1001, 333)])
def test_feed_forward_gradients_of_few_rows_are_rounded_once(dtype, R, C, F):
    """Up to 32 rows: within half a step of the 64-bit value, and of what fp32 sums of up to 2048 products leave (2048 2^-24 of the products' norms, taken as of the row's largest)."""
    K = _kernels()
    g = S._g(R, C, F)
    t = [torch.randn(R, C, generator=g).to(dtype), *((torch.randn(F, C, generator=g) / C ** 0.5).to(dtype) for _ in range(2))]
    gy = torch.randn(R, F, generator=g).to(dtype)
    a, b = [v.cuda().requires_grad_(True) for v in t], [v.double().requires_grad_(True) for v in t]
    got = torch.autograd.grad(K.gated_feed_forward(*a), a, gy.cuda())
    want = torch.autograd.grad(O.gated_feed_forward(*b), b, gy.double())
    for p, q in zip(got, want):
        off, half = (p.cpu().double() - q).abs(), torch.finfo(dtype).eps / 2
        assert bool((off <= half * 1.001 * q.abs() + 2048 * 2.0 ** -24 * q.abs().max() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all())


def test_feed_forward_gradients_that_are_wanted():
    """Only x's, only one weight's: what the whole call gives."""
    K = _kernels()
    g = S._g(9)
    t = [torch.randn(90, 72, generator=g).bfloat16().cuda(), *((torch.randn(50, 72, generator=g) / 8).bfloat16().cuda() for _ in range(2))]
    gy = torch.randn(90, 50, generator=g).bfloat16().cuda()

    def run(wanted):
        leaf = [v.clone().requires_grad_(w) for v, w in zip(t, wanted)]
        K.gated_feed_forward(*leaf).backward(gy)
        return [v.grad for v in leaf]
    whole = run((True, True, True))
    for wanted in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        for a, b, w in zip(run(wanted), whole, wanted):
            assert (a is None) if not w else torch.equal(a, b)


# ---- the lookup
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,C", [(1, 8), (5, 24), (1000, 7), (300, 520), (70000, 3), (2, 4100)])
@pytest.mark.parametrize("kind", ["one", "none", "runs", "each"])
def test_embedding_of_every_distribution(dtype, V, C, kind):
    """All places of one token, none with any, runs about the sizes that the sums are cut at, every token once."""
    K = _kernels()
    if kind == "one":
        tokens = torch.full((5000,), V // 2)
    elif kind == "none":
        tokens = torch.tensor([-1, V, -100, 1 << 40, -(1 << 40), V + 5] * 30)
    elif kind == "runs":
        tokens = torch.cat([torch.full((n,), i % V) for i, n in enumerate([63, 1, 64, 65, 127, 128, 129, 1, 2, 62, 64, 64, 300])])
        tokens = tokens[torch.randperm(len(tokens), generator=S._g(1))]
    else:
        tokens = torch.randperm(V, generator=S._g(2))[:6000]
    w, gy = torch.randn(V, C, generator=S._g(3)).to(dtype).cuda().requires_grad_(True), torch.randn(len(tokens), C, generator=S._g(4)).to(dtype).cuda()
    for t in [tokens.cuda()] + ([tokens.int().cuda()] if kind != "none" else []):
        out = K.embedding(t, w, 0.5)
        (grad,) = torch.autograd.grad(out, w, gy)
        S.check_lookup(tokens, w, 0.5, gy, out, grad)


def test_embedding_sums_in_the_places_order():
    """Of one token: fp32 sums of 8 places at a time (as few as 4096 are cut), in order, added in order.  Values that cancel only so."""
    K = _kernels()
    w = torch.zeros(3, 8, device="cuda", requires_grad=True)
    gy = torch.tensor([2.0 ** 30, 1.0, -2.0 ** 30] * 40 + [3.0]).repeat_interleave(8).view(-1, 8).cuda()
    tokens = torch.ones(121, dtype=torch.long, device="cuda")
    (a,) = torch.autograd.grad(K.embedding(tokens, w), w, gy)
    total = torch.zeros(8)
    for part in gy.cpu().split(8):
        s = part[0].clone()
        for row in part[1:]:
            s += row
        total += s
    assert torch.equal(a[1].cpu(), total) and not a[0].any() and not a[2].any()


# ---- the same bits every time, another stream, captured graphs, threads of a pass
def _calls():
    """name -> (leaves, function of them, gradients): a training call of each"""
    K = _kernels()
    g = S._g(11)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()
    tokens = torch.randint(0, 99, (3000,), generator=g).cuda()
    return {"recurrence": ([r(2, 700, 128), r(2, 700, 128), r(2, 700, 128), r(128).float() - 4, r(2, 700, 128), r(2, 128).float()],
                           lambda x, a, i, d, z, s: K.gated_recurrence(x, a, i, d, z, s), [r(2, 700, 128), r(2, 128).float()]),
            "feed_forward": ([r(130, 99), r(200, 99) / 10, r(200, 99) / 10], lambda x, a, b: (K.gated_feed_forward(x, a, b),), [r(130, 200)]),
            "embedding": ([r(99, 72)], lambda w: (K.embedding(tokens, w, 3.0),), [r(3000, 72)])}


def _train(name, leaves=None):
    values, f, grads = _calls()[name]
    leaf = [v.requires_grad_(True) for v in (leaves or values)]
    out = f(*leaf)
    return [*out, *torch.autograd.grad(out, leaf, grads)]


@pytest.mark.parametrize("name", ["recurrence", "feed_forward", "embedding"])
def test_the_same_bits_on_another_stream(name):
    want = _train(name)
    assert all(torch.equal(a, b) for a, b in zip(want, _train(name)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:          # two at once, each with workspaces of its own
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(_train(name))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(want, g))


@pytest.mark.parametrize("name", ["recurrence", "feed_forward", "embedding"])
def test_a_training_call_in_a_graph(name):
    """Forward and backward captured once, replayed on new inputs with eager work between the replays."""
    values, f, grads = _calls()[name]

    def step():
        leaf = [v.detach().requires_grad_(True) for v in values]
        out = f(*leaf)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaf, grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            for v in values:
                v.mul_(0.9).add_(0.01 * k)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_two_graphs_do_not_share_a_workspace():
    """Captured apart, replayed in turn and again: each finds its own results."""
    K = _kernels()
    x = [torch.randn(1, 4000, 64, device="cuda").bfloat16() for _ in range(2)]
    decay = torch.randn(64, device="cuda") - 4
    want = [K.gated_recurrence(t, t, t, decay) for t in x]
    graphs, outs = [], []
    for t in x:
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(K.gated_recurrence(t, t, t, decay))
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_single_tokens_in_a_graph():
    K = _kernels()
    v, _ = S.recurrence_inputs(torch.bfloat16, 4, 1, 64)
    c = S._cuda(v, leaf=False)
    start = c["state"].clone()
    w = [torch.randn(96, 64, device="cuda").bfloat16() / 8 for _ in range(2)]
    table, tokens = torch.randn(50, 64, device="cuda").bfloat16(), torch.zeros(4, 1, dtype=torch.long, device="cuda")

    def step():
        c["x"].copy_(K.embedding(tokens, table, 8.0))
        y, _ = K.gated_recurrence(**c, out_state=c["state"])
        return K.gated_feed_forward(y, *w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    rows = [torch.randint(0, 50, (4, 1), device="cuda") for _ in range(4)]
    eager = []
    c["state"].copy_(start)
    for t in rows:
        tokens.copy_(t)
        eager.append(step().clone())
    c["state"].copy_(start)
    for t, want in zip(rows, eager):
        tokens.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_a_state_overwritten_in_place_is_noticed():
    """out_state raises its tensor's version, so that a backward that had saved it refuses."""
    K = _kernels()
    v, _ = S.recurrence_inputs(torch.float32, 2, 1, 8)
    c = S._cuda(v, leaf=False)
    s = c.pop("state")
    w = torch.ones(2, 8, device="cuda", requires_grad=True)
    product = (s * w).sum()
    with torch.no_grad():
        K.gated_recurrence(**c, state=s, out_state=s)
    with pytest.raises(RuntimeError):
        product.backward()
    with torch.inference_mode():
        t = torch.zeros(2, 8, device="cuda")
        K.gated_recurrence(**c, state=t, out_state=t)


def test_states_and_decays_of_other_types():
    """Read in fp32 whatever they are; the new state is fp32, gradients come in the inputs' types."""
    K = _kernels()
    v, grads = S.recurrence_inputs(torch.bfloat16, 2, 40, 16)
    for kind in (torch.bfloat16, torch.float64):
        c = S._cuda({**v, "decay": v["decay"].to(kind), "state": v["state"].to(kind)})
        f = S._cuda({**v, "decay": v["decay"].to(kind).float(), "state": v["state"].to(kind).float()})
        a, b = K.gated_recurrence(**c), K.gated_recurrence(**f)
        assert a[1].dtype == torch.float32 and all(torch.equal(p, q) for p, q in zip(a, b))
        torch.autograd.backward(a, [g.cuda() for g in grads])
        torch.autograd.backward(b, [g.cuda() for g in grads])
        for n in ("decay", "state"):
            assert c[n].grad.dtype == kind and torch.equal(c[n].grad, f[n].grad.to(kind))


def test_gradients_that_do_not_come():
    """Only the state's or only y's gradient: the other is zero."""
    K = _kernels()
    v, grads = S.recurrence_inputs(torch.float32, 2, 100, 24)
    for k in range(2):
        c, w = S._cuda(v), S._double(v)
        K.gated_recurrence(**c)[k].backward(grads[k].cuda())
        O.gated_recurrence(**w)[k].backward(grads[k].double())
        for n in ("x", "r", "i", "decay", "state"):
            assert_close(c[n].grad, w[n].grad, RTOL[torch.float32], n)
        assert k == 0 or not c["z"].grad.any()


def test_offsets_beyond_32_bits():
    K = _kernels()
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    g = torch.Generator(device="cuda").manual_seed(1)
    # two sequences 4 GiB apart in one buffer
    D, T, far = 64, 40, (1 << 31) + 24
    buffer = torch.empty(far + T * 4 * D, dtype=torch.bfloat16, device="cuda")
    x = buffer.as_strided((2, T, 4 * D), (far, 4 * D, 1))
    x.copy_(torch.randn(2, T, 4 * D, device="cuda", generator=g))
    decay = torch.randn(D, device="cuda", generator=g) - 4
    run = lambda t: K.gated_recurrence(t[..., :D], t[..., D:2 * D], t[..., 2 * D:3 * D], decay, z=t[..., 3 * D:])
    assert all(torch.equal(a, b) for a, b in zip(run(x), run(x.contiguous())))
    del buffer, x
    # results past 2^32 elements: the last sequences are what they are alone
    B, T, D = 260, 4096, 4100
    x = torch.randn(1, T, D, device="cuda", generator=g).bfloat16()
    y, s = K.gated_recurrence(x.expand(B, T, D), x.expand(B, T, D), x.expand(B, T, D), decay.repeat(65)[:D])
    one, e = K.gated_recurrence(x, x, x, decay.repeat(65)[:D])
    for b in (0, B - 1):
        assert_close(y[b:b + 1], one, RTOL[torch.bfloat16])
        assert_close(s[b:b + 1], e, RTOL[torch.float32])
    del x, y
    # a table past 2^32 elements and its gradient
    V, C = (1 << 20) + 3, 4104
    table = torch.zeros(V, C, dtype=torch.bfloat16, device="cuda")
    table[-2:] = 3.0
    tokens = torch.tensor([V - 1, 0, V - 2, V - 1, V], device="cuda")
    out = K.embedding(tokens, table.requires_grad_(True), 0.5)
    assert (out[[0, 2, 3]] == 1.5).all() and not out[[1, 4]].any()
    (grad,) = torch.autograd.grad(out, table, torch.ones_like(out))
    assert (grad[-1] == 1).all() and (grad[-2] == 0.5).all() and (grad[0] == 0.5).all() and not grad[1:-2].any()


def test_many_rows_and_sequences():
    """More rows, sequences and places than the common sizes: each gives what it gives alone."""
    K = _kernels()
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    x, a, b = r(300000, 64), r(48, 64) / 8, r(48, 64) / 8
    out = K.gated_feed_forward(x, a, b)
    assert torch.equal(out[-100:], K.gated_feed_forward(x[-100:], a, b)) and torch.equal(out[:1], K.gated_feed_forward(x[:1], a, b))
    s, d = r(9000, 2, 6), r(6).float() - 3
    y, e = K.gated_recurrence(s, s, s, d)
    assert torch.equal(y[-5:], K.gated_recurrence(s[-5:], s[-5:], s[-5:], d)[0])
    tokens = torch.randint(0, 1000, (700001,), device="cuda", generator=g)
    w, gy = r(1000, 16).requires_grad_(True), r(700001, 16)
    (grad,) = torch.autograd.grad(K.embedding(tokens, w), w, gy)
    S.check_lookup(tokens, w, 1.0, gy, K.embedding(tokens, w), grad)
    # around what is sorted at once, in small and large tiles, and what every tile adds up for itself; keys of two digits
    w = torch.zeros(70000, 4, device="cuda", requires_grad=True)
    for n in (1, 4095, 4096, 4097, 48 * 1024, 48 * 1024 + 1, 1 << 18, (1 << 18) + 1):
        tokens, gy = torch.randint(-3, 70000, (n,), device="cuda", generator=g), r(n, 4).float()
        (grad,) = torch.autograd.grad(K.embedding(tokens, w), w, gy)
        S.check_lookup(tokens, w, 1.0, gy, K.embedding(tokens, w), grad)


def test_single_rows_and_places():
    """x without a batch, a place without one."""
    K = _kernels()
    g = S._g(13)
    x, a, b, w = torch.randn(24, generator=g).cuda(), *(torch.randn(10, 24, generator=g).cuda() for _ in range(2)), torch.randn(5, 24, generator=g).cuda()
    leaf = [t.requires_grad_(True) for t in (x, a, b, w)]
    one, whole = K.gated_feed_forward(x, a, b), K.gated_feed_forward(x[None], a, b)
    assert one.shape == (10,) and torch.equal(one, whole[0])
    row = K.embedding(torch.tensor(3, device="cuda"), w, 2.0)
    assert row.shape == (24,) and torch.equal(row, 2 * w[3])
    grads = torch.autograd.grad(one.sum() + row.sum(), leaf)
    assert [t.shape for t in grads] == [t.shape for t in leaf] and torch.equal(grads[3], torch.zeros(5, 24, device="cuda").index_fill(0, torch.tensor([3], device="cuda"), 2.0))


# ---- refusals
def test_refusals():
    import rwkv_wkv_hip as W
    K = _kernels()
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    x, d = z(2, 5, 8), z(8)
    for bad in (lambda: K.gated_recurrence(x, x, z(2, 5, 9), d), lambda: K.gated_recurrence(x, x.half(), x, d), lambda: K.gated_recurrence(x, x, x, z(9)),
                lambda: K.gated_recurrence(x, x, x, d, state=z(2, 9)), lambda: K.gated_recurrence(x, x, x, d, z=z(2, 4, 8)), lambda: K.gated_recurrence(x, x, x, d, lengths=z(2)),
                lambda: K.gated_recurrence(x[0], x[0], x[0], d), lambda: K.gated_recurrence(x, x, x, d, out_state=z(2, 8).half()),
                lambda: K.gated_recurrence(x[:, :1].requires_grad_(True), x[:, :1], x[:, :1], d, out_state=z(2, 8)),
                lambda: K.gated_feed_forward(x, z(6, 9), z(6, 9)), lambda: K.gated_feed_forward(x, z(6, 8), z(7, 8)), lambda: K.gated_feed_forward(x, z(6, 8).half(), z(6, 8)),
                lambda: K.gated_feed_forward(x[:0], z(6, 8), z(6, 8)), lambda: K.embedding(z(3), z(4, 8)), lambda: K.embedding(z(3, dtype=torch.long), z(4)),
                lambda: K.embedding(z(0, dtype=torch.long), z(4, 8))):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: K.gated_recurrence(x.double(), x.double(), x.double(), d), lambda: K.gated_recurrence(x[:, :0], x[:, :0], x[:, :0], d),
                lambda: K.gated_feed_forward(x, z(6, 8), z(6, 8), "tanh"), lambda: K.gated_feed_forward(x.double(), z(6, 8).double(), z(6, 8).double()),
                lambda: K.gated_feed_forward(x, z(0, 8), z(0, 8)), lambda: K.embedding(z(3, dtype=torch.long), z(4, 8).double())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(W.WKVError):
        K.gated_recurrence(x, x, x, d.cpu())
    with pytest.raises(W.WKVError):
        s = z(2, 8)
        K.gated_recurrence(x, x, x, d, state=s, out_state=s)                     # in place for single tokens only
    with pytest.raises(W.WKVError):
        K.embedding(torch.zeros(3, dtype=torch.long), z(4, 8))
    with pytest.raises(RuntimeError):                                            # a forward-mode tangent is not dropped
        import torch.autograd.forward_ad as fw
        with fw.dual_level():
            K.gated_feed_forward(fw.make_dual(x, x), z(6, 8), z(6, 8))
