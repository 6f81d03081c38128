"""The state space operators and sampling at their edges: what is not finite, types that differ, buffers that autograd holds, sizes past a grid's
threads, and the kernels' many-row, many-token and many-sequence forms.  Oracle and tolerances as in test_gpu_ssm.py unless a test says otherwise."""
import math

import pytest
import torch

from oracle import ssm as O
from tests import test_gpu_ssm as S
from tests.util import assert_close

pytestmark = pytest.mark.gpu
RTOL = S.RTOL


@pytest.mark.parametrize("weights", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("times", [1, 8, 22, 74])
@pytest.mark.parametrize("thousandths", [3, 7, 13])
def test_rows_in_8_bits_round_once(weights, times, thousandths):
    """y / scale where it lies in the middle of two values of 8 bits: a row of ones, so that y is the weight, of every such middle times the scale.  The
    quotient in fp32 is exact, the one rounding goes to even."""
    from rwkv_wkv_hip import ssm as K
    steps = [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (1 + m / 8) * 2.0 ** e <= 448]
    middles = torch.tensor([(a + b) / 2 for a, b in zip(steps, steps[1:])] + [448.0], dtype=torch.float64).repeat(times)
    weight = (middles * (thousandths / 1024)).to(weights)
    assert weights == torch.bfloat16 or torch.equal(weight.double(), middles * (thousandths / 1024))
    q, scale, _ = K.rms_norm_fp8(torch.ones(3, len(weight), dtype=torch.bfloat16, device="cuda"), weight.cuda(), eps=0.0)
    want = weight.float().abs().max() / 448
    assert (scale.cpu() == want).all()
    assert torch.equal(q.cpu().view(torch.uint8), (weight.float() / want).to(torch.float8_e4m3fn).view(torch.uint8).expand(3, -1))


# ---- 8 bits
@pytest.mark.parametrize("C", [64, 100, 646, 2560, 8200])
def test_rows_in_8_bits_that_are_not_finite(C):
    """A row with a NaN or an infinity has the scale max |y| / 448, which is NaN (an infinity: its norm is NaN); its neighbours are what they are without it."""
    from rwkv_wkv_hip import ssm as K
    g = S._g(C, 3)
    x, w = torch.randn(7, C, generator=g).bfloat16().cuda(), (torch.rand(C, generator=g) + 0.5).bfloat16().cuda()
    q, scale, _ = K.rms_norm_fp8(x, w)
    bad = x.clone()
    bad[1, C // 2], bad[3, 5], bad[5, 7] = math.nan, math.inf, -math.inf
    q2, scale2, _ = K.rms_norm_fp8(bad, w)
    assert scale2[1::2].isnan().sum() == 3 and q2[1::2].float().isnan().all()
    assert torch.equal(q2.view(torch.uint8)[::2], q.view(torch.uint8)[::2]) and torch.equal(scale2[::2], scale[::2])
    # from one weight: every row's largest value
    w2 = w.clone()
    w2[C - 1] = math.nan
    q2, scale2, _ = K.rms_norm_fp8(x, w2)
    assert scale2.isnan().all() and q2.float().isnan().all()
    w2[C - 1] = math.inf
    q2, scale2, _ = K.rms_norm_fp8(x, w2)
    assert scale2.isinf().all() and not q2[:, :-1].float().any() and q2[:, -1].float().isnan().all()


# ---- sizes past a grid's threads
def test_sums_of_more_columns_than_a_grid_has_threads():
    """B and C of 2^27 elements and 64 sequences: the sum of their gradients' shares takes 2^32 threads.  Sequences are compared with calls of their own
    (cut in time elsewhere: within the tolerances)."""
    from rwkv_wkv_hip import ssm as K
    free, _ = torch.cuda.mem_get_info()
    if free < 32 << 30:
        pytest.skip("needs 32 GB")
    B, T, D, N = 64, 1 << 17, 16, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.empty(s, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    v = dict(x=r(B, T, D), dt=r(B, T, D), B=r(B, T, N), C=r(B, T, N))
    A, gy = -torch.rand(D, N, device="cuda", generator=g) - 0.1, r(B, T, D)

    def run(rows):
        leaf = {n: t[rows].clone().requires_grad_(True) for n, t in v.items()}
        y, _ = K.selective_scan(A=A, **leaf)
        return [y, *torch.autograd.grad(y, list(leaf.values()), gy[rows])]

    whole = run(slice(None))
    for b in (0, 37, 63):
        for got, want in zip(whole, run(slice(b, b + 1))):
            assert_close(got[b], want[0].cpu(), RTOL[torch.bfloat16])


def test_scan_of_more_workgroups_than_a_grid_has_threads():
    """4096 sequences of 4096 channels with a B and C each: 2^24 workgroups.  A sequence gives what it gives alone."""
    from rwkv_wkv_hip import ssm as K
    free, _ = torch.cuda.mem_get_info()
    if free < 32 << 30:
        pytest.skip("needs 32 GB")
    B, T, D = 4096, 2, 4096
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.empty(s, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    v = dict(x=r(B, T, D), dt=r(B, T, D), B=r(B, T, D, 1), C=r(B, T, D, 1))
    A, gy = -torch.rand(D, 1, device="cuda", generator=g) - 0.1, r(B, T, D)

    def run(rows):
        leaf = {n: t[rows].clone().requires_grad_(True) for n, t in v.items()}
        y, s = K.selective_scan(A=A, **leaf)
        return [y, s, *torch.autograd.grad(y, list(leaf.values()), gy[rows])]

    whole = run(slice(None))
    for b in (0, 2047, 4093):
        for got, want in zip(whole, run(slice(b, b + 3))):
            assert torch.equal(got[b:b + 3], want)


# ---- values that are not finite, decays that grow
@pytest.mark.parametrize("N", [16, 20, 4])
@pytest.mark.parametrize("T,lengths", [(1, [0, 1, 1]), (40, [0, 17, 40])])
def test_a_state_that_forgets_everything(N, T, lengths):
    """A = -infinity: nothing is left of the state before a token; where there is no token (behind a sequence's end) it stays."""
    from rwkv_wkv_hip import ssm as K
    v, _ = S._scan_inputs(torch.float32, 3, T, 24, N, lengths=lengths)
    v["A"][3, 1], v["A"][7], v["A"][8, N - 1] = -math.inf, -math.inf, -math.inf
    ref = O.selective_scan(**{n: t.double() if t.is_floating_point() else t for n, t in v.items()})
    for a, b in zip(K.selective_scan(**S._cuda(v, leaf=False)), ref):
        assert_close(a, b, RTOL[torch.float32])
    for a, b in zip(K.selective_scan(**S._cuda(v, leaf=True)), ref):
        assert_close(a, b, RTOL[torch.float32])


def test_growth_past_what_32_bits_hold_from_nothing():
    """A > 0 in a sequence that is cut in time: a segment's growth alone passes 2^128, but there is nothing yet that grows, and backwards no gradient."""
    from rwkv_wkv_hip import ssm as K
    v, grads = S._scan_inputs(torch.float32, 1, 2048, 24, 16, state=False)
    v["A"], v["dt"], v["dt_bias"] = torch.full((24, 16), 0.5), torch.full((1, 2048, 24), 1.0), torch.full((24,), 0.2)
    token = torch.arange(2048)[None, :, None]
    v["x"] = v["x"] * (token >= 2048 - 60)
    S._compare(K.selective_scan, O.selective_scan, v, [grads[0] * (token < 60), grads[1] * 0], ("y", "state"))


def test_growth_of_a_small_state():
    """What comes in is small enough that the growth through a segment, too large for 32 bits by itself, leaves it finite."""
    from rwkv_wkv_hip import ssm as K
    v, _ = S._scan_inputs(torch.float32, 1, 256, 8, 16, gate=False, skip=False, bias=False)
    v["A"], v["dt"], v["x"] = torch.full((8, 16), 0.5), torch.full((1, 256, 8), 3.0), torch.zeros(1, 256, 8)
    v["state"] = v["state"] * 1e-35
    v["dt"][:, 64:] = -100.0
    ref = O.selective_scan(**{n: t.double() for n, t in v.items()})
    for a, b in zip(K.selective_scan(**S._cuda(v, leaf=False)), ref):
        assert_close(a, b, RTOL[torch.float32])


@pytest.mark.parametrize("T", [40, 200])
def test_a_channel_that_is_not_finite_leaves_other_groups_alone(T):
    """Groups of 5 channels in workgroups of more, sequences in one piece and cut in time: the first channel's state gradient, decay and step are not finite, the
    second group's gradients are what they are without."""
    from rwkv_wkv_hip import ssm as K
    for N in (16, 24, 64):
        v, grads = S._scan_inputs(torch.float32, 2, T, 10, N, 2)
        runs = []
        for bad in (False, True):
            c = S._cuda(v, leaf=False)
            gs = grads[1].cuda()
            if bad:
                gs[:, 0], c["A"][0, 1:], c["dt"][:, T - 9, 0] = math.inf, math.nan, math.nan
            c = {n: t.requires_grad_(True) for n, t in c.items()}
            runs.append((c, torch.autograd.grad(list(K.selective_scan(**c)), list(c.values()), [grads[0].cuda(), gs])))
        for n, a, b in zip(v, *(r[1] for r in runs)):
            if n in ("B", "C"):
                assert torch.isfinite(a).all() and torch.equal(a[:, :, 1], b[:, :, 1]), n


@pytest.mark.parametrize("N", [16, 40])
def test_gradients_behind_a_sequence_are_zero(N):
    """Of B and C too, in the tile the sequence ends in, whatever gradient comes in through the state."""
    from rwkv_wkv_hip import ssm as K
    v, grads = S._scan_inputs(torch.float32, 3, 40, 12, N, lengths=[21, 0, 40])
    grads[1][0, 3], grads[1][1, 5, 2] = math.inf, math.nan
    c = S._cuda(v)
    torch.autograd.backward(list(K.selective_scan(**c)), [a.cuda() for a in grads])
    for n in ("x", "dt", "z", "B", "C"):
        assert not c[n].grad[0, 21:].any() and not c[n].grad[1].any(), n
    assert torch.isfinite(c["B"].grad[2]).all()


# ---- buffers
def test_a_state_overwritten_in_place_is_noticed():
    """What autograd has saved and out_state has overwritten since raises in the backward pass, as after any operation in place."""
    from rwkv_wkv_hip import ssm as K
    r = lambda *s: torch.randn(*s, device="cuda")
    w, window, state = r(8, 4), r(2, 3, 8), r(2, 8, 16)
    A, one, b = -torch.rand(8, 16, device="cuda"), r(2, 1, 8), r(2, 1, 16)
    scale = torch.ones((), device="cuda", requires_grad=True)

    y, _ = K.causal_conv(r(2, 5, 8).requires_grad_(True), w, state=window)
    before = window._version
    with torch.no_grad():
        K.causal_conv(one, w, state=window, out_state=window)
    assert window._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()

    z = state * scale
    before = state._version
    with torch.no_grad():
        K.selective_scan(one, one, A, b, b, state=state, out_state=state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()

    with torch.inference_mode():          # (tensors without a version)
        s = torch.zeros(2, 8, 16, device="cuda")
        t = torch.zeros(2, 3, 8, device="cuda")
        assert K.selective_scan(one, one, A, b, b, state=s, out_state=s)[1].data_ptr() == s.data_ptr()
        assert K.causal_conv(one, w, state=t, out_state=t)[1].data_ptr() == t.data_ptr()


# ---- types that differ
@pytest.mark.parametrize("x,weight,bias", [(torch.bfloat16, torch.bfloat16, torch.float32), (torch.float16, torch.float16, torch.float32), (torch.bfloat16, torch.float32, torch.bfloat16),
                                           (torch.float32, torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16, torch.float16)])
def test_causal_conv_of_parameters_in_two_types(x, weight, bias):
    """Neither parameter is held in fewer bits than it has: the fp32 one's gradient is right to fp32."""
    from rwkv_wkv_hip import ssm as K
    v, grads = S._conv_inputs(x, 2, 37, 48, 4, parameters=torch.float32)
    v["weight"], v["bias"] = v["weight"].to(weight), v["bias"].to(bias)
    S._compare(K.causal_conv, O.causal_conv, v, grads, ("y", "state"))


@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, 100.0625), (torch.float16, 70000.0)])
def test_causal_conv_reads_a_bias_in_its_own_bits(dtype, value):
    """bias - value + x: what a bias of 16 bits would lose is all that is left."""
    from rwkv_wkv_hip import ssm as K
    whole = 100.0 if dtype == torch.bfloat16 else 65504.0
    x = torch.ones(1, 3, 8, dtype=dtype, device="cuda")
    y, _ = K.causal_conv(x, torch.tensor([0.0, -whole], dtype=dtype, device="cuda").expand(8, 2), torch.full((8,), value, device="cuda"), silu=False)
    assert (y.float() == value - whole).all()


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_a_state_leaves_in_32_bits(T, dtype):
    """Whatever type the state comes in; its gradient goes back in that type."""
    from rwkv_wkv_hip import ssm as K
    v, grads = S._scan_inputs(torch.float32, 2, T, 24, 16)
    v["state"] = v["state"].to(dtype)
    c = S._cuda(v, leaf=False)
    y, s = K.selective_scan(**c)
    ref = O.selective_scan(**{n: t.double() for n, t in v.items()})
    assert s.dtype == torch.float32
    assert_close(s, ref[1], RTOL[torch.float32])
    assert_close(y, ref[0], RTOL[torch.float32])
    got, want = S._cuda(v), S._double(v)
    torch.autograd.backward(list(K.selective_scan(**got)), [a.cuda() for a in grads])
    torch.autograd.backward(list(O.selective_scan(**want)), [a.double() for a in grads])
    assert got["state"].grad.dtype == dtype
    assert_close(got["state"].grad, want["state"].grad, RTOL[torch.bfloat16 if dtype == torch.bfloat16 else torch.float32])


# ---- sampling
def test_sampling_refuses_logits_that_want_a_gradient():
    from rwkv_wkv_hip import WKVError, sampling
    l, u = torch.randn(2, 9, device="cuda", requires_grad=True), torch.rand(2, device="cuda")
    with pytest.raises(WKVError):
        sampling.sample(l, u)
    want = sampling.sample(l.detach(), u)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(sampling.sample(l, u), want))


@pytest.mark.parametrize("dtype", S.TYPES)
def test_zeros_of_both_signs_are_the_likeliest_alike(dtype):
    """In every order, within a lane's piece and in different lanes' and wavefronts'."""
    from tests.test_gpu_sampling import _check
    rows = []
    for zeros in ([0.0, -0.0, -1.0], [-0.0, 0.0, -1.0], [-0.0, -1.0, -0.0], [-1.0, -0.0, 0.0]):
        for apart in (1, 8, 512, 3000):
            row = torch.full((9001,), -5.0)
            row[0:3 * apart:apart] = torch.tensor(zeros)
            rows.append(row)
    l = torch.stack(rows).to(dtype)
    assert torch.signbit(l[l == 0]).any() and not torch.signbit(l[l == 0]).all()
    u = torch.linspace(0, 0.999, len(l))
    for k in (dict(), dict(top_k=2), dict(top_p=0.5), dict(temperature=0.0)):
        _check(l, u, **k)
        _check(l, u.flip(0), **k)


# ---- the forms that many rows, tokens and sequences take
@pytest.mark.parametrize("dtype,N,apart", [(torch.bfloat16, 16, 0), (torch.bfloat16, 16, 1), (torch.float32, 16, 0), (torch.float16, 20, 0), (torch.bfloat16, 8, 3)])
@pytest.mark.parametrize("ragged", [False, True])
def test_single_tokens_of_many_sequences(dtype, N, apart, ragged):
    """Four sequences to a lane, the last lanes with two; B and C at an offset that allows no whole loads; sequences without a token; the state in place."""
    from rwkv_wkv_hip import ssm as K
    B, D = 66, 8200 if N == 8 else 4100
    v, _ = S._scan_inputs(dtype, B, 1, D, N, lengths=[i % 3 != 1 for i in range(B)] if ragged else None)
    ref = O.selective_scan(**{n: t.double() if t.is_floating_point() else t for n, t in v.items()})
    c = S._cuda(v, leaf=False)
    wide = torch.zeros(B, 1, 2 * N + 4, dtype=dtype, device="cuda")
    for n, at in (("B", apart), ("C", apart + N)):
        wide[..., at:at + N] = c[n][:, :, 0]
        c[n] = wide[..., at:at + N]
    for out in K.selective_scan(**c), K.selective_scan(**c, out_state=c["state"]):
        for a, b in zip(out, ref):
            assert_close(a, b, RTOL[a.dtype])
    assert out[1].data_ptr() == c["state"].data_ptr()


def _conv_in_64_bits(x, weight, bias, state, lengths):
    W, T = weight.shape[1], x.shape[1]
    live = (torch.arange(T, device=x.device) < lengths[:, None])[..., None]
    xx = torch.cat([state, torch.where(live, x, 0.0)], 1)
    pre = bias + sum(weight[:, k] * xx[:, k:k + T] for k in range(W))
    rows = (lengths[:, None] + torch.arange(W - 1, device=x.device))[..., None].expand_as(state)
    return torch.where(live, pre * torch.sigmoid(pre), 0.0), xx.gather(1, rows)


@pytest.mark.parametrize("dtype,B,T,D,W", [(torch.bfloat16, 8, 1061, 4096, 4), (torch.float32, 8, 1000, 2046, 3), (torch.float16, 8, 1061, 1023, 4), (torch.bfloat16, 8, 300, 4096, 2),
                                           (torch.bfloat16, 8, 530, 4096, 4)])
def test_causal_conv_by_long_runs(dtype, B, T, D, W):
    """16 to 64 tokens to a lane, the sequences' ends and the last run's anywhere in a run; forward and backward, of four channels to a lane, two and one."""
    from rwkv_wkv_hip import ssm as K
    g = S._g(B, T, D, W)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    v = dict(x=r(B, T, D), weight=r(D, W) * 0.5, bias=r(D), state=r(B, W - 1, D))
    lengths = torch.tensor([T, 0, 1, 63, 64, 129, T - 1, T], device="cuda")
    gy, gs = r(B, T, D), r(B, W - 1, D)
    leaf, want = ({n: f(t).detach().requires_grad_(True) for n, t in v.items()} for f in (torch.clone, torch.Tensor.double))
    out, ref = K.causal_conv(**leaf, lengths=lengths), _conv_in_64_bits(**want, lengths=lengths)
    got, exact = (torch.autograd.grad(list(o), list(l.values()), [gy.to(o[0].dtype), gs.to(o[0].dtype)]) for o, l in ((out, leaf), (ref, want)))
    for a, b, n in zip([*out, *got], [*ref, *exact], ["y", "state", *v]):
        # (a parameter's gradient is a sum over 8 T tokens: fp32 errors of their magnitudes, not of the sum's)
        assert_close(a, b, RTOL[a.dtype] if n not in ("weight", "bias") else max(RTOL[a.dtype], 2e-4), n)


@pytest.mark.parametrize("rows,C", [(2500, 1032), (2500, 1030), (2500, 1029), (2500, 777), (2500, 2048), (1100, 2560), (1100, 6002), (1100, 4097), (1100, 8200), (5000, 1000)])
def test_rms_norm_of_more_rows_than_workgroups(rows, C):
    """Each workgroup of the backward takes several rows, one after another."""
    S.test_rms_norm(torch.bfloat16, torch.float32, rows, C)


# ---- sums over many tokens
def test_gradient_of_A_over_many_tokens():
    """2048 tokens that are all alike, of a width at which no sequence is cut: every token adds the same to gA, so that a running sum's roundings go one way.  A tile's
    16 are added up first: 16 + 128 roundings in a row, of 2^-24 each, are 8.6e-6 at the most; the terms themselves, whose state and gradient are fixed points of
    recurrences that forget three quarters and more per token, have some 2e-6.  One after another they would have 2048 roundings."""
    from rwkv_wkv_hip import ssm as K
    T, D, N = 2048, 16384, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.rand(*s, device="cuda", generator=g)
    x, raw, gy, b, c = r(1, 1, D) + 0.5, r(1, 1, D) + 1.0, r(1, 1, D) + 0.5, r(1, 1, N) + 0.5, r(1, 1, N) + 0.5
    A = (-1.0 - r(D, N)).requires_grad_(True)
    wide = lambda t: t.expand(1, T, -1)
    y, _ = K.selective_scan(wide(x), wide(raw), A, wide(b), wide(c))
    got, = torch.autograd.grad(y, A, wide(gy))
    with torch.no_grad():
        step = torch.nn.functional.softplus(raw[0, 0].double())[:, None]
        a = torch.exp(step * A.double())
        u, v = step * x[0, 0].double()[:, None] * b[0, 0].double(), c[0, 0].double() * gy[0, 0].double()[:, None]
        # h[t] = u (1 - a^t) / (1 - a), its gradient v (1 - a^(T-t+1)) / (1 - a); gA = step sum over t of g[t] a h[t-1]
        t = torch.arange(1, T + 1, device="cuda", dtype=torch.float64)
        terms = sum(((1 - a ** (T - k + 1)) * (1 - a ** (k - 1)) for k in t.tolist()[:40] + t.tolist()[-40:])) + (T - 80)          # (a^40 < 2^-53)
        want = step * u * v * a * terms / (1 - a) ** 2
    assert_close(got / want, torch.ones_like(want), 6e-6)          # (taken twice: of the value and of the root mean square)


def test_gradients_of_a_state_that_forgets_everything():
    """A = -infinity gives what an A gives that is finite and whose every exponential is zero: autograd through the definition would multiply zeros by infinities."""
    from rwkv_wkv_hip import ssm as K
    runs = []
    for a in (-math.inf, -1e30):
        v, grads = S._scan_inputs(torch.float32, 2, 40, 24, 16, lengths=[23, 40])
        v["A"][3, 1], v["A"][7] = a, a
        c = S._cuda(v)
        out = K.selective_scan(**c)
        torch.autograd.backward(list(out), [g.cuda() for g in grads])
        runs.append([*out, *(c[n].grad for n in c if n != "lengths")])
    for a, b in zip(*runs):
        assert torch.isfinite(a).all() and torch.equal(a, b)
