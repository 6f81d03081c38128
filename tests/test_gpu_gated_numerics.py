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


@pytest.mark.parametrize("T", [1, 2, 140])
def test_a_gate_far_shut_leaves_zero(T):
    """h silu(z) of a large state and a gate far below zero: silu(z) is zero there, whatever h z would be.  A single token gives what a prompt gives."""
    D = 70
    z = torch.full((1, T, D), -1e10, device="cuda")
    zero = torch.zeros(1, T, D, device="cuda")
    y, h = _kernels().gated_recurrence(zero, torch.full_like(zero, -200.0), zero, torch.zeros(D, device="cuda"), z=z, state=torch.full((1, D), 1e30, device="cuda"))
    assert bool((y == 0).all()) and bool((h == 1e30).all())


@pytest.mark.parametrize("T", [1, 2, 140])
def test_a_gate_far_shut_takes_no_gradient(T):
    """The same backwards: silu's slope is zero there, and gy h, which fp32 does not hold, is never formed."""
    D = 70
    full = lambda v: torch.full((1, T, D), v, device="cuda")
    leaf = [t.requires_grad_(True) for t in (full(1.0), full(-200.0), full(0.0), full(-1e10), torch.full((1, D), 1e30, device="cuda"))]
    x, r, i, z, state = leaf
    y, _ = _kernels().gated_recurrence(x, r, i, torch.zeros(D, device="cuda"), z=z, state=state)
    for t in torch.autograd.grad(y, leaf, full(1e10)):
        assert bool((t == 0).all())


@pytest.mark.parametrize("T", [1, 2, 140])
@pytest.mark.parametrize("which", ["r", "i"])
def test_a_gate_at_its_end_takes_no_gradient(T, which):
    """A shut r keeps a large state, an open i lets a large input through: the sigmoid's slope is zero, and the incoming gradient times the state or the input, which fp32 does not
    hold, is never formed."""
    D = 70
    full = lambda v: torch.full((1, T, D), v, device="cuda")
    shut = which == "r"
    x, r, i = (t.requires_grad_(True) for t in (full(0.0 if shut else 1e30), full(-200.0 if shut else 2.0), full(0.0 if shut else 200.0)))
    decay = torch.full((D,), 3.0, device="cuda", requires_grad=True)
    y, _ = _kernels().gated_recurrence(x, r, i, decay, state=torch.full((1, D), 1e30, device="cuda") if shut else None)
    grads = torch.autograd.grad(y, (r, decay) if shut else (i,), full(1e10))
    for t in grads:
        assert bool((t == 0).all())


def _slopes(x, wg, wu, gy):
    """In 64 bits, for silu: dg and du and what fp32 leaves of them: g and u are fp32 sums (c of their terms' sizes), slopes and slopes' slopes below 1.2."""
    g, u = x @ wg.t(), x @ wu.t()
    p = torch.sigmoid(g)
    act, slope = g * p, p * (1 + g * (1 - p))
    c = (x.shape[1] + 32) * 2.0 ** -23
    G, U = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()
    off_g = gy.abs() * (1.2 * c * (U + G * u.abs() + c * G * U) + 2.0 ** -20 * u.abs())
    return gy * u * slope, gy * act, off_g, gy.abs() * (1.2 * c * G + 2.0 ** -20 * act.abs())


@pytest.mark.parametrize("R,C,F", [(1, 72, 200), (20, 99, 130), (32, 256, 515), (33, 256, 515), (300, 72, 1030), (700, 520, 1100)])
@pytest.mark.parametrize("size", [1e-7, 1e-5, 1e-3, 3e4])
@pytest.mark.parametrize("wide", [2.0 ** -5, 2.0 ** 5])
def test_fp16_slopes_have_the_range_of_fp32(R, C, F, size, wide):
    """Gradients coming in small as a mean loss' or as large as fp16 goes; the slopes between are no results, and neither overflow nor underflow shows.  ``wide`` scales the weights up
    and x down, so that one of the two kinds of results has fp16's normal range where the slopes themselves have not.

    An element: its rounding, 2^-11 or 2^-25; the slopes' rounding 2^-11, or of two parts 2^-22, and 2^-39 of the largest slope where that leaves fp16's normal
    range (2^-25 of 2^14); fp32 sums.  What is past fp16's largest number is infinite, as any result."""
    K = _kernels()
    g = S._g(R, C, F)
    n = lambda *s: torch.randn(*s, generator=g)
    x = (n(R, C) / wide).half()
    wg, wu = ((n(F, C) * (wide / C ** 0.5)).half() for _ in range(2))
    gy = (n(R, F).clamp(-2, 2) * size).half()
    leaf = [t.cuda().requires_grad_(True) for t in (x, wg, wu)]
    got = torch.autograd.grad(K.gated_feed_forward(*leaf), leaf, gy.cuda())
    x, wg, wu, gy = (t.double() for t in (x, wg, wu, gy))
    dg, du, off_g, off_u = _slopes(x, wg, wu, gy)
    e = 2.0 ** -22 if R <= 32 else 2.0 ** -11
    tiny = 2.0 ** -39 * torch.stack([dg.abs().max(), du.abs().max()]).max()
    bad_g, bad_u = (e * d.abs() + tiny + (1 + e) * o for d, o in ((dg, off_g), (du, off_u)))
    sums = lambda terms: (terms + 32) * 2.0 ** -23 * (1 + e)
    for name, a, ref, size_, off in (("x", got[0], dg @ wg + du @ wu, dg.abs() @ wg.abs() + du.abs() @ wu.abs(), bad_g @ wg.abs() + bad_u @ wu.abs()),
                                     ("w_gate", got[1], dg.t() @ x, dg.t().abs() @ x.abs(), bad_g.t() @ x.abs()), ("w_up", got[2], du.t() @ x, du.t().abs() @ x.abs(), bad_u.t() @ x.abs())):
        a, wrong = a.cpu().double(), off + sums(2 * F if name == "x" else R) * (size_ + off)
        bound = 2.0 ** -11 * ref.abs() + (1 + 2.0 ** -11) * wrong + 2.0 ** -25
        inside, outside = ref.abs() + wrong < 65504, ref.abs() - wrong > 65536
        worst = ((a - ref).abs() / bound)[inside].max().item() if inside.any() else 0.0
        assert worst <= 1, f"gradient of {name}: {worst:.3g} of the bound"          # (NaN is not)
        assert bool((a == ref.sign() * float("inf"))[outside].all()), f"gradient of {name} past fp16"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R", [1, 7, 32, 40])
def test_an_infinite_gradient_is_infinite(dtype, R):
    """One place's incoming gradient is infinite: what it reaches is infinite of the sign that the formula gives (NaN only where the formula adds both signs), the rest is
    finite and off by no more than the test above allows: both roundings, the slopes' in two parts up to 32 rows, fp32 sums, and g and u from fp32 sums."""
    K = _kernels()
    C, F = 96, 70
    g = S._g(R, 3)
    x, wg, wu, gy = (torch.randn(*s, generator=g).to(dtype) for s in ((R, C), (F, C), (F, C), (R, F)))
    gy[R // 2, 5] = float("inf")
    leaf = [t.cuda().requires_grad_(True) for t in (x, wg, wu)]
    got = torch.autograd.grad(K.gated_feed_forward(*leaf), leaf, gy.cuda())
    x, wg, wu, gy = (t.double() for t in (x, wg, wu, gy))
    dg, du, off_g, off_u = _slopes(x, wg, wu, gy)
    e = torch.finfo(dtype).eps / 2
    finite = lambda t: torch.where(torch.isfinite(t), t, 0.0).abs()
    bad_g, bad_u = ((e * e if R <= 32 else e) * finite(d) + 2 * finite(o) for d, o in ((dg, off_g), (du, off_u)))
    each = lambda p, q: (p @ wg.abs() + q @ wu.abs(), p.t() @ x.abs(), q.t() @ x.abs())
    for a, ref, size, off in zip(got, (dg @ wg + du @ wu, dg.t() @ x, du.t() @ x), each(finite(dg), finite(du)), each(bad_g, bad_u)):
        a = a.cpu().double()
        assert torch.equal(a.isnan(), ref.isnan()) and torch.equal(a.isinf(), ref.isinf()) and bool((a == ref)[ref.isinf()].all())
        bound = e * ref.abs() + (1 + e) * (off + (2 * F + 32) * 2.0 ** -23 * (size + off)) + 2.0 ** -24
        assert bool(((a - ref).abs() <= bound)[torch.isfinite(ref)].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("R", [3, 50])
def test_a_shut_unit_takes_no_gradient(dtype, name, R):
    """g far below zero: value and slope of the activation are zero, and gy u, which fp32 does not hold, is never formed."""
    C, F = 16, 24
    x, wg = torch.ones(R, C, dtype=dtype, device="cuda"), torch.full((F, C), -1e4, dtype=dtype, device="cuda")
    wu = torch.full((F, C), 1e30, dtype=dtype, device="cuda")
    leaf = [t.requires_grad_(True) for t in (x, wg, wu)]
    y = _kernels().gated_feed_forward(*leaf, name)
    assert bool((y == 0).all())
    for t in torch.autograd.grad(y, leaf, torch.full_like(y, 1e10)):
        assert bool((t == 0).all())


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -2.0])
@pytest.mark.parametrize("C", [16, 7])
def test_a_place_without_a_token_is_zero_whatever_the_scale(dtype, scale, C):
    """The others are the scale times their rows; a zero without a sign where there is no token."""
    tokens = torch.tensor([0, -1, 2, 3, -100, 1], device="cuda")
    w = torch.arange(1, 3 * C + 1, device="cuda").view(3, C).to(dtype)
    out = _kernels().embedding(tokens, w, scale)
    none = (tokens < 0) | (tokens >= 3)
    assert bool((out[none] == 0).all()) and not out[none].signbit().any()
    assert torch.equal(out[~none], (w[tokens[~none]].float() * scale).to(dtype)) or (scale != scale and out[~none].isnan().all())


@pytest.mark.parametrize("first", [0, 1, 5, 8, 13])
def test_embedding_sums_by_runs_of_the_sorted_places(first):
    """Three tokens, of which the first's count moves the borders of the others' runs: up to 4096 places of up to 1024 channels, fp32 sums of 8 sorted places at a time, in order, added in
    order.  Values whose sums depend on the grouping."""
    n = torch.tensor([2.0 ** 30, 1.0, -2.0 ** 30, 3.0, 2.0 ** 29])
    tokens = torch.cat([torch.zeros(first, dtype=torch.long), torch.tensor([1, 2, 1]).repeat(31), torch.tensor([-1, 3])])
    gy = n.repeat(len(tokens))[:len(tokens)].repeat_interleave(8).view(-1, 8).contiguous()

    def runs(tokens, gy):
        order = torch.where((tokens >= 0) & (tokens < 3), tokens, 3).argsort(stable=True)
        total = torch.zeros(3, 8)
        for at in range(0, len(order), 8):
            sums = {}
            for p in order[at:at + 8].tolist():
                t = int(tokens[p])
                if 0 <= t < 3:
                    sums[t] = sums[t] + gy[p] if t in sums else gy[p].clone()
            for t, s in sums.items():
                total[t] += s
        return total

    w = torch.zeros(3, 8, device="cuda", requires_grad=True)
    (a,) = torch.autograd.grad(_kernels().embedding(tokens.cuda(), w), w, gy.cuda())
    assert torch.equal(a.cpu(), runs(tokens, gy))


def test_embedding_sums_are_grouped_by_the_whole_call():
    """The grouping that the documentation states, by a case small enough to follow: 2^30, 1, -2^30, 1 and six zeros before them of another token.  Alone they lie in one run: 2^30 + 1 is 2^30 in fp32, so 1
    is left.  Behind six others the run of 8 ends after the 1: 2^30 and then (-2^30 + 1 = -2^30): nothing is left."""
    K = _kernels()
    w = torch.zeros(2, 8, device="cuda", requires_grad=True)
    gy = torch.tensor([0.0] * 6 + [2.0 ** 30, 1.0, -2.0 ** 30, 1.0]).repeat_interleave(8).view(-1, 8).cuda()
    tokens = torch.tensor([0] * 6 + [1] * 4, device="cuda")
    (alone,) = torch.autograd.grad(K.embedding(tokens[6:], w), w, gy[6:].contiguous())
    (behind,) = torch.autograd.grad(K.embedding(tokens, w), w, gy)
    assert bool((alone[1] == 1).all()) and bool((behind[1] == 0).all()) and not behind[0].any()


@pytest.mark.parametrize("dtype", S.TYPES)
def test_a_recorded_single_token_reads_itself_alone(dtype):
    """A call of one token is a call of two that ends after the first, to the bit, whatever is not finite in it: an open gate of plus infinity makes infinite gradients, not NaN."""
    B, D = 2, 66
    g = S._g(B, D)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    x, a, i, z, gy = (r(B, 2, D) for _ in range(5))
    state, decay, gs = torch.randn(B, D, generator=g).cuda(), torch.randn(D, generator=g).cuda(), torch.randn(B, D, generator=g).cuda()
    z[0, 0, ::5] = float("inf")

    def run(T, lengths):
        leaf = [t.clone().requires_grad_(True) for t in (*(v[:, :T] for v in (x, a, i, z)), decay, state)]
        y, new = _kernels().gated_recurrence(*leaf[:3], leaf[4], z=leaf[3], state=leaf[5], lengths=lengths)
        grads = torch.autograd.grad([y, new], leaf, [gy[:, :T].contiguous(), gs])
        return [y[:, :1], new, *(t[:, :1] for t in grads[:4]), *grads[4:]]

    one, two = run(1, None), run(2, torch.ones(B, dtype=torch.int32, device="cuda"))
    for p, q in zip(one, two):
        assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p.nan_to_num(7.0), q.nan_to_num(7.0))
    assert one[2][0, 0, ::5].isinf().all() and torch.isfinite(one[2][1].float()).all()


@pytest.mark.parametrize("R", [5, 90])
def test_fp16_slopes_scale_with_what_a_replay_holds(R):
    """A captured training call finds its power of two on every replay: gradients that come in 2^-20 and 2^12 times as large give what the eager call gives, to the bit."""
    K = _kernels()
    g = S._g(R, 8)
    n = lambda *s: torch.randn(*s, generator=g).half().cuda()
    leaf = [t.requires_grad_(True) for t in (n(R, 64), n(48, 64) / 8, n(48, 64) / 8)]
    leaf = [t.detach().requires_grad_(True) for t in leaf]
    gy, base = n(R, 48), n(R, 48)
    step = lambda: torch.autograd.grad(K.gated_feed_forward(*leaf), leaf, gy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for power in (0, -20, 12, -20):
        gy.copy_((base.float() * 2.0 ** power).half())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and b.any()
