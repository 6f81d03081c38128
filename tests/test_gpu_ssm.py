"""The state space operators on the HIP kernels against the oracle in 64 bits (oracle/ssm.py, gradients by autograd through it).

Tolerances, of |ref| + rms(ref) per element.  The oracle has the same (rounded) inputs in 64 bits, so what is off is the kernels' fp32 arithmetic and
the rounding of an output to its type: bf16 2^-9 and fp16 2^-11 of a value, taken twice; fp32 arithmetic: decays and exponentials
are right to a few 2^-23, and over the few hundred tokens here at most their sum, some 5e-5, taken twice."""
import pytest
import torch

from oracle import ssm as O
from tests.util import assert_close

pytestmark = pytest.mark.gpu
RTOL = {torch.float32: 1e-4, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _g(*seed):
    n = 17
    for s in seed:
        n = n * 1009 + int(s)
    return torch.Generator().manual_seed(n % (1 << 31))


def _double(v):
    return {n: t.double().requires_grad_(True) if torch.is_tensor(t) and t.is_floating_point() else t for n, t in v.items()}


def _cuda(v, leaf=True):
    return {n: t.cuda().requires_grad_(leaf and t.is_floating_point()) if torch.is_tensor(t) else t for n, t in v.items()}


def _compare(kernel, oracle, v, grads, names):
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


# ---- the convolution
def _conv_inputs(dtype, B, T, D, W, bias=True, state=True, lengths=None, parameters=None):
    g = _g(B, T, D, W)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    v = dict(x=r(B, T, D), weight=(torch.randn(D, W, generator=g) * 0.5).to(parameters or dtype))
    if bias:
        v["bias"] = torch.randn(D, generator=g).to(parameters or dtype)
    if state:
        v["state"] = r(B, W - 1, D)
    if lengths is not None:
        v["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    return v, [r(B, T, D), r(B, W - 1, D)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D,W", [(1, 1, 64, 4), (2, 2, 24, 4), (1, 3, 1, 3), (2, 7, 33, 2), (3, 65, 520, 4), (1, 257, 512, 3), (2, 130, 130, 4)])
def test_causal_conv(dtype, B, T, D, W):
    from rwkv_wkv_hip import ssm as K
    v, grads = _conv_inputs(dtype, B, T, D, W)
    _compare(K.causal_conv, O.causal_conv, v, grads, ("y", "state"))


@pytest.mark.parametrize("options", [dict(bias=False), dict(state=False), dict(bias=False, state=False), dict(parameters=torch.float32)])
@pytest.mark.parametrize("silu", [True, False])
def test_causal_conv_options(options, silu):
    from rwkv_wkv_hip import ssm as K
    v, grads = _conv_inputs(torch.bfloat16, 2, 37, 48, 4, **options)
    _compare(lambda **k: K.causal_conv(silu=silu, **k), lambda **k: O.causal_conv(silu=silu, **k), v, grads, ("y", "state"))


@pytest.mark.parametrize("T,lengths", [(70, [0, 1, 70]), (70, [2, 3, 64]), (4, [1, 2, 4]), (1, [0, 1, 1])])
@pytest.mark.parametrize("state", [True, False])
def test_causal_conv_lengths(T, lengths, state):
    """What lies behind a sequence's end is not read: there it is NaN on the GPU, zero in the oracle."""
    from rwkv_wkv_hip import ssm as K
    v, grads = _conv_inputs(torch.float32, 3, T, 40, 4, state=state, lengths=lengths)
    behind = torch.arange(T)[None, :, None] >= v["lengths"][:, None, None]

    def kernel(x, **k):
        return K.causal_conv(torch.where(behind.cuda(), torch.nan, x), **k)

    _compare(kernel, O.causal_conv, v, grads, ("y", "state"))


# ---- the scan
def _scan_inputs(dtype, B, T, D, N, G=1, gate=True, skip=True, bias=True, state=True, lengths=None, flat=False):
    g = _g(B, T, D, N, G)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    vectors = (B, T, N) if flat else (B, T, G, N)
    v = dict(x=r(B, T, D), dt=(torch.randn(B, T, D, generator=g) - 1).to(dtype), A=-torch.rand(D, N, generator=g) * 4 - 0.01, B=r(*vectors), C=r(*vectors))
    if gate:
        v["z"] = r(B, T, D)
    if skip:
        v["D"] = torch.randn(D, generator=g)
    if bias:
        v["dt_bias"] = torch.randn(D, generator=g)
    if state:
        v["state"] = torch.randn(B, D, N, generator=g)
    if lengths is not None:
        v["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    return v, [r(B, T, D), torch.randn(B, D, N, generator=g)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D,N,G", [(1, 1, 64, 16, 1), (2, 2, 5, 16, 1), (1, 16, 32, 16, 1), (2, 17, 33, 16, 1), (1, 130, 96, 16, 2), (3, 40, 6, 1, 3),
                                       (1, 300, 20, 8, 1), (2, 33, 40, 24, 2), (1, 290, 36, 32, 1), (1, 50, 10, 64, 1), (2, 35, 12, 61, 2)])
def test_selective_scan(dtype, B, T, D, N, G):
    from rwkv_wkv_hip import ssm as K
    v, grads = _scan_inputs(dtype, B, T, D, N, G)
    _compare(K.selective_scan, O.selective_scan, v, grads, ("y", "state"))


@pytest.mark.parametrize("options", [dict(gate=False), dict(skip=False), dict(bias=False), dict(state=False), dict(flat=True),
                                     dict(gate=False, skip=False, bias=False, state=False)])
@pytest.mark.parametrize("T", [1, 37, 270])
def test_selective_scan_options(options, T):
    from rwkv_wkv_hip import ssm as K
    v, grads = _scan_inputs(torch.float32, 2, T, 24, 16, **options)
    _compare(K.selective_scan, O.selective_scan, v, grads, ("y", "state"))


@pytest.mark.parametrize("T,lengths", [(300, [0, 1, 300]), (300, [16, 17, 255]), (40, [39, 0, 20]), (1, [0, 1, 1])])
def test_selective_scan_lengths(T, lengths):
    from rwkv_wkv_hip import ssm as K
    v, grads = _scan_inputs(torch.float32, 3, T, 18, 16, lengths=lengths)
    behind = torch.arange(T)[None, :, None] >= v["lengths"][:, None, None]

    def kernel(x, dt, z, B, C, **k):
        spoil = lambda t: torch.where(behind.cuda() if t.dim() == 3 else behind.cuda()[..., None], torch.nan, t)
        return K.selective_scan(spoil(x), spoil(dt), z=spoil(z), B=spoil(B), C=spoil(C), **k)

    _compare(kernel, O.selective_scan, v, grads, ("y", "state"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,N", [(1, 8, 16), (3, 37, 4), (2, 65, 8), (5, 12, 32), (2, 9, 64), (2, 7, 1), (3, 11, 20), (2, 6, 50)])
def test_single_token_without_a_gradient(dtype, B, D, N):
    """The kernel of its own, also with the state updated in place."""
    from rwkv_wkv_hip import ssm as K
    v, _ = _scan_inputs(dtype, B, 1, D, N)
    ref = O.selective_scan(**{n: t.double() for n, t in v.items()})
    c = _cuda(v, leaf=False)
    for out in K.selective_scan(**c), K.selective_scan(**c, out_state=c["state"]):
        for a, b in zip(out, ref):
            assert_close(a, b, RTOL[a.dtype])
    assert out[1].data_ptr() == c["state"].data_ptr()
    v, _ = _conv_inputs(dtype, B, 1, D, 4)
    ref = O.causal_conv(**{n: t.double() for n, t in v.items()})
    c = _cuda(v, leaf=False)
    for out in K.causal_conv(**c), K.causal_conv(**c, out_state=c["state"]):
        for a, b in zip(out, ref):
            assert_close(a, b, RTOL[a.dtype])


def test_tokens_one_by_one_are_the_prompt():
    from rwkv_wkv_hip import ssm as K
    v, _ = _scan_inputs(torch.float32, 2, 20, 24, 16)
    c = _cuda(v, leaf=False)
    whole, end = K.selective_scan(**c)
    s = c["state"].clone()
    for t in range(20):
        one = {n: a[:, t:t + 1] if n in ("x", "dt", "z", "B", "C") else a for n, a in c.items() if n != "state"}
        y, s = K.selective_scan(**one, state=s, out_state=s)
        assert_close(y, whole[:, t:t + 1], RTOL[torch.float32])
    assert_close(s, end, RTOL[torch.float32])


@pytest.mark.parametrize("B,T,D,N", [(1, 2048, 24, 16), (1, 1000, 100, 16), (2, 1030, 8, 40)])
def test_few_channels_and_many_tokens(B, T, D, N):
    """Sequences that are cut in time."""
    from rwkv_wkv_hip import ssm as K
    v, grads = _scan_inputs(torch.float32, B, T, D, N)
    _compare(K.selective_scan, O.selective_scan, v, grads, ("y", "state"))


def test_slow_decays_do_not_drift():
    """Steps of 0.001 and A = -1: a thousand tokens are remembered, and their decays' errors must not add up in one direction."""
    from rwkv_wkv_hip import ssm as K
    g = _g(3)
    B, T, D, N = 1, 3000, 16, 16
    v = dict(x=torch.rand(B, T, D, generator=g), dt=torch.full((B, T, D), -6.907), A=-torch.ones(D, N), B=torch.ones(B, T, 1, N), C=torch.ones(B, T, 1, N))
    ref = O.selective_scan(**{n: t.double() for n, t in v.items()})
    y, s = K.selective_scan(**_cuda(v, leaf=False))
    assert_close(s, ref[1], 2e-5)
    assert_close(y, ref[0], 2e-5)


def test_strided_operands():
    """Slices of wider tensors at any offset, as projections leave them; gradients flow into the wide tensors."""
    from rwkv_wkv_hip import ssm as K
    g = _g(5)
    B, T, D, N, R = 2, 21, 40, 16, 3
    v = dict(xz=torch.randn(B, T, 2 * D + 1, generator=g), low=torch.randn(T, B, D, generator=g), bc=torch.randn(B, T, R + 2 * N, generator=g),
             A=-torch.rand(D, N, generator=g), state=torch.randn(D, B, N, generator=g))

    def split(fn):
        def call(xz, low, bc, A, state):
            return fn(xz[..., 1:D + 1], low.transpose(0, 1), A, bc[..., R:R + N], bc[..., R + N:], z=xz[..., D + 1:], state=state.transpose(0, 1))
        return call

    grads = [torch.randn(B, T, D, generator=g), torch.randn(B, D, N, generator=g)]
    _compare(split(K.selective_scan), split(O.selective_scan), v, grads, ("y", "state"))
    w = torch.randn(D, 4, generator=g)
    v = dict(xz=torch.randn(B, T, 2 * D, generator=g).bfloat16(), w=w.bfloat16())
    conv = lambda fn: lambda xz, w: fn(xz[..., D:], w)
    _compare(conv(K.causal_conv), conv(O.causal_conv), v, [torch.randn(B, T, D, generator=g).bfloat16(), torch.randn(B, 3, D, generator=g).bfloat16()], ("y", "state"))


def test_broadcast_inputs_get_summed_gradients():
    """One B and C for the batch, one time step for the channels (expanded tensors of stride zero)."""
    from rwkv_wkv_hip import ssm as K
    g = _g(7)
    B, T, D, N = 3, 19, 24, 16
    v = dict(x=torch.randn(B, T, D, generator=g), dt=torch.randn(B, T, 1, generator=g), A=-torch.rand(1, N, generator=g), b=torch.randn(T, N, generator=g), c=torch.randn(T, N, generator=g))
    wide = lambda fn: lambda x, dt, A, b, c: fn(x, dt.expand(B, T, D), A.expand(D, N), b.expand(B, T, N), c.expand(B, T, N))
    _compare(wide(K.selective_scan), wide(O.selective_scan), v, [torch.randn(B, T, D, generator=g), torch.randn(B, D, N, generator=g)], ("y", "state"))


@pytest.mark.parametrize("op", ["scan", "conv", "norm"])
def test_gradients_against_differences(op):
    """Along random directions, the kernels' gradient against central differences of the 64-bit definition (their own error: 1e-8)."""
    from rwkv_wkv_hip import ssm as K
    if op == "scan":
        v, grads = _scan_inputs(torch.float32, 2, 50, 12, 16, 2)
        kernel, oracle = K.selective_scan, O.selective_scan
    elif op == "conv":
        v, grads = _conv_inputs(torch.float32, 2, 50, 24, 4)
        kernel, oracle = K.causal_conv, O.causal_conv
    else:
        g = _g(11)
        r = lambda *s: torch.randn(*s, generator=g)
        v, grads = dict(x=r(6, 40), weight=r(40), residual=r(6, 40)), [r(6, 40), r(6, 40)]
        kernel, oracle = (lambda **k: K.rms_norm(k["x"], k["weight"], 1e-5, k["residual"])), (lambda **k: O.rms_norm(k["x"], k["weight"], 1e-5, k["residual"]))
    got = _cuda(v)
    torch.autograd.backward(list(kernel(**got)), [a.cuda() for a in grads])
    value = lambda w: sum((a * b.double()).sum() for a, b in zip(oracle(**w), grads))
    g = _g(13)
    for n, t in v.items():
        along = torch.randn(t.shape, generator=g).double()
        at = lambda e: value({m: u.double() + (e * along if m == n else 0) for m, u in v.items()})
        want = float(at(1e-5) - at(-1e-5)) / 2e-5
        have = float((got[n].grad.cpu().double() * along).sum())
        size = float((got[n].grad.cpu().double().abs() * along.abs()).sum())
        assert abs(have - want) <= 1e-5 * size + 1e-6 * abs(want), (n, have, want)


def test_nothing_comes_back_where_nothing_goes_in():
    """No gradient of the outputs or of the state alone; a state handed on without one."""
    from rwkv_wkv_hip import ssm as K
    v, grads = _scan_inputs(torch.float32, 1, 20, 8, 16)
    for which in (0, 1):
        want, got = _double(v), _cuda(v)
        ref, out = O.selective_scan(**want), K.selective_scan(**got)
        ref[which].backward(grads[which].double())
        out[which].backward(grads[which].cuda())
        for n in v:
            r = want[n].grad if want[n].grad is not None else torch.zeros_like(want[n])
            assert_close(got[n].grad, r, RTOL[torch.float32], n)


def test_results_repeat_to_the_bit():
    from rwkv_wkv_hip import ssm as K
    v, grads = _scan_inputs(torch.bfloat16, 2, 700, 200, 16)
    runs = []
    for _ in range(3):
        c = _cuda(v)
        out = K.selective_scan(**c)
        torch.autograd.backward(list(out), [g.cuda() for g in grads])
        runs.append([*out, *(t.grad for t in c.values())])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


def test_non_finite_values_stay_in_their_channel():
    from rwkv_wkv_hip import ssm as K
    v, _ = _scan_inputs(torch.float32, 2, 40, 24, 16)
    v["x"][0, 7, 3] = torch.nan
    v["dt"][1, 9, 5] = torch.inf
    c = _cuda(v, leaf=False)
    y, s = K.selective_scan(**c)
    ref = O.selective_scan(**{n: t.double() for n, t in v.items()})
    assert torch.equal(torch.isfinite(y).cpu(), torch.isfinite(ref[0])) and torch.equal(torch.isfinite(s).cpu(), torch.isfinite(ref[1]))
    assert torch.isfinite(y[0, :7]).all() and not torch.isfinite(y[0, 7:, 3]).any()


# ---- the norm
@pytest.mark.parametrize("dtype,residual", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                            (torch.float16, torch.float16), (torch.float16, torch.float32), (torch.bfloat16, None)])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 8), (5, 100), (2, 513), (4, 768), (3, 2048), (2, 2560), (2, 4104), (2, 8200), (1500, 64)])
def test_rms_norm(dtype, residual, rows, C):
    from rwkv_wkv_hip import ssm as K
    g = _g(rows, C)
    r = lambda *s: torch.randn(*s, generator=g)
    v = dict(x=r(rows, C).to(dtype), weight=(r(C) + 1).to(dtype))
    if residual is not None:
        v["residual"] = (2 * r(rows, C)).to(residual)
    gy, gr = r(rows, C).to(dtype), r(rows, C).to(residual or dtype)
    want, got = _double(v), _cuda(v)
    ref, out = O.rms_norm(want["x"], want["weight"], 1e-5, want.get("residual")), K.rms_norm(got["x"], got["weight"], 1e-5, got.get("residual"))
    assert out[1].dtype == (residual or dtype)
    for a, b in zip(out, ref):
        assert_close(a, b, RTOL[a.dtype])
    torch.autograd.backward(list(ref), [gy.double(), gr.double()])
    torch.autograd.backward(list(out), [gy.cuda(), gr.cuda()])
    for n in v:
        # (backwards the sum is the rounded one: its rounding once more)
        assert_close(got[n].grad, want[n].grad, RTOL[v[n].dtype] + (RTOL[residual or dtype] if (residual or dtype) != torch.float32 else 0), n)


@pytest.mark.parametrize("shape,strided", [((2, 3, 40), False), ((4, 64), True), ((64,), False)])
def test_rms_norm_shapes(shape, strided):
    from rwkv_wkv_hip import ssm as K
    g = _g(len(shape))
    x = torch.randn(*shape[:-1], 2 * shape[-1] + 1, generator=g)[..., 1:shape[-1] + 1] if strided else torch.randn(*shape, generator=g)
    res, w = torch.randn(*shape, generator=g), torch.randn(shape[-1], generator=g)
    y, r = K.rms_norm(x.cuda() if not strided else torch.cat([x[..., :1], x, x], -1).cuda()[..., 1:shape[-1] + 1], w.cuda(), 1e-3, res.cuda())
    ref = O.rms_norm(x.double(), w.double(), 1e-3, res.double())
    assert y.shape == x.shape
    assert_close(y, ref[0], RTOL[torch.float32])
    assert_close(r, ref[1], RTOL[torch.float32])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,C", [(1, 8), (3, 100), (4, 768), (2, 2048), (65, 2560), (2, 8200)])
def test_rms_norm_fp8(dtype, rows, C):
    """q * scale against y: half a step of a 4-bit significand (2^-4 of the value; below 2^-6 of the largest of 448, half of 2^-9 scales)."""
    from rwkv_wkv_hip import ssm as K
    g = _g(rows, C, 8)
    x, w = torch.randn(rows, C, generator=g).to(dtype), torch.randn(C, generator=g).to(dtype)
    res = torch.randn(rows, C, generator=g)
    x[0] = 0
    res[0] = 0
    with torch.no_grad():
        q, scale, r = K.rms_norm_fp8(x.cuda(), w.cuda(), 1e-5, res.cuda())
    ref = O.rms_norm(x.double(), w.double(), 1e-5, res.double())[0]
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows, 1) and r.dtype == torch.float32
    top = ref.abs().amax(1, keepdim=True)
    assert_close(scale, torch.where(top > 0, top / 448, 1.0), 1e-5)
    back, s = q.cpu().double() * scale.cpu().double(), scale.cpu().double()
    assert ((back - ref).abs() <= (2.0 ** -4 + 1e-5) * ref.abs() + (2.0 ** -10 + 1e-6) * s).all()
    assert not back[0].any()


# ---- refusals
def test_refusals():
    import rwkv_wkv_hip as W
    from rwkv_wkv_hip import ssm as K
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)
    x, A, b = z(2, 5, 8), z(8, 16), z(2, 5, 16)
    with pytest.raises(AssertionError):
        K.selective_scan(x, x, z(9, 16), b, b)                                   # A of other channels
    with pytest.raises(AssertionError):
        K.selective_scan(x, x, A, b, z(2, 5, 8))                                 # C of other states
    with pytest.raises(AssertionError):
        K.selective_scan(x, x.half(), A, b, b)                                   # two types
    with pytest.raises(AssertionError):
        K.selective_scan(x, x, A, b, b, state=z(2, 8, 8))
    with pytest.raises(ValueError):
        K.selective_scan(x, x, z(8, 65), z(2, 5, 65), z(2, 5, 65))               # too many states
    with pytest.raises(ValueError):
        K.selective_scan(x, x, A, z(2, 5, 3, 16), z(2, 5, 3, 16))                # groups that do not divide the channels
    with pytest.raises(ValueError):
        K.selective_scan(x.double(), x.double(), A, b.double(), b.double())
    with pytest.raises(ValueError):
        K.selective_scan(x[:, :0], x[:, :0], A, b[:, :0], b[:, :0])              # no tokens
    with pytest.raises(W.WKVError):
        K.selective_scan(x, x, A.cpu(), b, b)
    with pytest.raises(W.WKVError):
        s = z(2, 8, 16)
        K.selective_scan(x, x, A, b, b, state=s, out_state=s)                    # in place for single tokens only
    with pytest.raises(AssertionError):
        K.selective_scan(x[:, :1].requires_grad_(True), x[:, :1], A, b[:, :1], b[:, :1], out_state=z(2, 8, 16))
    for taps in (1, 5):
        with pytest.raises(ValueError):
            K.causal_conv(x, z(8, taps))
    with pytest.raises(AssertionError):
        K.causal_conv(x, z(8, 4), state=z(2, 4, 8))
    with pytest.raises(AssertionError):
        K.causal_conv(x, z(8, 4), lengths=z(2))
    with pytest.raises(AssertionError):
        K.rms_norm(x, z(9))
    with pytest.raises(AssertionError):
        K.rms_norm(x, z(8), residual=x.half())
    with pytest.raises(W.WKVError):
        K.rms_norm_fp8(x.requires_grad_(True), z(8))


# ---- streams and graphs
def test_another_stream():
    from rwkv_wkv_hip import ssm as K
    v, _ = _scan_inputs(torch.float32, 2, 300, 24, 16)
    c = _cuda(v, leaf=False)
    want = K.selective_scan(**c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = K.selective_scan(**c)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_single_tokens_in_a_graph():
    """A serving loop's step, its state updated in place, replayed with eager work between the replays."""
    from rwkv_wkv_hip import ssm as K
    v, _ = _scan_inputs(torch.bfloat16, 4, 1, 64, 16)
    c = _cuda(v, leaf=False)
    w, window = torch.randn(64, 4, device="cuda").bfloat16(), torch.randn(4, 3, 64, device="cuda").bfloat16()
    start = c["state"].clone(), window.clone()
    x = c.pop("x")

    def step():
        u, _ = K.causal_conv(x, w, state=window, out_state=window)
        return K.selective_scan(u, **c, out_state=c["state"])[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    xs = [torch.randn_like(x) for _ in range(4)]
    c["state"].copy_(start[0]); window.copy_(start[1])
    eager = []
    for t in xs:
        x.copy_(t)
        eager.append(step().clone())
    c["state"].copy_(start[0]); window.copy_(start[1])
    for t, want in zip(xs, eager):
        x.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_offsets_beyond_32_bits():
    """Sequences, rows and tokens that lie more than 2^32 bytes apart in one buffer give what their copies side by side give."""
    from rwkv_wkv_hip import sampling, ssm as K
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    D, N, far = 64, 16, (1 << 31) + 24            # elements of two bytes: 4 GiB and a little between two sequences
    buffer = torch.empty(far + 64 * 1024, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    view = lambda *s: buffer.as_strided(s, (far,) + tuple(torch.empty(s[1:], device="meta").stride()))
    for T in (1, 40):
        x = view(2, T, 6 * D)
        x.copy_(torch.randn(2, T, 6 * D, device="cuda", generator=g))
        part = lambda t, i, n=D: t[..., i * D:i * D + n]
        A = -torch.rand(D, N, device="cuda", generator=g)
        run = lambda t: K.selective_scan(part(t, 0), part(t, 1), A, part(t, 2, N), part(t, 3, N), z=part(t, 4))
        w = torch.randn(D, 4, device="cuda", generator=g).bfloat16()
        for f in (run, lambda t: K.causal_conv(part(t, 5), w)):
            assert all(torch.equal(a, b) for a, b in zip(f(x), f(x.contiguous())))
    rows = view(2, 300)
    rows.copy_(torch.randn(2, 300, device="cuda", generator=g))
    weight, u = torch.ones(300, device="cuda"), torch.tensor([0.3, 0.8], device="cuda")
    for f in (lambda t: K.rms_norm(t, weight, 1e-5, t), lambda t: sampling.sample(t, u, top_p=0.9)):
        assert all(torch.equal(a, b) for a, b in zip(f(rows), f(rows.contiguous())))
    # 300 tokens of 16 MiB: offsets within one sequence, and those of the result, pass 2^32 bytes
    B, T, D = 1, 300, 1 << 23
    x = torch.randn(B, T, 8, device="cuda", generator=g).bfloat16().repeat_interleave(D // 8, -1)
    y, s = K.causal_conv(x, w[:1].expand(D, 4))
    small, end = K.causal_conv(x[..., ::D // 8].contiguous(), w[:1].expand(8, 4))
    assert torch.equal(y[..., ::D // 8], small) and torch.equal(y[..., D // 8 - 1::D // 8], small) and torch.equal(s[..., ::D // 8], end)


@pytest.mark.parametrize("dtype,residual", [(torch.bfloat16, None), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,C", [(1, 16), (37, 24), (33, 64), (517, 72), (16, 128), (1023, 136), (9, 256), (77, 264), (4999, 512), (70, 520), (600, 1024), (9, 1),
                                    (700, 255), (41, 257), (3, 1023), (30000, 128), (50, 2), (81, 100), (30, 250), (19, 646), (7, 1022), (5, 2050), (3, 4098)])
def test_rms_norm_of_narrow_rows(dtype, residual, rows, C):
    """Several rows to a wavefront or workgroup, the last ones short of a whole one."""
    test_rms_norm(dtype, residual, rows, C)


@pytest.mark.parametrize("rows,C", [(37, 24), (1023, 128), (517, 256), (45, 511), (700, 777), (21, 90), (9, 646), (3, 2050)])
def test_rms_norm_fp8_of_narrow_rows(rows, C):
    test_rms_norm_fp8(torch.bfloat16, rows, C)


def test_more_rows_than_a_grid_of_threads():
    """Rows whose threads pass 2^32, from one row that stands for all: each gives what it gives alone."""
    from rwkv_wkv_hip import sampling, ssm as K
    free, _ = torch.cuda.mem_get_info()
    if free < 64 << 30:
        pytest.skip("needs 64 GB")
    rows, C = (1 << 24) + 5, 1032
    x, w = torch.randn(1, C, device="cuda").bfloat16(), torch.randn(C, device="cuda")
    q, scale, _ = K.rms_norm_fp8(x.expand(rows, C), w)
    one, s, _ = K.rms_norm_fp8(x, w)
    assert (scale == s).all()
    bits = one.view(torch.uint8)
    for part in q.view(torch.uint8).split(1 << 21):
        assert (part == bits).all()
    rows = (1 << 22) + 5
    u = torch.rand(rows, device="cuda")
    logits = torch.randn(1, 9, device="cuda")
    token, logprob = sampling.sample(logits.expand(rows, 9), u)
    for at in (0, rows // 2 - 7, rows - 20):
        a, b = sampling.sample(logits.expand(20, 9).contiguous(), u[at:at + 20].clone())
        assert torch.equal(token[at:at + 20], a) and torch.equal(logprob[at:at + 20], b)
    assert token.min() >= 0 and token.max() < 9


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,D,W", [(2, 37, 2, 4), (3, 50, 130, 3), (1, 300, 646, 4), (2, 9, 258, 2), (1, 1, 66, 4), (2, 70, 131, 4)])
def test_causal_conv_of_widths_not_in_fours(dtype, B, T, D, W):
    from rwkv_wkv_hip import ssm as K
    v, grads = _conv_inputs(dtype, B, T, D, W)
    _compare(lambda **k: K.causal_conv(**k), lambda **k: O.causal_conv(**k), v, grads, ["y", "state"])


@pytest.mark.parametrize("from_,step", [(2, 2), (1, 2), (2, 3), (4, 2), (0, 2)])
def test_causal_conv_of_slices_that_begin_anywhere(from_, step):
    """A slice of a wider tensor whose address or row distance allows four channels to a lane, two or one."""
    from rwkv_wkv_hip import ssm as K
    x = torch.randn(2, 40, 64 * step + 2 * step, generator=_g(from_, step)).bfloat16().cuda()
    w = torch.randn(64, 4, generator=_g(3)).cuda()
    part = x[..., from_:from_ + 64]
    for a, b in zip(K.causal_conv(part, w), K.causal_conv(part.contiguous(), w)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,C", [(3, 4100), (5, 6002), (2, 8190)])
def test_rms_norm_of_wide_rows_in_pairs(rows, C):
    test_rms_norm(torch.bfloat16, torch.float32, rows, C)
    test_rms_norm_fp8(torch.bfloat16, rows, C)
