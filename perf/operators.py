"""The operators of a state space block and of the end of a serving loop, as cases to time and to check.

A case is a dict of plain values.  ``op`` says which operator, ``way`` which direction of use:

    op      conv     the short causal convolution over the tokens, a filter per channel, with its SiLU
            scan     the selective state space scan with its gate
            norm     the residual's addition and the root-mean-square norm
            sample   one token per row of logits: temperature, top-k, top-p and min-p, from a given random number per row
    way     decode   one token per sequence, no autograd: a serving loop's call
            prefill  a prompt, no autograd
            train    forward and backward, every gradient
            fp8      (norm) the normalised rows in 8 bits with a scale per row, no autograd
            draw     (sample) the one way there is

``T`` counts tokens, ``D`` channels, ``N`` states per channel, ``G`` groups of channels with an input and output vector of
their own, ``taps`` filter taps, ``V`` the vocabulary.  ``ragged``: the sequences of the batch end at lengths of their own, zero
among them.  ``carry``: a state comes in.

Where ``own`` is false ``run`` computes the operators in elementary torch operations, in 32 bits whatever the inputs'
type; where it is true it calls the package.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-5
_LOG2E = 1.4426950408889634
_ONE = 2 ** 31            # the weight of a row's likeliest token


def _package():
    at = os.path.join(os.getcwd(), "rwkv-infctx-trainer_amd")
    if not os.path.isdir(os.path.join(at, "rwkv_wkv_hip")):
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rwkv-infctx-trainer_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import rwkv_wkv_hip
    return rwkv_wkv_hip


def listed():
    return [
        # a server that batches 64 users: the filter's window moves on by one token
        dict(name="conv decode batch", op="conv", way="decode", B=64, T=1, D=4096, taps=4, io="bf16", ragged=False, carry=True),
        # a training batch, a state carried in and its gradient out
        dict(name="conv train", op="conv", way="train", B=8, T=4096, D=4096, taps=4, io="bf16", ragged=False, carry=True),
        # one user's chat: the smallest scan there is, made once per layer and token
        dict(name="scan decode", op="scan", way="decode", B=1, T=1, D=4096, N=16, G=1, io="bf16", gate=True, ragged=False, carry=True),
        # 64 users at the width of two 2560-channel streams: the states are all there is to move
        dict(name="scan decode batch", op="scan", way="decode", B=64, T=1, D=5120, N=16, G=1, io="bf16", gate=True, ragged=False, carry=True),
        # four prompts of no particular lengths in one call, fp16
        dict(name="scan prefill ragged", op="scan", way="prefill", B=4, T=777, D=4096, N=16, G=1, io="fp16", gate=True, ragged=True, carry=False),
        # a small model in fp32 at an odd length
        dict(name="scan train small fp32", op="scan", way="train", B=2, T=301, D=1536, N=16, G=1, io="fp32", gate=True, ragged=False, carry=False),
        # a batch of truncated BPTT segments: states carried in, gradients through the states handed out
        dict(name="scan train", op="scan", way="train", B=8, T=2048, D=4096, N=16, G=1, io="bf16", gate=True, ragged=False, carry=True),
        # single tokens of 64 users on their way into an 8-bit projection
        dict(name="norm decode fp8", op="norm", way="fp8", rows=64, D=2048, io="bf16", residual="bf16"),
        # a long prompt on its way into an 8-bit projection
        dict(name="norm prefill fp8", op="norm", way="fp8", rows=4096, D=4096, io="bf16", residual="fp32"),
        # the norm of a 2560-channel layer in training, the residual kept in 32 bits
        dict(name="norm train", op="norm", way="train", rows=8 * 4096, D=2560, io="bf16", residual="fp32"),
        # one user's next token
        dict(name="sample one", op="sample", way="draw", B=1, V=65536, io="fp32", masked=False),
        # a batch of users, each with settings of its own, some of the vocabulary masked
        dict(name="sample batch", op="sample", way="draw", B=200, V=50277, io="bf16", masked=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choices(["conv", "scan", "norm", "sample"], [20, 45, 20, 15])[0]
    io = rng.choices(["bf16", "fp16", "fp32"], [60, 20, 20])[0]
    if op == "sample":
        V = _log_int(rng, 1000, 131072)
        return dict(op=op, way="draw", B=_log_int(rng, 1, min(256, 200 * 65536 // V)), V=V, io=io, masked=rng.random() < 0.5)
    if op == "norm":
        D = _log_int(rng, 64, 8192)
        rows = _log_int(rng, 1, min(32768, 32768 * 2560 // D))
        return dict(op=op, way=rng.choice(["fp8", "train"]), rows=rows, D=D, io=io, residual=rng.choice([io, "fp32"]))
    way = rng.choices(["decode", "prefill", "train"], [25, 30, 45])[0]
    D = _log_int(rng, 256, 8192)
    T = 1 if way == "decode" else _log_int(rng, 2, 4096)
    if op == "conv":
        B = _log_int(rng, 1, 128 if way == "decode" else max(1, min(16, 8 * 2048 * 4096 // (T * D))))
        return dict(op=op, way=way, B=B, T=T, D=D, taps=rng.choice([2, 3, 4]), io=io, ragged=way != "decode" and rng.random() < 0.3,
                    carry=way == "decode" or rng.random() < 0.5)
    N = rng.choice([8, 16, 16, 16, 32])
    G = rng.choice([1, 1, 1, 2])
    D = G * max(1, D // G)
    B = _log_int(rng, 1, 128 if way == "decode" else max(1, min(16, 8 * 2048 * 4096 * 16 // (T * D * N))))
    return dict(op=op, way=way, B=B, T=T, D=D, N=N, G=G, io=io, gate=rng.random() < 0.8, ragged=way != "decode" and rng.random() < 0.3,
                carry=way == "decode" or rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------------------------------------------
class _Make:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=self.g)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=self.g)

    def lengths(self, B, T):
        n = (self.uniform(B) * (T + 1)).to(torch.int32)
        n[0] = 0 if B > 1 else T - T // 4
        n[-1] = T if B > 1 else n[-1]
        return n


def prepare(case, seed):
    m = _Make(seed)
    s = dict(case=case)
    op, train = case["op"], case["way"] == "train"
    io = _TYPES[case["io"]]
    if op == "sample":
        B, V = case["B"], case["V"]
        # a model's logits: most of the vocabulary far below a few tens of likely tokens, the likeliest apart from each other
        l = m.normal(B, V, std=2.0) + 6.0 * (m.uniform(B, V) < 30.0 / V)
        if case["masked"]:
            l = l.masked_fill(m.uniform(B, V) < 0.3, -math.inf)
        s["logits"] = l.to(io)
        s["u"] = m.uniform(B)
        pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (B,), device="cuda", generator=m.g)]
        s["temperature"] = pick(0.0, 0.6, 0.8, 1.0, 1.0, 1.3)
        s["top_k"] = pick(0, 0, 20, 50, 1000).int()
        s["top_p"] = pick(1.0, 0.5, 0.9, 0.95)
        s["min_p"] = pick(0.0, 0.0, 0.05)
        return s
    D = case["D"]
    if op == "norm":
        s["x"] = m.normal(case["rows"], D).to(io)
        s["residual"] = m.normal(case["rows"], D, std=2.0).to(_TYPES[case["residual"]])
        s["weight"] = m.uniform(D, lo=0.5, hi=1.5).to(io)
        if train:
            s["gy"], s["gres"] = m.normal(case["rows"], D).to(io), m.normal(case["rows"], D).to(_TYPES[case["residual"]])
        return s
    B, T = case["B"], case["T"]
    if case["ragged"]:
        s["lengths"] = m.lengths(B, T)
    if op == "conv":
        W = case["taps"]
        # the left half of the projection that makes the stream and its gate
        s["x"] = m.normal(B, T, 2 * D).to(io)[..., :D]
        s["weight"], s["bias"] = m.uniform(D, W, lo=-W ** -0.5, hi=W ** -0.5).to(io), m.normal(D, std=0.1).to(io)
        if case["carry"]:
            s["state"] = m.normal(B, W - 1, D).to(io)
        if train:
            s["gy"], s["gstate"] = m.normal(B, T, D).to(io), m.normal(B, W - 1, D).to(io)
        return s
    N, G = case["N"], case["G"]
    s["x"] = torch.nn.functional.silu(m.normal(B, T, D)).to(io)
    if case["gate"]:
        s["z"] = m.normal(B, T, 2 * D).to(io)[..., D:]
    # time steps as a fresh layer has them: the bias sets 0.001 .. 0.1 over the channels, the projection moves them
    step = torch.exp(m.uniform(D, lo=math.log(1e-3), hi=math.log(0.1)))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["dt"] = m.normal(B, T, D, std=0.5).to(io)
    s["A"] = -torch.arange(1, N + 1, device="cuda").float().expand(D, N) * torch.exp(m.normal(D, N, std=0.1))
    s["D"] = m.uniform(D, lo=0.5, hi=1.5)
    # the input and output vectors: slices of the projection that also makes the time step's low-rank input
    R = max(1, D // 16)
    bc = m.normal(B, T, R + 2 * G * N).to(io)
    s["B"], s["C"] = bc[..., R:R + G * N].unflatten(-1, (G, N)), bc[..., R + G * N:].unflatten(-1, (G, N))
    if case["carry"]:
        s["state"] = m.normal(B, D, N, std=0.3)
    if train:
        s["gy"], s["gstate"] = m.normal(B, T, D).to(io), m.normal(B, D, N, std=0.3)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _valid(s, B, T):
    """(B, T, 1): the tokens that there are."""
    n = s.get("lengths")
    return torch.ones(B, T, 1, dtype=torch.bool, device="cuda") if n is None else (torch.arange(T, device="cuda") < n[:, None])[..., None]


def _plain_conv(s):
    case = s["case"]
    B, T, D, W, io = case["B"], case["T"], case["D"], case["taps"], s["x"].dtype
    w, ok = s["weight"].float(), _valid(s, B, T)
    before = s["state"].float() if "state" in s else torch.zeros(B, W - 1, D, device="cuda")
    xx = torch.cat([before, torch.where(ok, s["x"].float(), 0.0)], 1)
    at = s["lengths"].long() if "lengths" in s else torch.full((B,), T, device="cuda")
    rows = (at[:, None] + torch.arange(W - 1, device="cuda"))[..., None].expand(B, W - 1, D)
    windows = xx.unfold(1, W, 1)                                            # (B, T, D, W)
    pre = (windows * w).sum(-1) + s["bias"].float()
    sig = torch.sigmoid(pre)
    y, state = torch.where(ok, pre * sig, 0.0).to(io), xx.gather(1, rows).to(io)
    if "gy" not in s:
        return y, state
    gpre = torch.where(ok, s["gy"].float() * sig * (1 + pre * (1 - sig)), 0.0)
    gweight, gbias = (gpre[..., None] * windows).sum((0, 1)), gpre.sum((0, 1))
    padded = torch.nn.functional.pad(gpre, (0, 0, W - 1, W - 1))
    gxx = (padded.unfold(1, W, 1) * w.flip(1)).sum(-1).scatter_add(1, rows, s["gstate"].float())
    out = [y, state, torch.where(ok, gxx[:, W - 1:], 0.0).to(io), gweight.to(io), gbias.to(io)]
    return out + [gxx[:, :W - 1].to(io)] if "state" in s else out


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dimension 1 from nothing, and the running products of a: by doubling steps."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return a, b


def _plain_scan(s):
    case = s["case"]
    B, T, D, N, G, io = case["B"], case["T"], case["D"], case["N"], case["G"], s["x"].dtype
    ok = _valid(s, B, T)
    real = lambda t: torch.where(ok, t.float(), 0.0)
    x, A = real(s["x"]), s["A"]
    raw = real(s["dt"]) + s["dt_bias"]
    dt = torch.where(ok, _softplus(raw), 0.0)
    over = lambda t: real(t.flatten(2)).unflatten(-1, (G, N)).repeat_interleave(D // G, 2)      # (B, T, D, N)
    b, c = over(s["B"]), over(s["C"])
    h0 = s["state"] if "state" in s else torch.zeros(B, D, N, device="cuda")
    a = torch.exp(dt[..., None] * A)
    through, h = _recurrence(a, (dt * x)[..., None] * b)
    h = h + through * h0[:, None]
    del through
    ypre = (h * c).sum(-1) + s["D"] * x
    gate = real(s["z"]) if "z" in s else None
    sig = None if gate is None else torch.sigmoid(gate)
    y = torch.where(ok, ypre if gate is None else ypre * gate * sig, 0.0).to(io)
    state = h[:, -1]
    if "gy" not in s:
        return y, state.clone()
    gout = real(s["gy"])
    gy = gout if gate is None else gout * gate * sig
    # the state's gradient runs the other way: g[t] = c[t] gy[t] + a[t+1] g[t+1]
    back = torch.cat([torch.ones_like(a[:, :1]), a.flip(1)[:, :-1]], 1)
    through, g = _recurrence(back, (c * gy[..., None]).flip(1))
    g = (g + through * s["gstate"][:, None]).flip(1)
    del through, back
    hp = torch.cat([h0[:, None], h[:, :-1]], 1) * a                          # what is left of the state before
    sx = (g * b).sum(-1)
    gdt = (g * hp * A).sum(-1) + sx * x
    graw = torch.where(ok, gdt * torch.sigmoid(raw), 0.0)
    split = lambda t: t.unflatten(2, (G, D // G)).sum(3)
    out = [y, state.clone(), torch.where(ok, sx * dt + gy * s["D"], 0.0).to(io), graw.to(io), (g * hp * dt[..., None]).sum((0, 1)),
           split(g * (dt * x)[..., None]).to(io), split(h * gy[..., None]).to(io), (gy * x).sum((0, 1)), graw.sum((0, 1))]
    if gate is not None:
        out.append((gout * ypre * sig * (1 + gate * (1 - sig))).to(io))
    if "state" in s:
        out.append(a[:, 0] * g[:, 0])
    return out


def _plain_norm(s):
    x, w = s["x"], s["weight"].float()
    r = x.float() + s["residual"].float()
    rstd = torch.rsqrt(r.square().mean(1, keepdim=True) + _EPS)
    xhat = r * rstd
    y = xhat * w
    if s["case"]["way"] == "fp8":
        top = y.abs().amax(1, keepdim=True)
        scale = torch.where(top > 0, top / 448.0, 1.0)
        return (y / scale).to(torch.float8_e4m3fn), scale, r.to(s["residual"].dtype)
    gw = s["gy"].float() * w
    g = s["gres"].float() + rstd * (gw - xhat * (gw * xhat).mean(1, keepdim=True))
    return y.to(x.dtype), r.to(s["residual"].dtype), g.to(x.dtype), g.to(s["residual"].dtype), (s["gy"].float() * xhat).sum(0).to(s["weight"].dtype)


def _plain_sample(s):
    l, u, t, k, p, least = s["logits"].float(), s["u"], s["temperature"], s["top_k"].long()[:, None], s["top_p"], s["min_p"]
    l = torch.where(l.isnan(), -math.inf, l)
    top = l.amax(1, keepdim=True)
    warm = t >= 1e-6
    scale = torch.full_like(t, _LOG2E) / torch.where(warm, t, 1.0)
    # weights are whole 2^-31ths of the likeliest token's, so that no sum depends on its order
    x = torch.where(l > -math.inf, torch.where(l == top, 0.0, (l - top) * scale[:, None]), -math.inf)
    w = (torch.exp2(x) * _ONE).round().long()
    order = x.sort(dim=1, descending=True, stable=True).indices
    sorted_w, rank = w.gather(1, order), torch.arange(l.shape[1], device="cuda")
    k = torch.where(warm[:, None], k, 1)
    kept = ((k <= 0) | (rank < k)) & (sorted_w >= (least.double() * _ONE).ceil().long().clamp(1, _ONE)[:, None])
    sorted_w = sorted_w * kept
    total, upto = sorted_w.sum(1), sorted_w.cumsum(1)
    need = torch.where(p < 1, (p.double() * total.double()).ceil().long().clamp(min=1), total)
    kept &= upto - sorted_w < need[:, None]
    w = w * torch.zeros_like(kept).scatter(1, order, kept)
    upto = w.cumsum(1)
    total = upto[:, -1]
    target = torch.minimum((u.double() * total.double()).floor().long(), total - 1)
    token = (upto <= target[:, None]).sum(1)
    weight = w.gather(1, token.clamp(max=l.shape[1] - 1)[:, None])[:, 0]
    some = total > 0
    logprob = torch.where(some, (weight.double() / total.clamp(min=1).double()).log(), -math.inf).float()
    return torch.where(some, token, -1), logprob


# ---- the package's own ----------------------------------------------------------------------------------------------
def _leaves(s, names):
    return {n: s[n].detach().requires_grad_(True) for n in names if n in s}


def _own_conv(s):
    K = _package().ssm
    if "gy" not in s:
        return K.causal_conv(s["x"], s["weight"], s["bias"], state=s.get("state"), lengths=s.get("lengths"))
    v = _leaves(s, ("x", "weight", "bias", "state"))
    y, state = K.causal_conv(v["x"], v["weight"], v["bias"], state=v.get("state"), lengths=s.get("lengths"))
    return [y, state, *torch.autograd.grad([y, state], list(v.values()), [s["gy"], s["gstate"]])]


def _own_scan(s):
    K = _package().ssm
    names = ("x", "dt", "A", "B", "C", "D", "dt_bias", "z", "state")
    v = _leaves(s, names) if "gy" in s else {n: s[n] for n in names if n in s}
    y, state = K.selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], D=v["D"], z=v.get("z"), dt_bias=v["dt_bias"], state=v.get("state"),
                                lengths=s.get("lengths"))
    if "gy" not in s:
        return y, state
    return [y, state, *torch.autograd.grad([y, state], list(v.values()), [s["gy"], s["gstate"]])]


def _own_norm(s):
    K = _package().ssm
    if s["case"]["way"] == "fp8":
        return K.rms_norm_fp8(s["x"], s["weight"], _EPS, residual=s["residual"])
    v = _leaves(s, ("x", "residual", "weight"))
    y, r = K.rms_norm(v["x"], v["weight"], _EPS, residual=v["residual"])
    return [y, r, *torch.autograd.grad([y, r], list(v.values()), [s["gy"], s["gres"]])]


def _own_sample(s):
    return _package().sampling.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def run(state):
    f = {"conv": (_plain_conv, _own_conv), "scan": (_plain_scan, _own_scan), "norm": (_plain_norm, _own_norm), "sample": (_plain_sample, _own_sample)}
    return f[state["case"]["op"]][own](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    op, way, b = case["op"], case["way"], _SIZE[case["io"]]
    if op == "sample":
        n = case["B"] * case["V"]
        return dict(bytes=n * b + 28 * case["B"], flops=4 * n)
    D = case["D"]
    if op == "norm":
        n, r = case["rows"] * D, _SIZE[case["residual"]]
        if way == "fp8":
            return dict(bytes=n * (b + 2 * r + 1) + 4 * case["rows"], flops=6 * n)
        return dict(bytes=n * (b + 2 * r + b) + n * (2 * b + 3 * r), flops=18 * n)
    B, T = case["B"], case["T"]
    n, train = B * T * D, way == "train"
    if op == "conv":
        W, states = case["taps"], B * (case["taps"] - 1) * D * b
        bytes_ = 2 * n * b + (1 + case["carry"]) * states + D * (W + 1) * b
        return dict(bytes=bytes_ + (3 * n * b + (1 + case["carry"]) * states + D * (W + 1) * 2 * b if train else 0), flops=n * (2 * W + 4) * (4 if train else 1))
    N, gate = case["N"], case["gate"]
    streams, vectors, states = n * b * (3 + gate), 2 * B * T * case["G"] * N * b, (1 + case["carry"]) * B * D * N * 4
    parameters = D * (N + 2) * 4
    if not train:
        return dict(bytes=streams + vectors + states + parameters, flops=n * (6 * N + 12))
    # backward: the streams and the gradient coming in, their gradients going out
    return dict(bytes=2 * streams + n * b * (1 + gate) + 3 * vectors + 2 * states + 2 * parameters, flops=n * (24 * N + 50))


# ---- 64 bits, token by token -------------------------------------------------------------------------------------------
def _exact_conv(s):
    case = s["case"]
    B, T, D, W = case["B"], case["T"], case["D"], case["taps"]
    n = s["lengths"].long() if "lengths" in s else torch.full((B,), T, device="cuda")
    live = (torch.arange(T, device="cuda") < n[:, None])[..., None]
    x, w = s["x"].double().masked_fill(~live, 0.0), s["weight"].double()
    at = lambda t: x[:, t] if t >= 0 else (s["state"][:, t + W - 1].double() if "state" in s else torch.zeros_like(x[:, 0]))
    y, gx, gbias, gw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros(D, dtype=torch.float64, device="cuda"), torch.zeros_like(w)
    gbefore = torch.zeros(B, W - 1, D, dtype=torch.float64, device="cuda")
    state = torch.zeros_like(gbefore)
    for i in range(W - 1):
        rows = n - (W - 1) + i
        inside = x.gather(1, rows.clamp(min=0)[:, None, None].expand(B, 1, D))[:, 0]
        early = s["state"].double().gather(1, (rows + W - 1).clamp(max=W - 2)[:, None, None].expand(B, 1, D))[:, 0] if "state" in s else torch.zeros_like(inside)
        state[:, i] = torch.where(rows[:, None] >= 0, inside, early)
    for t in range(T):
        pre = s["bias"].double().expand(B, D).clone()
        for k in range(W):
            pre += w[:, k] * at(t - (W - 1) + k)
        sig = 1 / (1 + torch.exp(-pre))
        y[:, t] = (pre * sig).masked_fill(~live[:, t], 0.0)
        if "gy" in s:
            gp = (s["gy"][:, t].double() * (sig + pre * sig * (1 - sig))).masked_fill(~live[:, t], 0.0)
            gbias += gp.sum(0)
            for k in range(W):
                r = t - (W - 1) + k
                gw[:, k] += (gp * at(r)).sum(0)
                (gx[:, r] if r >= 0 else gbefore[:, r + W - 1]).add_(gp * w[:, k])
    if "gy" not in s:
        return y, state
    for i in range(W - 1):
        rows = n - (W - 1) + i
        g = s["gstate"][:, i].double()
        for b in range(B):
            r = int(rows[b])
            (gx[b, r] if r >= 0 else gbefore[b, r + W - 1]).add_(g[b])
    out = [y, state, gx, gw, gbias]
    return out + [gbefore] if "state" in s else out


def _exact_scan(s):
    case = s["case"]
    B, T, D, N, G = case["B"], case["T"], case["D"], case["N"], case["G"]
    n = s["lengths"].long() if "lengths" in s else torch.full((B,), T, device="cuda")
    A, skip, bias = s["A"].double(), s["D"].double(), s["dt_bias"].double()
    h = s["state"].double() if "state" in s else torch.zeros(B, D, N, dtype=torch.float64, device="cuda")
    wide = lambda v, t, live: v[:, t].double().masked_fill(~live[..., None], 0.0)[:, :, None].expand(B, G, D // G, N).reshape(B, D, N)
    row = lambda v, t, live: v[:, t].double().masked_fill(~live, 0.0)
    y = torch.zeros(B, T, D, dtype=torch.float64, device="cuda")
    ys, hs = torch.zeros_like(y), [h]
    train = "gy" in s
    for t in range(T):
        live = (t < n)[:, None]
        x = row(s["x"], t, live)
        dt = torch.logaddexp(row(s["dt"], t, live) + bias, torch.zeros_like(x)).masked_fill(~live, 0.0)
        h = torch.exp(dt[..., None] * A) * h + (dt * x)[..., None] * wide(s["B"], t, live)
        ys[:, t] = (h * wide(s["C"], t, live)).sum(-1) + skip * x
        z = row(s["z"], t, live) if "z" in s else None
        y[:, t] = (ys[:, t] if z is None else ys[:, t] * z / (1 + torch.exp(-z))).masked_fill(~live, 0.0)
        if train:
            hs.append(h)
    if not train:
        return y, h
    g = s["gstate"].double()
    gx, gdt, gz = torch.zeros_like(y), torch.zeros_like(y), torch.zeros_like(y)
    gA, gD, gbias = torch.zeros_like(A), torch.zeros_like(skip), torch.zeros_like(bias)
    gB = torch.zeros(B, T, G, N, dtype=torch.float64, device="cuda")
    gC = torch.zeros_like(gB)
    for t in reversed(range(T)):
        live = (t < n)[:, None]
        x, raw, go = row(s["x"], t, live), row(s["dt"], t, live) + bias, row(s["gy"], t, live)
        dt = torch.logaddexp(raw, torch.zeros_like(raw)).masked_fill(~live, 0.0)
        gy = go
        if "z" in s:
            z = row(s["z"], t, live)
            sig = 1 / (1 + torch.exp(-z))
            gy = go * z * sig
            gz[:, t] = go * ys[:, t] * (sig + z * sig * (1 - sig))
        b, c, a = wide(s["B"], t, live), wide(s["C"], t, live), torch.exp(dt[..., None] * A)
        g = g + c * gy[..., None]
        gC[:, t] = (hs[t + 1] * gy[..., None]).view(B, G, D // G, N).sum(2)
        gB[:, t] = (g * (dt * x)[..., None]).view(B, G, D // G, N).sum(2)
        u = (g * b).sum(-1)
        ga = g * hs[t] * a
        gA += (ga * dt[..., None]).sum(0)
        gx[:, t] = (u * dt + gy * skip).masked_fill(~live, 0.0)
        gr = (((ga * A).sum(-1) + u * x) / (1 + torch.exp(-raw))).masked_fill(~live, 0.0)
        gdt[:, t] = gr
        gD += (gy * x).sum(0)
        gbias += gr.sum(0)
        g = g * a
    out = [y, h, gx, gdt, gA, gB, gC, gD, gbias]
    return out + ([gz] if "z" in s else []) + ([g] if "state" in s else [])


def _exact_norm(s):
    r, w = s["x"].double() + s["residual"].double(), s["weight"].double()
    inv = (r.pow(2).sum(1, keepdim=True) / r.shape[1] + _EPS).pow(-0.5)
    if s["case"]["way"] == "fp8":
        y = r * inv * w
        scale = y.abs().max(1, keepdim=True).values / 448
        return y / scale, scale, r
    g = s["gy"].double() * w
    gr = inv * g - r * inv.pow(3) * (g * r).sum(1, keepdim=True) / r.shape[1] + s["gres"].double()
    return r * inv * w, r, gr, gr, (s["gy"].double() * r * inv).sum(0)


def _exact_sample(s):
    logprob = []
    for b in range(s["logits"].shape[0]):
        l = s["logits"][b].double()
        t, k, p, least = (float(s[n][b]) for n in ("temperature", "top_k", "top_p", "min_p"))
        l = l.masked_fill(l.isnan(), -math.inf)
        if t < 1e-6:
            t, k = 1.0, 1
        value, index = l.sort(dim=0, descending=True, stable=True)
        w = torch.round(torch.exp((value - value[0]) / t) * _ONE)
        w = w[:int(k)] if k > 0 else w
        w = w[w >= max(1.0, least * _ONE)]
        if p < 1:
            w = w[(w.cumsum(0) - w) < p * w.sum()]
        by_index = index[:len(w)].argsort()
        w = w[by_index]
        at = int((w.cumsum(0) <= math.floor(float(s["u"][b]) * float(w.sum()))).sum())
        logprob.append(torch.log(w[min(at, len(w) - 1)] / w.sum()))
    return None, torch.stack(logprob)


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm, "sample": _exact_sample}[case["op"]](s)
