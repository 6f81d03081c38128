"""The operators of a gated recurrence model under torch.autocast with fp32 parameters: the feed-forward's projections are cast as torch's own are."""
import pytest
import torch
import torch.nn.functional as F

from tests.test_gpu_gated_block import VOCABULARY, Block

pytestmark = pytest.mark.gpu
LOW = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("io", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R", [1, 70])
def test_feed_forward_under_autocast(low, io, R):
    """Different types: the bits of the call on operands that are cast by hand, the gradients in the operands' own types; switched off inside, types have to agree as ever.  One type: as
    without autocast."""
    from rwkv_wkv_hip import gated as K
    g = torch.Generator(device="cuda").manual_seed(R)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    leaf = [t.requires_grad_(True) for t in (n(R, 40).to(io), n(56, 40), n(56, 40))]
    one = io if io == torch.float32 else low
    gy = n(R, 56).to(one)
    want = K.gated_feed_forward(*(t.to(one) for t in leaf), "gelu")
    expected = torch.autograd.grad(want, leaf, gy)
    with torch.autocast("cuda", dtype=low):
        got = K.gated_feed_forward(*leaf, "gelu")
        with torch.no_grad():
            assert torch.equal(K.gated_feed_forward(*leaf, "gelu"), want)
        if io != torch.float32:
            with torch.autocast("cuda", enabled=False), pytest.raises(AssertionError):
                K.gated_feed_forward(*leaf, "gelu")
    assert got.dtype == one and torch.equal(got, want)
    for a, b, t in zip(torch.autograd.grad(got, leaf, gy), expected, leaf):
        assert a.dtype == t.dtype and torch.equal(a, b)


@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("T,lengths", [(1, None), (33, None), (70, [70, 0, 20])])
def test_block_under_autocast(low, T, lengths):
    """From tokens through the lookup and the block: what the same steps give with every projection's operands cast by hand, outputs, states and all gradients."""
    from rwkv_wkv_hip import gated as K
    from rwkv_wkv_hip.ssm import causal_conv, rms_norm
    m = Block().cuda()
    g = torch.Generator(device="cuda").manual_seed(T)
    tokens = torch.randint(-1, VOCABULARY, (3, T), device="cuda", generator=g)
    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def by_hand(m, x, residual, state, lengths):
        linear = lambda t, p: F.linear(t.to(low), p.weight.to(low))
        h, residual = rms_norm(x, m.norm_weight, m.eps, residual)
        u, z = linear(h, m.in_proj).chunk(2, -1)
        u, window = causal_conv(u, m.conv_weight, m.conv_bias, state[0], lengths, silu=False)
        r, i = linear(u, m.gate_proj).chunk(2, -1)
        y, h = K.gated_recurrence(u, r, i, m.decay, z=z, state=state[1], lengths=lengths)
        n, residual = rms_norm(linear(y, m.out_proj), m.ff_norm_weight, m.eps, residual)
        return linear(K.gated_feed_forward(*(t.to(low) for t in (n, m.ff_gate, m.ff_up)), m.activation), m.ff_down), residual, (window, h)

    def run(block, autocast):
        with torch.autocast("cuda", dtype=low, enabled=autocast):
            x = K.embedding(tokens, m.table, 2.0)
            out, residual, state = block(m, x, None, K.block_state(m, 3, low), L)
            out, residual, state = block(m, out, residual, state, L)
        results = [out, residual, *state]
        loss = sum((o.float() * torch.randn(o.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))).sum() for o in results)
        return results, torch.autograd.grad(loss, list(m.parameters()))

    (got, grads), (want, expected) = run(K.block_forward, True), run(by_hand, False)
    assert got[0].dtype == low and got[1].dtype == torch.float32
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for (n, p), a, b in zip(m.named_parameters(), grads, expected):
        # (a parameter's two uses: autocast casts it once and adds both gradients in 16 bits, by hand it is cast twice and they are added in fp32: two half steps)
        assert a.dtype == p.dtype and torch.isfinite(a).all(), n
        assert bool(((a - b).abs() <= torch.finfo(low).eps * (b.abs() + b.abs().max())).all()), n


def test_a_call_without_gradients_leaves_no_copy_behind():
    """A recorded call after one without autograd, both under one autocast: the weights' gradients come."""
    from rwkv_wkv_hip import gated as K
    n = lambda *s: torch.randn(*s, device="cuda")
    x, wg, wu = n(9, 40).bfloat16(), n(56, 40).requires_grad_(True), n(56, 40).requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with torch.no_grad():
            first = K.gated_feed_forward(x, wg, wu)
        out = K.gated_feed_forward(x, wg, wu)
    assert out.requires_grad and torch.equal(first, out)
    for t in torch.autograd.grad(out.float().sum(), (wg, wu)):
        assert t.dtype == torch.float32 and t.any()


def test_types_that_autocast_does_not_cast_are_refused():
    from rwkv_wkv_hip import gated as K
    n = lambda *s: torch.randn(*s, device="cuda")
    for record in (True, False):
        with torch.autocast("cuda", dtype=torch.bfloat16), torch.set_grad_enabled(record):
            with pytest.raises((ValueError, AssertionError)):
                K.gated_feed_forward(n(9, 40).double(), n(56, 40), n(56, 40))
            with pytest.raises((ValueError, AssertionError)):
                K.gated_feed_forward(n(9, 40).bfloat16(), n(56, 40).double(), n(56, 40))
