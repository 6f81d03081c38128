"""No-GPU checks of the C ABI of a gated recurrence model's operators: bad arguments are answered before anything is launched, and workspace queries follow the
sizes."""
import ctypes

import pytest
import torch

from tests.test_ssm_abi_cpu import L, NULL, ODD, ONE, rows  # noqa: F401

at = ctypes.c_void_p


def test_recurrence(L):  # noqa: F811
    def forward(B=2, T=8, D=64, dtype=1, x=None, r=None, decay=ONE, z=True, state_in=NULL, y=ONE, out=ONE, checkpoints=NULL, ws=ONE, size=1 << 40):
        return L.wkv_gated_recurrence_forward(NULL, B, T, D, dtype, 8.0, x or rows(), r or rows(), rows(), decay, rows() if z else NULL, state_in, NULL, y, out,
                                              checkpoints, ws, size)
    assert forward() == -6 and forward(z=False) == -6                       # (no device)
    assert forward(state_in=ONE) == -8 and forward(state_in=ONE, T=1) == -6                      # a single token may have its state in place
    assert forward(state_in=ONE, T=1, checkpoints=ONE) == -8 and forward(state_in=at((1 << 40) + 16), T=1) == -8          # but neither a recorded call nor half of it
    for k in ({"B": 0}, {"T": 0}, {"D": 0}, {"B": 70000}, {"T": (1 << 24) + 1}, {"D": 1 << 24}, {"B": 60000, "D": 1 << 23}, {"T": -1}):
        assert forward(**k) == -1, k
    assert forward(dtype=3) == -3 and forward(decay=NULL) == -2 and forward(y=NULL) == -2 and forward(out=NULL) == -2
    assert forward(x=rows(p=None)) == -2 and forward(r=rows(p=at((1 << 40) + 1))) == -4 and forward(decay=ODD) == -4 and forward(out=ODD) == -4 and forward(y=ODD) == -4
    assert forward(r=rows(token=63)) == -1 and forward(r=rows(token=1 << 24)) == -1 and forward(T=1, r=rows(token=0)) == -6
    assert L.wkv_gated_recurrence_forward(NULL, 2, 8, 64, 1, 8.0, NULL, rows(), rows(), ONE, NULL, NULL, NULL, ONE, ONE, NULL, ONE, 1 << 40) == -2
    need = L.wkv_gated_recurrence_forward_workspace(1, 8192, 64, 1)
    assert need > 0 and forward(B=1, T=8192, size=need - 1) == -5 and forward(B=1, T=8192, ws=NULL) == -2
    assert L.wkv_gated_recurrence_forward_workspace(9, 1, 64, 1) == 0 and L.wkv_gated_recurrence_forward_workspace(9, 0, 64, 1) == 0
    assert L.wkv_gated_recurrence_checkpoint_bytes(2, 65, 40, 1) == 2 * 2 * 40 * 4 and L.wkv_gated_recurrence_checkpoint_bytes(2, 64, 40, 7) == 0

    back = L.wkv_gated_recurrence_backward_workspace(2, 64, 64, 1)

    def backward(z=True, checkpoints=ONE, gy=ONE, gs=NULL, gx=ONE, gz=ONE, gdecay=ONE, gstate=NULL, ws=ONE, size=back):
        return L.wkv_gated_recurrence_backward(NULL, 2, 64, 64, 1, 8.0, rows(), rows(), rows(), ONE, rows() if z else NULL, NULL, checkpoints, gy, gs, gx, ONE, ONE,
                                               gdecay, gz, gstate, ws, size)
    assert back > 0 and backward() == -6 and backward(z=False, gz=NULL) == -6 and backward(gs=ONE, gstate=at(1 << 41)) == -6
    assert backward(size=back - 1) == -5 and backward(ws=NULL) == -2 and backward(gz=NULL) == -2 and backward(checkpoints=NULL) == -2 and backward(gy=NULL) == -2
    assert backward(gs=ONE, gstate=ONE) == -8 and backward(gx=ODD) == -4 and backward(gdecay=NULL) == -2


def test_feed_forward(L):  # noqa: F811
    def forward(R=100, C=64, F=48, dtype=1, act=0, x=ONE, stride=64, w=ONE, h=ONE, kept=NULL, ws=ONE, size=1 << 40):
        return L.wkv_gated_product_forward(NULL, R, C, F, dtype, act, x, stride, w, ONE, h, kept, ws, size)
    assert forward() == -6 and forward(act=2) == -6 and forward(R=1) == -6
    for k in ({"R": 0}, {"C": 0}, {"F": 0}, {"R": -5}, {"R": (1 << 21) + 1}, {"C": (1 << 20) + 8, "stride": (1 << 20) + 8}, {"F": 1 << 20}, {"stride": 63},
              {"stride": (1 << 21) + 8}, {"R": 1 << 21, "F": 1 << 15}):
        assert forward(**k) == -1, k
    assert forward(dtype=3) == -3 and forward(act=3) == -7 and forward(act=-1) == -7
    assert forward(x=NULL) == -2 and forward(w=NULL) == -2 and forward(h=NULL) == -2
    assert forward(h=ODD) == -4 and forward(x=at((1 << 40) + 2)) == -4 and forward(stride=66) == -4 and forward(w=ODD) == -4
    # rows that are not whole pieces of 16 bytes begin anywhere, but at an element
    assert forward(C=63, x=at((1 << 40) + 2), stride=65) == -6 and forward(C=63, x=at((1 << 40) + 1), stride=65) == -4
    # many rows that are not whole pieces are copied to such that are
    big = dict(R=20000, C=1001, F=2731, stride=1001)
    need = L.wkv_gated_product_forward_workspace(20000, 1001, 2731, 1)
    assert need == (20000 + 2 * 2731) * 1024 * 2 and forward(**big, size=need - 1) == -5 and forward(**big, ws=NULL) == -2 and forward(**big) == -6
    assert L.wkv_gated_product_forward_workspace(20000, 1000, 2731, 1) == 0 and L.wkv_gated_product_forward_workspace(100, 63, 48, 1) == 0
    assert L.wkv_gated_product_kept_bytes(3, 64, 50, 1) == 3 * 2 * 64 * 4 and L.wkv_gated_product_kept_bytes(3, 64, 0, 1) == 0

    size_of = L.wkv_gated_product_backward_workspace
    back = size_of(100, 64, 48, 1, 1, 1)

    def backward(kept=ONE, gh=ONE, gx=ONE, gg=ONE, gu=ONE, ws=ONE, size=back, x=ONE, stride=64):
        return L.wkv_gated_product_backward(NULL, 100, 64, 48, 1, 0, x, stride, ONE, ONE, kept, gh, gx, gg, gu, ws, size)
    assert back > 0 and backward() == -6 and backward(size=back - 1) == -5 and backward(ws=NULL) == -2
    assert backward(gx=NULL, gg=NULL, gu=NULL) == -2 and backward(gg=NULL) == -2 and backward(gx=NULL) == -6 and backward(gg=NULL, gu=NULL) == -6
    assert backward(kept=NULL) == -2 and backward(gh=NULL) == -2 and backward(gx=ODD) == -4 and backward(kept=ODD) == -4 and backward(x=ODD) == -4 and backward(stride=8) == -1
    # one of the two sides takes no more than both, whatever the tiles
    for R, C, F in ((1, 8, 8), (100, 63, 48), (70, 2048, 7000), (5000, 520, 1500), (300, 1001, 2731)):
        for dt in (0, 1, 2):
            assert max(size_of(R, C, F, dt, 1, 0), size_of(R, C, F, dt, 0, 1)) <= size_of(R, C, F, dt, 1, 1)


def test_embedding(L):  # noqa: F811
    forward = lambda n=5, V=7, C=64, dt=1, ib=8, t=ONE, w=ONE, o=ONE: L.wkv_embedding_forward(NULL, n, V, C, dt, ib, 1.0, t, w, o)
    assert forward() == -6 and forward(ib=4, t=at((1 << 40) + 4)) == -6
    for k in ({"n": 0}, {"V": 0}, {"C": 0}, {"n": (1 << 28) + 1}, {"V": (1 << 24) + 1}, {"C": (1 << 23) + 1}, {"n": 1 << 28, "C": 32}, {"n": -1}):
        assert forward(**k) == -1, k
    assert forward(dt=5) == -3 and forward(ib=2) == -3 and forward(t=NULL) == -2 and forward(w=NULL) == -2 and forward(o=NULL) == -2
    assert forward(t=at((1 << 40) + 4)) == -4 and forward(w=ODD) == -4 and forward(o=ODD) == -4
    need = L.wkv_embedding_backward_workspace(5, 7, 64)
    backward = lambda t=ONE, g=ONE, stride=64, gt=ONE, ws=ONE, size=need: L.wkv_embedding_backward(NULL, 5, 7, 64, 1, 8, 1.0, t, g, stride, gt, ws, size)
    assert need > 0 and backward() == -6 and backward(size=need - 1) == -5 and backward(ws=NULL) == -2 and backward(t=NULL) == -2 and backward(gt=NULL) == -2
    assert backward(g=at((1 << 40) + 2), stride=65) == -6 and backward(g=at((1 << 40) + 1)) == -4 and backward(gt=ODD) == -4 and backward(ws=ODD) == -4


def test_front_end_refuses_cpu_tensors_and_unknown_activations():
    import rwkv_wkv_hip as W
    z = torch.zeros
    with pytest.raises(W.WKVError):
        W.gated.gated_recurrence(z(1, 2, 8), z(1, 2, 8), z(1, 2, 8), z(8))
    with pytest.raises(W.WKVError):
        W.gated.gated_feed_forward(z(2, 8), z(4, 8), z(4, 8))
    with pytest.raises(W.WKVError):
        W.gated.embedding(z(2, dtype=torch.long), z(4, 8))
    with pytest.raises(ValueError):
        W.gated.gated_feed_forward(z(2, 8), z(4, 8), z(4, 8), "tanh")
