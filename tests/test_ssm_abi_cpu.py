"""No-GPU checks of the state space operators' C ABI: bad arguments are answered before anything is launched, and workspace
queries follow the sizes."""
import ctypes
import os

import pytest
import torch

ONE, NULL, ODD = ctypes.c_void_p(1 << 40), None, ctypes.c_void_p((1 << 40) + 6)


class Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("batch", ctypes.c_longlong), ("token", ctypes.c_longlong), ("group", ctypes.c_longlong)]


@pytest.fixture(scope="module")
def L():
    from rwkv_wkv_hip import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    if torch.cuda.is_available():
        pytest.skip("the pointers are not memory")
    return _lib.lib()


def rows(p=ONE, batch=1 << 10, token=64, group=16):
    return ctypes.byref(Rows(p, batch, token, group))


def scan(L, B=2, T=8, D=64, N=16, G=1, dtype=1, x=None, z=True, A=ONE, state_in=ONE, y=ONE, out=ONE, checkpoints=NULL, ws=ONE, size=1 << 40):
    x = rows() if x is None else x
    return L.wkv_selective_scan_forward(NULL, B, T, D, N, G, dtype, x, rows(), A, rows(), rows(), ONE, rows() if z else NULL, ONE, state_in, NULL, y, out,
                                        checkpoints, ws, size)


def test_scan(L):
    assert scan(L) == -8 and scan(L, state_in=NULL) == -6                    # the state in place; no device
    assert scan(L, T=1) == -6                                                # a single token may have it in place
    assert scan(L, T=1, checkpoints=ONE) == -8
    assert scan(L, T=0) == -1 and scan(L, N=65) == -1 and scan(L, N=0) == -1 and scan(L, G=3) == -1 and scan(L, B=70000) == -1
    assert scan(L, dtype=5) == -3
    assert scan(L, A=NULL) == -2 and scan(L, y=NULL) == -2
    assert L.wkv_selective_scan_forward(NULL, 2, 8, 64, 16, 1, 1, NULL, rows(), ONE, rows(), rows(), ONE, NULL, ONE, NULL, NULL, ONE, ONE, NULL, ONE, 1 << 40) == -2
    assert scan(L, x=rows(p=None)) == -2 and scan(L, x=rows(p=ctypes.c_void_p(7))) == -4 and scan(L, x=rows(token=1 << 24)) == -1
    assert scan(L, A=ODD) == -4 and scan(L, out=ODD, state_in=NULL) == -4
    need = L.wkv_selective_scan_forward_workspace(1, 4096, 64, 16, 1, 1)
    assert need > 0 and scan(L, B=1, T=4096, state_in=NULL, size=need - 1) == -5 and scan(L, B=1, T=4096, state_in=NULL, ws=NULL) == -2
    assert L.wkv_selective_scan_forward_workspace(1, 1, 64, 16, 1, 1) == 0
    assert L.wkv_selective_scan_checkpoint_bytes(2, 33, 64, 20, 1, 1) == 2 * 3 * 64 * 32 * 4
    back = L.wkv_selective_scan_backward_workspace(2, 64, 64, 16, 1, 1)
    args = [rows(), rows(), ONE, rows(), rows(), ONE, rows(), ONE, NULL]
    grads = [ONE] * 12
    call = lambda a=args, g=grads, ws=ONE, n=back: L.wkv_selective_scan_backward(NULL, 2, 64, 64, 16, 1, 1, *a, *g, ws, n)
    assert call() == -8 and call(n=back - 1) == -5 and call(ws=NULL) == -2                 # gstate_in over gstate_out
    assert call(g=[NULL] + [ONE] * 11) == -2 and call(g=[ONE, ODD] + [ONE] * 10) == -4
    assert call(g=[ONE] * 9 + [NULL, ONE, ONE]) == -2                                     # a gate without its gradient


def test_convolution(L):
    call = lambda B=2, T=8, D=64, W=4, dtype=1, pd=1, x=None, w=ONE, s=NULL, y=ONE, out=ONE: L.wkv_causal_conv_forward(
        NULL, B, T, D, W, dtype, pd, 1, rows() if x is None else x, w, ONE, s, NULL, y, out)
    assert call() == -6 and call(s=ONE) == -8 and call(s=ONE, T=1) == -6
    assert call(W=1) == -1 and call(W=5) == -1 and call(T=0) == -1 and call(D=-1) == -1
    assert call(dtype=9) == -3 and call(dtype=1, pd=2) == -3 and call(dtype=1, pd=0) == -6
    assert call(w=NULL) == -2 and call(y=NULL) == -2 and call(x=rows(p=None)) == -2
    assert call(w=ODD) == -4 and call(x=rows(p=ctypes.c_void_p(9))) == -4
    need = L.wkv_causal_conv_backward_workspace(2, 8, 64, 4, 1)
    assert need > 0 and L.wkv_causal_conv_backward_workspace(2, 8, 64, 9, 1) == 0
    back = lambda n=need, g=(ONE, NULL, ONE, ONE, ONE, ONE): L.wkv_causal_conv_backward(NULL, 2, 8, 64, 4, 1, 1, 1, rows(), ONE, ONE, NULL, NULL, *g, ONE, n)
    assert back() == -6 and back(need - 1) == -5 and back(g=(ONE, ONE, ONE, ONE, ONE, ONE)) == -8 and back(g=(NULL, NULL, ONE, ONE, ONE, ONE)) == -2


def test_norm(L):
    call = lambda rows_=4, C=64, dt=1, rt=0, wt=1, x=ONE, r=ONE, w=ONE, y=ONE, q=NULL, s=NULL: L.wkv_rms_norm_forward(
        NULL, rows_, C, dt, rt, wt, 1e-5, x, 64, r, 64, w, y, q, s, ONE, NULL)
    assert call() == -6 and call(y=NULL, q=ONE, s=ONE) == -6
    assert call(rows_=0) == -1 and call(C=0) == -1 and call(dt=4) == -3 and call(rt=2) == -3 and call(wt=2) == -3
    assert call(y=NULL) == -2 and call(x=NULL) == -2 and call(q=ONE) == -2 and call(w=ODD) == -4 and call(r=ctypes.c_void_p(6)) == -4
    need = L.wkv_rms_norm_backward_workspace(4, 64)
    back = lambda n=need, x=ONE, r=NULL, gy=ONE: L.wkv_rms_norm_backward(NULL, 4, 64, 1, 0, 1, x, 64, r, 64, ONE, ONE, gy, NULL, ONE, NULL, ONE, ONE, n)
    assert back() == -6 and back(need - 1) == -5 and back(x=NULL) == -2 and back(gy=NULL) == -2 and back(x=NULL, r=ONE) == -6


def test_sampling(L):
    call = lambda rows_=2, V=100, dt=1, l=ONE, u=ONE, t=ONE, p=ONE: L.wkv_sample(NULL, rows_, V, dt, l, 100, u, NULL, 1.0, NULL, 0, NULL, 1.0, NULL, 0.0, t, p)
    assert call() == -6
    assert call(rows_=0) == -1 and call(V=0) == -1 and call(V=(1 << 20) + 1) == -1 and call(dt=3) == -3
    assert call(l=NULL) == -2 and call(u=NULL) == -2 and call(t=NULL) == -2 and call(p=NULL) == -2
    assert call(l=ctypes.c_void_p(5)) == -4 and call(t=ctypes.c_void_p(4)) == -4


def test_front_end_refuses_cpu_tensors():
    import rwkv_wkv_hip as W
    z = torch.zeros
    with pytest.raises(W.WKVError):
        W.ssm.causal_conv(z(1, 2, 8), z(8, 4))
    with pytest.raises(W.WKVError):
        W.ssm.selective_scan(z(1, 2, 8), z(1, 2, 8), z(8, 4), z(1, 2, 4), z(1, 2, 4))
    with pytest.raises(W.WKVError):
        W.ssm.rms_norm(z(2, 8), z(8))
    with pytest.raises(W.WKVError):
        W.ssm.rms_norm_fp8(z(2, 8), z(8))
    with pytest.raises(W.WKVError):
        W.sampling.sample(z(2, 8), z(2))
