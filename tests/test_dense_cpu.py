"""CPU tier: the C ABI of the dense operators rejects bad arguments before it launches anything, the Python surface fails loudly
without a CUDA device, and the oracle's quantiser is what its definition says."""
import ctypes

import pytest
import torch

from oracle import dense_oracle as orc
from pyhip_b200 import _lib

P = 4096        # a non-null, 16-byte aligned address that no rejected call touches


@pytest.fixture(scope="module")
def L():
    _lib.build()
    return _lib.lib()


def _linear(L, x=P, stride=64, dt=_lib.T_BF16, xs=None, w=P, ws=P, bias=None, T=40, N=32, K=64, out=_lib.T_BF16, variant=0, work=P, size=1 << 20, y=P):
    return L.b200moe_linear_int8(x, stride, dt, xs, w, ws, bias, T, N, K, out, variant, work, size, None, y, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(N=0), dict(K=0), dict(K=24), dict(K=1 << 17), dict(out=_lib.T_FP32), dict(dt=4), dict(dt=-1),
                                 dict(variant=3), dict(x=None), dict(w=None), dict(ws=None), dict(y=None), dict(w=P + 8), dict(y=P + 2), dict(work=None),
                                 dict(work=P + 4), dict(size=4 * 64), dict(dt=_lib.T_INT8), dict(dt=_lib.T_INT8, xs=P, stride=80),
                                 dict(dt=_lib.T_INT8, xs=P, x=P + 1), dict(K=16400, stride=16400)])
def test_linear_int8_arguments(L, bad):
    assert _linear(L, **bad) < 0
    assert L.b200moe_last_error()


def test_empty_calls_launch_nothing(L):
    assert _linear(L, T=0, x=None, y=None, work=None, size=0) == 0
    assert L.b200moe_quantize_int8(None, 64, 0, 64, _lib.T_BF16, None, None, None) == 0
    assert _norm(L, T=0) == 0


def _norm(L, y=P, ys=64, r=None, rs=0, w=None, gate=None, gs=0, wn=P, T=4, H=64, dt=_lib.T_BF16, bits=0, kind=_lib.GATE_NONE, h=None, n=P, q=None, qs=None):
    return L.b200moe_block_norm(y, ys, r, rs, w, gate, gs, wn, T, H, dt, bits, kind, 1.0, 1e-6, h, n, q, qs, None, None)


@pytest.mark.parametrize("bad", [dict(T=-1), dict(H=0), dict(H=16385), dict(dt=3), dict(kind=4), dict(kind=1), dict(gate=P), dict(ys=-1),
                                 dict(wn=None), dict(n=None), dict(q=P), dict(qs=P), dict(y=None)])
def test_block_norm_arguments(L, bad):
    assert _norm(L, **bad) < 0


def test_block_norm_bwd_arguments(L):
    def call(y=P, r=None, w=P, gate=None, wn=None, T=4, H=64, dt=_lib.T_BF16, kind=0, rstd=P, dh=P, dn=None, dy=P, dr=None, dw=P, dg=None, dwn=None,
             work=P, size=1 << 20):
        return L.b200moe_block_norm_bwd(y, 64, r, 64, w, gate, 0, wn, T, H, dt, 0, kind, 1.0, rstd, dh, dn, dy, dr, dw, dg, dwn, work, size, None)

    b = ctypes.c_int64()
    assert L.b200moe_block_norm_bwd_workspace(4, 64, 3, ctypes.byref(b)) < 0
    assert L.b200moe_block_norm_bwd_workspace(4, 64, _lib.T_BF16, None) < 0
    for bad in (dict(H=0), dict(dt=4), dict(kind=2), dict(w=None), dict(dwn=P), dict(dr=P), dict(dg=P), dict(dn=P), dict(rstd=None), dict(y=None),
                dict(work=None), dict(size=16)):
        assert call(**bad) < 0, bad


def test_router_arguments(L):
    def call(x=P, stride=16, T=4, E=16, K=2, dt=_lib.T_FP32, scoring=0, cu=None, S=1, w=P, ids=P, counts=P, bal=P, z=P, lse=None, seg=None, coef=None,
             stats=None, work=P, size=1 << 20):
        return L.b200moe_router_forward(x, stride, T, E, K, dt, scoring, 1, None, cu, S, w, ids, counts, bal, z, lse, seg, coef, stats, work, size, None)

    for bad in (dict(T=-1), dict(E=0), dict(E=1025), dict(K=0), dict(K=17), dict(K=33, E=64, stride=64), dict(dt=3), dict(scoring=2), dict(S=0),
                dict(S=2), dict(stride=-1), dict(x=None), dict(w=None), dict(ids=None), dict(counts=None), dict(bal=None), dict(z=None), dict(lse=P),
                dict(work=None), dict(work=P + 4), dict(size=64)):
        assert call(**bad) < 0, bad

    def back(x=P, T=4, E=16, K=2, lse=P, seg=P, coef=P, stats=P, ids=P, w=P, out=P):
        return L.b200moe_router_backward(x, 16, T, E, K, 0, 0, 1, lse, seg, coef, stats, ids, w, None, None, None, out, None)

    for bad in (dict(x=None), dict(lse=None), dict(seg=None), dict(coef=None), dict(stats=None), dict(ids=None), dict(w=None), dict(out=None), dict(K=17)):
        assert back(**bad) < 0, bad
    assert back(T=0, x=None) == 0
    b = ctypes.c_int64()
    assert L.b200moe_router_workspace(4, 16, 1, ctypes.byref(b)) == 0 and b.value > 0
    assert L.b200moe_router_workspace(4, 2000, 1, ctypes.byref(b)) < 0


def test_python_surface_fails_loudly_without_cuda():
    from pyhip_b200 import fused_post_norm, fused_pre_norm, fused_router, linear_int8, quantize_int8
    x = torch.zeros(2, 64)
    for call in (lambda: linear_int8(x, torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)), lambda: quantize_int8(x),
                 lambda: fused_pre_norm(x, torch.ones(64)), lambda: fused_post_norm(x, x), lambda: fused_router(x, 2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_oracle_quantiser_rounds_to_nearest():
    x = torch.randn(50, 200, dtype=torch.float64).float()
    q, s = orc.quantize_int8(x)
    assert (q.abs() <= 127).all()
    assert ((q * s.double()[:, None] - x.double()).abs() <= s.double()[:, None] / 2).all()
