"""GPU tier: the norms' gradients for rows far from one.  Bounds as in test_gpu_norm.py: they are relative to each value's size, so
they hold at every scale at which a row's sum of squares and the results are normal 32-bit numbers."""
import pytest
import torch

from oracle import dense_oracle as orc
from pyhip_b200 import fused_post_norm
from test_gpu_norm import _grads, _inputs, _near, _randn

pytestmark = pytest.mark.gpu


# (H, plain or ring form): 288 is below the ring's widths, 1001 off the 16-byte grid; 7168 takes 8 values a thread
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(33, 288), (5, 1001), (40, 2880), (20, 7168)])
@pytest.mark.parametrize("scale,eps", [(2.0 ** 46, 1e-6), (2.0 ** 53, 1e-6), (2.0 ** 55, 1e-6), (2.0 ** -50, 1e-36)])
def test_gradients_of_large_and_small_rows(T, H, dtype, scale, eps):
    for k, (post, gate, nxt) in enumerate([(True, "token", True), (True, "channel", True), (True, None, False), (False, None, True), (True, "full", True)]):
        i = _inputs(T, H, dtype, dtype, post, gate, nxt, seed=T + H + k)
        i = dict(i, y=i["y"] * scale, residual=i["residual"] * scale)          # a power of two: exact
        o = orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 0.75, eps, i["next_weight"])
        dh, dn = _randn(T, H, seed=k, dtype=dtype), _randn(T, H, seed=k + 50, dtype=dtype) if nxt else None
        # part of the gradient lies along the rows, where it is the difference of two large terms that has to come out
        dh = dh + (i["y"] / scale).to(dtype)
        if nxt:
            dn = dn + (o["h"] / scale).to(dtype)
        for t in i.values():
            if t is not None:
                t.requires_grad_(True)
        r = fused_post_norm(i["y"], i["residual"], i["weight"], gate=i["gate"], residual_scale=0.75, eps=eps, next_weight=i["next_weight"])
        _near((r[0] if nxt else r).detach(), o["h"].detach(), o["h_size"].detach(), "h")
        if nxt:
            _near(r[1].detach(), o["n"].detach(), o["n_size"].detach(), "n")
        got = _grads(i, r, dh, dn)
        want = orc.block_norm_grads(o, i["residual"], i["weight"], i["gate"], 0.75, i["next_weight"], dh, dn)
        for name in want:
            _near(got[name], want[name][0].detach(), want[name][1].detach(), f"{name} (case {k})")
