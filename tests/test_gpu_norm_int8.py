"""GPU tier: 8-bit output of the norms where a CTA walks over many rows, so that the reductions of one row (one for each norm, one for
the largest value) alternate over two sets of slots with those of the next."""
import pytest
import torch

from oracle import dense_oracle as orc
from pyhip_b200 import fused_post_norm, fused_pre_norm
from test_gpu_norm import C, _inputs, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(5000, 96), (5000, 512), (3001, 1001), (2500, 2880), (1300, 7168), (700, 16384)])
@pytest.mark.parametrize("post,gate", [(True, "token"), (True, None), (False, "channel"), (False, None)])
def test_int8_rows_of_long_batches(T, H, dtype, post, gate):
    i = _inputs(T, H, dtype, dtype, post, gate, True, seed=T)
    run = lambda j: fused_post_norm(j["y"], j["residual"], j["weight"], gate=j["gate"], next_weight=j["next_weight"], quant="int8")  # noqa: E731
    h, q, s = run(i)
    o = orc.block_norm(i["y"], i["residual"], i["weight"], i["gate"], 1.0, 1e-6, i["next_weight"])
    _near(h, o["h"], o["h_size"], "h")
    # the scale is that of a row within C of the exact one; a value is within half a step of it (as for short batches)
    amax, slack = o["n"].abs().amax(-1), C * o["n_size"].amax(-1)
    assert ((s.double() * 127 - amax).abs() <= slack + amax * 2.0 ** -23).all()
    assert ((q.double() * s.double()[:, None] - o["n"]).abs() <= s.double()[:, None] * 0.5 + C * o["n_size"]).all()
    # a row is the same whatever else its CTA works on
    for lo in range(0, T, T // 7):
        part = slice(lo, min(lo + 100, T))
        few = run(dict(i, y=i["y"][part], residual=i["residual"][part], gate=i["gate"][part] if gate == "token" else i["gate"]))
        assert all(torch.equal(a, b[part]) for a, b in zip(few, (h, q, s)))
    a = fused_pre_norm(i["y"], i["next_weight"], residual=i["residual"], quant="int8")
    b = fused_pre_norm(i["y"][-50:], i["next_weight"], residual=i["residual"][-50:], quant="int8")
    assert all(torch.equal(v[-50:], w) for v, w in zip(a, b))
