"""GPU tier: what a bounded wait of the W8A8 layer leaves behind when it runs out.  The call is told to hold back one weight copy of its
first cluster (a flag of the C entry for this purpose), so that the products behind it never come: the waits give up after two
seconds, the kernel returns, and nothing that depends on the missing copy may look like a result."""
import subprocess
import sys

import pytest
import torch

from pyhip_b200 import _lib, int8_status, linear_int8, quantize_int8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _call(x, xs, w, ws, T, N, K, dt, out, variant, y, status):
    L = _lib.lib()
    bytes_ = (T * K + 255) // 256 * 256 + 4 * T
    scratch = torch.empty(bytes_, dtype=torch.uint8, device=DEV)
    _lib.check(L.b200moe_linear_int8(x.data_ptr(), K, dt, None if xs is None else xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, T, N, K, out, variant,
                                     scratch.data_ptr(), bytes_, None if status is None else status.data_ptr(), y.data_ptr(),
                                     torch.cuda.current_stream().cuda_stream), "linear_int8")
    torch.cuda.synchronize()


# split kernel over 1 and 8 CTAs of a cluster, its one-token form, and CTA pairs: tiles over the pairs, rows stored one by one, and
# two pairs that share K
@pytest.mark.parametrize("out", [_lib.T_BF16, _lib.T_FP16])
@pytest.mark.parametrize("T,N,K,variant", [(5, 300, 128, 1), (20, 300, 4096, 1), (1, 515, 2880, 1), (3000, 2824, 512, 2), (700, 1501, 4096, 2), (300, 512, 7168, 2)])
def test_a_wait_that_runs_out_leaves_no_plausible_values(T, N, K, variant, out):
    g = torch.Generator().manual_seed(T)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).to(DEV)
    ws = (torch.rand(N, generator=g) * 0.001 + 1e-5).to(DEV)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
    q, s = quantize_int8(x)
    rows = (x, None, _lib.T_BF16) if T == 1 else (q, s, _lib.T_INT8)
    args = (rows[0], rows[1], w, ws, T, N, K, rows[2], out)
    dtype = torch.bfloat16 if out == _lib.T_BF16 else torch.float16
    good, y = (torch.full((T, N), 77.0, dtype=dtype, device=DEV) for _ in range(2))
    _call(*args, variant, good, None)
    assert torch.isfinite(good).all()
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    _call(*args, variant | _lib.LINEAR_HOLD_BACK, y, status)
    assert int(status[0]) != 0
    lost = y.isnan()
    assert lost[0, 0] and torch.equal(y[~lost], good[~lost])
    tile = (min(T, 128), min(N, 128)) if variant == 1 else (min(T, 256), min(N, 128))      # of the first cluster, at least
    assert lost[:tile[0], :tile[1]].all()
    # the context, the library and the memory are as usable as before
    status.zero_()
    y.fill_(77.0)
    _call(*args, variant, y, status)
    assert torch.equal(y, good) and (status == 0).all()
    assert int8_status(DEV) == (0, 0)


CHILD = """
import ctypes, sys, torch
from pyhip_b200 import _lib, int8_status, linear_int8
q = torch.ones(20, 4096, dtype=torch.int8, device="cuda")
s, w, ws = torch.ones(20, device="cuda"), torch.ones(300, 4096, dtype=torch.int8, device="cuda"), torch.ones(300, device="cuda")
y = torch.empty(20, 300, dtype=torch.bfloat16, device="cuda")
L = _lib.lib()
assert int8_status() == (0, 0) and int8_status("cuda:0") == (0, 0) and int8_status(0) == (0, 0)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):                     # the device's first call of the layer, through the package and the C entry
    linear_int8(q, w, ws, x_scale=s)
    _lib.check(L.b200moe_linear_int8(q.data_ptr(), 4096, _lib.T_INT8, s.data_ptr(), w.data_ptr(), ws.data_ptr(), None, 20, 300, 4096, _lib.T_BF16,
                                     1 | HOLD, None, 0, None, y.data_ptr(), torch.cuda.current_stream().cuda_stream), "linear_int8")
assert int8_status() == (0, 0)
graph.replay()
word, cta = int8_status()
assert word != 0 and y.isnan().any(), (word, cta)
assert int8_status() == (word, cta)               # until the process ends
"""


def test_the_status_words_are_there_for_a_captured_first_call():
    code = CHILD.replace("HOLD", str(_lib.LINEAR_HOLD_BACK))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=str(_lib.PKG_DIR.parent))
    assert r.returncode == 0, r.stderr[-2000:]


def test_status_of_another_kind_of_device_is_refused():
    with pytest.raises(ValueError):
        int8_status("cpu")
