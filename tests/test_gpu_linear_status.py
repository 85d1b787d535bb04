"""GPU tier: what a bounded wait of the W8A8 layer leaves behind when it runs out.  The call is told to hold back one weight copy of its
first cluster (a flag of the C entry for this purpose), so that the products behind it never come: the waits give up after two
seconds and the kernel returns."""
import subprocess
import sys

import pytest

from pyhip_b200 import _lib, int8_status

pytestmark = pytest.mark.gpu


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
assert word != 0, (word, cta)
assert int8_status() == (word, cta)               # until the process ends
"""


def test_the_status_words_are_there_for_a_captured_first_call():
    code = CHILD.replace("HOLD", str(_lib.LINEAR_HOLD_BACK))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=str(_lib.PKG_DIR.parent))
    assert r.returncode == 0, r.stderr[-2000:]


def test_status_of_another_kind_of_device_is_refused():
    with pytest.raises(ValueError):
        int8_status("cpu")
