"""CPU tier: what loading the built libraries does when they are not of this source tree."""
import subprocess

import pytest

from pyhip_b200 import _lib


def _stub(path, names, version):
    src = path / "stub.c"
    src.write_text("".join(f"int {n}(void) {{ return {version}; }}\n" for n in names))
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(path / "stub.so"), str(src)], check=True)
    return path / "stub.so"


@pytest.mark.parametrize("names,version", [([n for n in _lib.EXPORTS if "router_" not in n], _lib.ABI_VERSION),      # built before an entry came
                                           (["b200moe_version"], _lib.ABI_VERSION - 1), (_lib.EXPORTS, _lib.ABI_VERSION + 1)])
def test_a_library_of_another_version_says_so(tmp_path, monkeypatch, names, version):
    monkeypatch.setattr(_lib, "LIB_PATH", _stub(tmp_path, names, version))
    with pytest.raises(RuntimeError, match="rebuild"):
        _lib.lib.__wrapped__()


def test_a_binding_for_another_torch_is_rebuilt_and_not_loaded(monkeypatch):
    import torch
    _lib.build()
    assert _lib._dense_fits() and _lib.dense.__wrapped__() is not None
    ran = []
    monkeypatch.setattr(_lib.subprocess, "run", lambda cmd, **_: ran.append(cmd) or subprocess.CompletedProcess(cmd, 0, "", ""))
    _lib.build()
    assert not ran
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    _lib.build()
    assert len(ran) == 1 and str(_lib.DENSE_PATH) in ran[0]
    with pytest.raises(ImportError, match="rebuild"):
        _lib.dense.__wrapped__()
