"""What build.py needs and when it rebuilds."""
import os
import subprocess
import sys
import time
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def builder():
    from __graft_entry__ import _load_builder
    return _load_builder()


def test_the_library_builds_without_torch():
    """A caller of the C ABI needs nvcc alone: the Python module is left out where torch cannot be imported."""
    code = f"""
import sys
sys.modules["torch"] = None
sys.path.insert(0, {ROOT!r})
from __graft_entry__ import _load_builder
b = _load_builder()
print(b.build() == b.OUT)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=1500)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.strip().endswith("True")


def test_the_python_module_follows_torch_and_python(builder, monkeypatch, tmp_path):
    """Built against the torch and Python that run: another version of either builds it again, the same ones do not."""
    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")
    monkeypatch.setattr(builder, "HOSTCALL", str(tmp_path / "dsuf_hostcall.so"))
    monkeypatch.setattr(builder, "HOSTCALL_FOR", str(tmp_path / "hostcall.for"))
    monkeypatch.setattr(builder, "subprocess", types.SimpleNamespace(run=run))
    assert builder.build_hostcall() == builder.HOSTCALL and len(runs) == 1
    builder.build_hostcall()
    assert len(runs) == 1
    import torch
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    builder.build_hostcall()
    assert len(runs) == 2
    builder.build_hostcall()
    assert len(runs) == 2
    old = time.time() - 10 ** 9
    os.utime(builder.HOSTCALL, (old, old))      # older than its sources
    builder.build_hostcall()
    assert len(runs) == 3
