"""When the torch binding is built, and what it refuses to be loaded into."""
import os
import subprocess
import sys
import time

import pytest

pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(monkeypatch, tmp_path):
    """The builder with a stamp and a binding of its own, and no compiler: what it would start is listed."""
    from rocal_b200 import build as B
    started = []
    monkeypatch.setattr(B, "HEAD_STAMP", str(tmp_path / "stamp"))
    monkeypatch.setattr(B, "HEAD_LIB", str(tmp_path / "_head.so"))
    monkeypatch.setattr(B.subprocess, "Popen", lambda command, **kw: started.append(command) or "process")
    (tmp_path / "_head.so").write_bytes(b"")
    future = time.time() + 1000
    os.utime(tmp_path / "_head.so", (future, future))
    return B, started


def test_a_binding_of_another_torch_is_out_of_date(build, monkeypatch):
    """The binding's file is newer than its sources in every case: what differs is what it was compiled against."""
    B, started = build
    with open(B.HEAD_STAMP, "w") as f:
        f.write(B.head_stamp())
    assert B.build_head() is None and not started
    with open(B.HEAD_STAMP, "w") as f:
        f.write(B.head_stamp().replace("torch ", "torch 1."))
    assert B.build_head() == "process" and len(started) == 1
    with open(B.HEAD_STAMP, "w") as f:
        f.write(B.head_stamp().replace(sys.prefix, "/elsewhere"))
    assert B.build_head() == "process" and len(started) == 2
    os.remove(B.HEAD_STAMP)                                    # nobody knows what it was compiled against
    assert B.build_head() == "process" and len(started) == 3
    assert "-ltorch_python" in started[0]


def test_the_library_builds_without_torch(build, monkeypatch, capsys):
    """The library needs no torch, and its build did not before there was a binding."""
    import importlib.util
    B, started = build
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    assert B.build_head() is None and B.build_head(force=True) is None and not started
    assert "not built" in capsys.readouterr().err


def test_the_version_is_torch_s_own(monkeypatch):
    """Also where torch has no package metadata (a build from sources on the path)."""
    import importlib.metadata

    import torch
    from rocal_b200 import build as B

    def missing(name):
        raise importlib.metadata.PackageNotFoundError(name)
    monkeypatch.setattr(importlib.metadata, "version", missing)
    assert B.head_versions() == "torch %s, Python %d.%d" % ((torch.__version__,) + sys.version_info[:2])


def test_a_torch_without_cuda_has_no_binding(build, monkeypatch, tmp_path):
    import importlib.machinery
    import importlib.util
    B, started = build
    spec = importlib.machinery.ModuleSpec("torch", None, origin=str(tmp_path / "torch" / "__init__.py"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: spec)
    assert B.build_head() is None and not started


def test_a_binding_of_another_torch_is_not_loaded(tmp_path):
    code = ("import sys, rocal_b200.build as B\nB.HEAD_STAMP = sys.argv[1]\n"
            "try:\n    import rocal_b200._torch\nexcept ImportError as e:\n    print('refused:', e)\nelse:\n    print('loaded')\n")

    def said(stamp):
        (tmp_path / "stamp").write_text(stamp)
        r = subprocess.run([sys.executable, "-c", code, str(tmp_path / "stamp")], cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        return r.stdout
    from rocal_b200 import build as B
    assert said(B.head_stamp()) == "loaded\n"
    assert "built for torch 1.0, Python 3.9" in said("torch 1.0, Python 3.9\n/elsewhere\n")
