"""What the build makes of the torch that it finds (no GPU)."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")

from secure_infer_b200 import _native, build  # noqa: E402


def python(code, **env):
    return subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, sys.argv[1])\n" + code, str(ROOT)],
                          env=dict(os.environ, **env), capture_output=True, text=True, timeout=300)


def test_the_library_is_built_without_torch():
    r = python("sys.modules['torch'] = None\nfrom secure_infer_b200 import build, _native\n"
               "build.subprocess.run = lambda *a, **k: None   # the library is there\n"
               "print(build.build()); _native.lib()")
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.strip() == str(_native.LIB_PATH) and "not built" in r.stderr


@pytest.fixture
def made(monkeypatch, tmp_path):
    """An extension newer than its sources, and what a build of it would run."""
    target, ran = tmp_path / "paged_python.so", []
    target.write_bytes(b"")
    monkeypatch.setattr(build, "PAGED", target)
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, check: ran.append(cmd))
    return target, ran


def test_another_torch_makes_the_extension_stale(made, monkeypatch):
    target, ran = made
    target.with_suffix(".torch").write_text(_native.paged_made_for())
    assert build.build_paged() == target and not ran
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build_paged()
    assert len(ran) == 1
    build.build_paged()   # the new one is remembered
    assert len(ran) == 1
    target.with_suffix(".torch").unlink()
    build.build_paged()
    assert len(ran) == 2


def test_an_extension_of_another_torch_is_not_loaded(made, monkeypatch):
    target, _ = made
    monkeypatch.setattr(_native, "_paged", None)
    monkeypatch.setattr(_native, "LIB_PATH", target.parent / "libsecure_infer.so")
    target.with_suffix(".torch").write_text("python 3.1, torch 0.1")
    with pytest.raises(_native.NativeLibraryMissing, match="torch 0.1.*build it again"):
        _native.paged_ops()


def test_the_extension_finds_its_own_library(tmp_path):
    """Another file of the library's name on LD_LIBRARY_PATH, as where the library that this one replaces is in use."""
    (tmp_path / "x.c").write_text("int secure_infer_other(void) { return 1; }\n")
    subprocess.run([os.environ.get("CC", "gcc"), "-shared", "-fPIC", "-o", str(tmp_path / "libsecure_infer.so"),
                    str(tmp_path / "x.c")], check=True)
    r = python("from secure_infer_b200 import _native\nprint(_native.paged_ops().attend)",
               LD_LIBRARY_PATH=f"{tmp_path}:{os.environ.get('LD_LIBRARY_PATH', '')}")
    assert r.returncode == 0, r.stderr[-2000:]
