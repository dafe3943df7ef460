"""What csm-hf_amd/build.py builds, with a compiler that only writes what it was asked for: the C libraries need neither torch nor g++, and the operators'
binding for torch tensors goes with the torch that it was built for."""
import importlib.util
import os
import shutil
import stat
import subprocess
import sys

import pytest
import torch

from csm_hf_amd import build as real_build, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COMPILER = '''#!%s
import sys
a = sys.argv[1:]
out = a[a.index("-o") + 1]
text = "\\n".join(a).encode()
for f in a:
    if f.endswith(".o") and f != out:
        text += open(f, "rb").read()
open(out, "wb").write(text)
open(%r, "a").write(out + "\\n")
'''


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """a copy of the sources, and hipcc and g++ in front of PATH that log what they wrote"""
    shutil.copytree(os.path.join(ROOT, "csm-hf_amd", "csrc"), tmp_path / "csm-hf_amd" / "csrc", ignore=shutil.ignore_patterns("build*", "*.o"))
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    shutil.copy(os.path.join(ROOT, "csm-hf_amd", "build.py"), tmp_path / "csm-hf_amd" / "build.py")
    tools = tmp_path / "bin"
    tools.mkdir()
    for name in ("hipcc", "g++"):
        (tools / name).write_text(COMPILER % (sys.executable, str(tmp_path / "log")))
        (tools / name).chmod(stat.S_IRWXU)
    monkeypatch.setenv("HIPCC", str(tools / "hipcc"))
    monkeypatch.setenv("PATH", f"{tools}:/usr/bin:/bin")
    return tmp_path


def _run(tree, *flags):
    return subprocess.run([sys.executable, *flags, str(tree / "csm-hf_amd" / "build.py")], capture_output=True, text=True)


def _built(tree):
    return {f for f in os.listdir(tree / "csm-hf_amd") if f.endswith(".so")}


def _module(tree):
    spec = importlib.util.spec_from_file_location("copied_build", tree / "csm-hf_amd" / "build.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_c_libraries_need_no_torch(tree):
    r = _run(tree, "-S")              # without site-packages there is no torch
    assert r.returncode == 0, r.stderr
    assert _built(tree) == {"libcsm_hip.so", "libcsm_ops.so"} and "_ops_binding.so" in r.stderr


def test_c_libraries_stand_where_the_binding_cannot_be_built(tree):
    (tree / "bin" / "g++").write_text("#!/bin/sh\necho no headers >&2\nexit 1\n")
    r = _run(tree)
    assert _built(tree) == {"libcsm_hip.so", "libcsm_ops.so"}
    assert r.returncode != 0 and "no headers" in r.stderr       # (but the command says so)
    b = _module(tree)
    os.utime(b.OPS_LIB)
    assert b.build_library() == b.LIB                           # the libraries are there: no error


def test_binding_is_built_anew_for_another_torch(tree, monkeypatch):
    b = _module(tree)
    b.build_library()
    assert _built(tree) == {"libcsm_hip.so", "libcsm_ops.so", "_ops_binding.so"} and b.binding_stamp() in open(b.OPS_BINDING, errors="replace").read()
    log = lambda: (tree / "log").read_text().split("\n")[:-1]  # noqa: E731
    n = len(log())
    b.build_library()
    assert len(log()) == n                                      # nothing is older than its sources
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    b.build_library()
    assert [os.path.basename(f) for f in log()[n:]] == ["binding.o", "_ops_binding.so"]
    assert "torch 0.0.1" in open(b.OPS_BINDING, errors="replace").read()


def test_binding_for_another_torch_is_refused_when_loaded(monkeypatch):
    monkeypatch.setattr(ops, "_binding", None)
    assert ops._load_binding().built_for == real_build.binding_stamp()
    monkeypatch.setattr(ops, "_binding", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(RuntimeError, match="built for another torch.*csm_hf_amd.build"):
        ops._load_binding()


def test_binding_without_a_stamp_is_refused_when_loaded(monkeypatch):
    monkeypatch.setattr(ops, "_binding", None)
    ops._load_binding()
    monkeypatch.setattr(ops, "_binding", None)
    monkeypatch.setattr(importlib.import_module(ops.__package__), "_ops_binding", object())
    with pytest.raises(RuntimeError, match="built for another torch.*csm_hf_amd.build"):
        ops._load_binding()
