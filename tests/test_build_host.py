"""CPU tests of the build's steps, with a compiler that only writes its output."""

import importlib.util
import os
import stat

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

COMPILER = """#!/bin/sh
echo "$0 $*" >> {log}
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then echo built > "$2"; fi
  shift
done
"""


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build module with its outputs and compilers under tmp_path."""
    spec = importlib.util.spec_from_file_location("ilqr_build_test", os.path.join(ROOT, "ca-ac-mpc_b200", "csrc", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.log = tmp_path / "log"
    mod.log.write_text("")
    for name, var in (("nvcc", "NVCC"), ("g++", "CXX")):
        f = tmp_path / name
        f.write_text(COMPILER.format(log=mod.log))
        f.chmod(f.stat().st_mode | stat.S_IXUSR)
        monkeypatch.setattr(mod, var, str(f))
    for var, name in (("OBJ_DIR", "obj"), ("LIB", "lib.so"), ("PROBE_LIB", "probe.so"), ("BINDING", "binding.so")):
        monkeypatch.setattr(mod, var, str(tmp_path / name))
    return mod


def _ran(mod):
    lines = mod.log.read_text().splitlines()
    mod.log.write_text("")
    return ["lib" if " -shared -o " in x else "probe" if "fma_probe" in x else "binding" if "ilqr_torch" in x else "object"
            for x in lines]


def test_everything_once(build):
    assert build.build() == build.LIB
    ran = _ran(build)
    assert set(ran) == {"object", "lib", "probe", "binding"} and ran[-3:] == ["lib", "probe", "binding"]
    build.build()
    assert _ran(build) == []


def test_without_what_the_binding_needs(build, monkeypatch, capsys):
    """The library and the probe are built, a binding of earlier sources goes."""
    with open(build.BINDING, "w") as f:
        f.write("old")
    os.utime(build.BINDING, (1, 1))
    monkeypatch.setattr(build, "CXX", "no-such-compiler-here")
    assert build.build() == build.LIB
    assert "binding" not in _ran(build) and os.path.exists(build.LIB) and os.path.exists(build.PROBE_LIB)
    assert not os.path.exists(build.BINDING) and "no-such-compiler-here" in capsys.readouterr().err
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": "/nowhere"})
    monkeypatch.setattr(build, "CXX", build.NVCC)
    assert build.binding_needs() == ["/nowhere/Python.h"]
    with open(build.BINDING, "w") as f:
        f.write("current")
    build.build()
    assert os.path.exists(build.BINDING) and "Python.h" in capsys.readouterr().err


def test_a_binding_that_does_not_compile_is_an_error_after_the_rest(build, monkeypatch):
    monkeypatch.setattr(build, "CXX", "/bin/false")
    with pytest.raises(RuntimeError, match="binding"):
        build.build()
    assert os.path.exists(build.LIB) and os.path.exists(build.PROBE_LIB)


def test_another_torch_or_python_rebuilds_the_binding(build, monkeypatch):
    """Also one whose files are older than the binding."""
    import torch
    build.build()
    _ran(build)
    for owner, name, value in ((torch, "__version__", "9.9.9"), (torch.version, "git_version", "0" * 40),
                               (build.sys, "version", "3.99")):
        with monkeypatch.context() as m:
            m.setattr(owner, name, value)
            build.build()
            assert _ran(build) == ["binding"], name
            build.build()
            assert _ran(build) == [], name
        build.build()
        assert _ran(build) == ["binding"], name
    os.utime(build.BINDING, (1, 1))
    build.build()
    assert _ran(build) == ["binding"]


def test_a_binding_that_failed_is_tried_again(build, monkeypatch):
    build.build()
    os.utime(build.BINDING, (1, 1))
    with monkeypatch.context() as m:
        m.setattr(build, "CXX", "/bin/false")
        with pytest.raises(RuntimeError, match="binding"):
            build.build()
    _ran(build)
    build.build()
    assert _ran(build) == ["binding"]
