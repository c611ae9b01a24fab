"""The build: the C library and the torch side of the training operators, of small sources in a folder of their own."""

import ctypes
import os
import shutil

import pytest

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")


@pytest.fixture
def build(tmp_path, monkeypatch):
    from nki_library_b200 import build
    if not os.path.exists(build._nvcc()) and shutil.which(build._nvcc()) is None:
        pytest.skip("no nvcc")
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "one.cu").write_text('extern "C" int one() { return 1; }\n')
    (csrc / "autograd.cpp").write_text("int two() { return 2; }\n")
    monkeypatch.setattr(build, "CSRC", str(csrc))
    monkeypatch.setattr(build, "BUILD", str(tmp_path / "build"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libone.so"))
    monkeypatch.setattr(build, "AUTOGRAD", str(tmp_path / "_two.so"))
    monkeypatch.setattr(build, "PKG", str(tmp_path))
    (tmp_path.parent / "include").mkdir(exist_ok=True)
    (tmp_path.parent / "include" / "b200moe.h").write_text("")
    return build


def test_the_library_does_not_need_the_torch_side(build, capfd):
    """A torch side that does not compile, link or start is reported; the library is there and nothing old beside it."""
    build.build_library()
    assert os.path.exists(build.AUTOGRAD)
    with open(os.path.join(build.CSRC, "autograd.cpp"), "w") as f:
        f.write("#error no headers\n")
    os.remove(build.LIB)
    assert build.build_library(force=True) == build.LIB
    assert ctypes.CDLL(build.LIB).one() == 1 and not os.path.exists(build.AUTOGRAD)
    assert "no headers" in capfd.readouterr().err


def test_no_compiler_for_the_torch_side(build, capfd, monkeypatch):
    monkeypatch.setattr(build, "_autograd_compile", lambda source, target: ["/nowhere/g++"])
    build.build_library()
    assert ctypes.CDLL(build.LIB).one() == 1
    assert "_two.so" in capfd.readouterr().err


def test_a_library_that_does_not_compile_raises(build):
    with open(os.path.join(build.CSRC, "one.cu"), "a") as f:
        f.write("#error not this one\n")
    with pytest.raises(RuntimeError, match="compilation failed"):
        build.build_library()


def test_another_torch_rebuilds_the_torch_side(build, monkeypatch):
    """Also where the build in between failed."""
    import torch
    build.build_library()
    first = os.stat(build.AUTOGRAD).st_mtime_ns
    build.build_library()
    assert os.stat(build.AUTOGRAD).st_mtime_ns == first
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    compile_ = build._autograd_compile
    monkeypatch.setattr(build, "_autograd_compile", lambda source, target: ["false"])
    build.build_library()
    assert not os.path.exists(build.AUTOGRAD)
    monkeypatch.setattr(build, "_autograd_compile", compile_)
    build.build_library()
    assert os.stat(build.AUTOGRAD).st_mtime_ns > first
