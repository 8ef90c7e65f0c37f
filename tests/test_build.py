"""What the build makes of a machine without all that the Python binding needs."""

from __future__ import annotations

import pytest

from lara_b200 import build


@pytest.fixture
def no_library(monkeypatch, tmp_path):
    """A library that is not built, whose compilation and link are recorded instead of run."""
    lib = tmp_path / "liblara_b200.so"
    monkeypatch.setattr(build, "LIB", lib)
    monkeypatch.setattr(build, "BINDING", tmp_path / "_binding.so")
    monkeypatch.setattr(build, "BUILD", tmp_path / "_build")
    monkeypatch.setattr(build, "_compile", lambda src, verbose: tmp_path / (src.stem + ".o"))
    run = build.subprocess.run

    def link(cmd, **kw):
        if "-shared" in cmd and str(lib.with_suffix(".so.tmp")) in cmd:
            lib.with_suffix(".so.tmp").write_bytes(b"")
            return build.subprocess.CompletedProcess(cmd, 0, "", "")
        return run(cmd, **kw)

    monkeypatch.setattr(build.subprocess, "run", link)
    return lib


def test_the_library_is_built_where_the_binding_fails(monkeypatch, no_library):
    def fails(force=False):
        raise RuntimeError("g++ failed")

    monkeypatch.setattr(build, "build_binding", fails)
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        build.build()
    assert no_library.exists()


@pytest.mark.parametrize("lacking", ["torch", "cuda", "g++", "headers"])
def test_the_binding_is_left_out_without_what_it_needs(monkeypatch, no_library, tmp_path, capsys, lacking):
    which, paths = build.shutil.which, build.sysconfig.get_paths
    if lacking == "torch":
        monkeypatch.setattr(build, "_torch_include", lambda: None)
    elif lacking == "cuda":
        (tmp_path / "torch" / "lib").mkdir(parents=True)
        monkeypatch.setattr(build, "_torch_include", lambda: tmp_path / "torch" / "include")
    elif lacking == "g++":
        monkeypatch.setattr(build.shutil, "which", lambda name: None if name == "g++" else which(name))
        monkeypatch.setenv("PATH", str(tmp_path))
    else:
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda *a, **kw: dict(paths(*a, **kw), include=str(tmp_path)))
    assert build.build() == no_library
    assert no_library.exists() and not (tmp_path / "_binding.so").exists()
    assert "left out" in capsys.readouterr().err
