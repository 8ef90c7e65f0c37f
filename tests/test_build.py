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


def _fake_torch(monkeypatch, tmp_path):
    root = tmp_path / "torch"
    (root / "lib").mkdir(parents=True)
    (root / "lib" / "libc10_cuda.so").write_bytes(b"")
    monkeypatch.setattr(build, "_torch_include", lambda: root / "include")
    return root / "version.py"


def test_the_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    version = _fake_torch(monkeypatch, tmp_path)
    out, built = tmp_path / build.BINDING.name, []
    monkeypatch.setattr(build, "BINDING", out)
    monkeypatch.setattr(build, "BUILD", tmp_path / "_build")

    def compiler(cmd, **kw):
        built.append(cmd)
        open(cmd[cmd.index("-o") + 1], "wb").close()
        return build.subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    for text, times in (("__version__ = '2.11.0'", 1), ("__version__ = '2.11.0'", 1), ("__version__ = '2.12.0'", 2),
                        ("__version__ = '2.12.0'", 2)):
        version.write_text(text)
        assert build.build_binding() == out and out.exists()
        assert len(built) == times


def test_the_binding_names_its_python_and_torch():
    import sysconfig

    import torch

    from lara_b200 import _binding

    assert build.BINDING.name.endswith(sysconfig.get_config_var("EXT_SUFFIX")) and "cpython" in build.BINDING.name
    assert torch.__version__.startswith(_binding.torch_version)


def test_a_binding_of_another_torch_is_refused():
    import subprocess
    import sys

    code = "import torch; torch.__version__ = '1.0.0'; import lara_b200.ops as o; x = torch.zeros((1, 1, 64)); o.qk_norm_rope(x, x)"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=build.PKG.parent)
    assert r.returncode != 0 and "built for torch" in r.stderr and "--force" in r.stderr


def test_the_front_end_works_without_the_binding():
    """Its own calls name what is missing; those that do not use it are there."""
    import subprocess
    import sys

    code = """if True:
        import sys
        sys.modules["lara_b200._binding"] = None
        import torch
        from lara_b200 import kvquant, ops, paged, parallel
        assert ops.Decoder and ops.gqa_prefill and paged.PagedKVCache and ops.rope_table(8, 8, device="cpu").shape == (8, 8)
        x = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
        try:
            ops.qk_norm_rope(x, x)
        except ImportError as e:
            print("refused:", e)
    """
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=build.PKG.parent)
    assert r.returncode == 0, r.stderr
    assert "refused: lara_b200._binding cannot be loaded" in r.stdout and "lara_b200.build" in r.stdout
