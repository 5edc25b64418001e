"""The native build compiles again what was compiled with other flags, from other sources, or not to the end."""
from pathlib import Path

import pytest

from deeplearning4j_amd.native import build as B


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of its own; commands are recorded and leave their output file."""
    src = tmp_path / "csrc"
    src.mkdir()
    for name in ("a.hip", "b.hip", "c.cpp", "common.h"):
        (src / name).write_text("// " + name)
    monkeypatch.setattr(B, "CSRC", src)
    monkeypatch.setattr(B, "OBJ", tmp_path / "_obj")
    for lib in ("HIP_LIB", "RT_LIB", "DEV_LIB"):
        monkeypatch.setattr(B, lib, tmp_path / (lib + ".so"))
    monkeypatch.setattr(B, "EXTRA_FLAGS", {"b.hip": ("-Dof_b",)})
    ran = []

    def run(cmd):
        ran.append([str(c) for c in cmd])
        if "fail" in ran[-1]:
            raise RuntimeError("command failed")
        Path(cmd[list(map(str, cmd)).index("-o") + 1]).write_text("object")
        return ""
    monkeypatch.setattr(B, "_run", run)

    def compiled():
        out = sorted(Path(c[c.index("-c") + 1]).name for c in ran if "-c" in c)
        linked = any("-shared" in c for c in ran)
        del ran[:]
        return out, linked
    return compiled


def test_nothing_is_compiled_twice(tree):
    B.build()
    assert tree() == (["a.hip", "b.hip", "c.cpp"], True)
    B.build()
    assert tree() == ([], False)
    B.build(force=True)
    assert tree() == (["a.hip", "b.hip", "c.cpp"], True)


def test_other_flags_compile_again(tree, monkeypatch):
    B.build()
    tree()
    monkeypatch.setattr(B, "EXTRA_FLAGS", {"b.hip": ("-Dof_b", "-O2")})
    B.build()
    assert tree() == (["b.hip"], True)
    monkeypatch.setattr(B, "HIP_FLAGS", B.HIP_FLAGS + ("-Dmore",))
    B.build()
    assert tree() == (["a.hip"], True)
    B.build()
    assert tree() == ([], False)


def test_objects_of_unknown_flags_compile_again(tree):
    B.build()
    tree()
    for f in B.OBJ.iterdir():
        if f.suffix != ".o":
            f.unlink()
    B.build()
    assert tree() == (["a.hip", "b.hip", "c.cpp"], True)


def test_a_failed_compilation_is_taken_up_again(tree, monkeypatch):
    B.build()
    tree()
    monkeypatch.setattr(B, "EXTRA_FLAGS", {"b.hip": ("fail",)})
    with pytest.raises(RuntimeError):
        B.build(jobs=1)
    tree()
    monkeypatch.setattr(B, "EXTRA_FLAGS", {"b.hip": ("-Dof_b",)})          # (back to the flags of the object that is there: it was not replaced)
    B.build()
    assert tree()[0] == ["b.hip"]
