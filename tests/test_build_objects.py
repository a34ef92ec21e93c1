"""When an object of the library is compiled anew: with a stand-in for the compiler, runs without a GPU."""

import os
from pathlib import Path

import pytest

from wave_b200 import build


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """compile(variant) -> whether the compiler ran; it writes an object and what that was made from, as nvcc does."""
    header = tmp_path / "part.cuh"
    source = tmp_path / "unit.cu"
    for p in (header, source):
        p.write_text("")
    objects = tmp_path / "objects"
    objects.mkdir()
    ran = []

    def run(cmd):
        ran.append(cmd)
        unit = Path(cmd[cmd.index("-o") + 1])
        unit.write_text("")
        Path(cmd[cmd.index("-MF") + 1]).write_text(f"{unit} : {source} \\\n    {header}\n")
        return ""

    monkeypatch.setattr(build, "_run", run)

    def compile(variant=(), verbose=False):
        before = len(ran)
        assert build._compile("nvcc", source, objects, list(variant), False, verbose) == objects / "unit.o"
        return len(ran) > before

    compile.touch = lambda p, to: os.utime(p, (to, to))
    compile.header, compile.source, compile.unit = header, source, objects / "unit.o"
    return compile


def test_an_object_is_reused_until_what_it_was_made_from_changes(compiler):
    assert compiler() and not compiler()
    compiler.touch(compiler.header, compiler.unit.stat().st_mtime + 10)
    assert compiler()


def test_an_object_of_other_flags_is_not_reused(compiler, monkeypatch):
    assert compiler() and not compiler()
    monkeypatch.setattr(build, "NVCC_FLAGS", [*build.NVCC_FLAGS, "-DSOMETHING"])
    assert compiler() and not compiler()
    assert compiler(["-DWB200_CHECKS"]) and compiler()


def test_an_object_that_was_not_finished_is_not_reused(compiler, monkeypatch):
    assert compiler()
    with monkeypatch.context() as m:
        m.setattr(build, "NVCC_FLAGS", ["-DOTHER"])

        def fail(cmd):
            compiler.unit.write_text("half")
            raise RuntimeError("nvcc failed")

        m.setattr(build, "_run", fail)
        with pytest.raises(RuntimeError):
            compiler()
    assert compiler()  # of the flags of before: the object on disk is another's


def test_a_verbose_build_compiles_and_leaves_a_usable_object(compiler):
    assert compiler() and compiler(verbose=True) and not compiler()
