"""CPU tests of the library's build cache: an object is reused only if it is whole and what made it is
unchanged (a fake compiler; nothing is compiled)."""
import subprocess
from pathlib import Path

import pytest

from ffn_optim_b200 import build


class FakeCompiler:
    """Writes the source's text as the object; `kill` dies half way through, as an interrupted compiler."""

    def __init__(self):
        self.compiled, self.version, self.kill = [], "release 1.0", False

    def __call__(self, cmd, **kwargs):
        if "--version" in cmd:
            return subprocess.CompletedProcess(cmd, 0, self.version, "")
        out, text = Path(cmd[cmd.index("-o") + 1]), Path(cmd[-1]).read_text()
        self.compiled.append(Path(cmd[-1]).name)
        out.write_text(text[:len(text) // 2] if self.kill else text)
        if self.kill:
            raise KeyboardInterrupt
        return subprocess.CompletedProcess(cmd, 0, "", "")


@pytest.fixture
def tree(tmp_path, monkeypatch):
    fake = FakeCompiler()
    monkeypatch.setattr(build.subprocess, "run", fake)
    monkeypatch.setattr(build, "nvcc", lambda: "nvcc")
    monkeypatch.setattr(build, "LIBDIR", tmp_path / "_lib")
    (tmp_path / "_lib").mkdir()
    source = tmp_path / "a.cu"
    source.write_text('#include "a.cuh"\nint one = 1;\n')
    (tmp_path / "a.cuh").write_text("int zero;\n")
    return fake, source


def compile_(source):
    return build._compile(source, False, False).read_text()


def test_objects_are_compiled_again_when_what_makes_them_changes(tree, monkeypatch):
    fake, source = tree
    compile_(source)
    compile_(source)
    assert len(fake.compiled) == 1
    source.with_suffix(".cuh").write_text("int zero = 0;\n")
    compile_(source)
    assert len(fake.compiled) == 2
    fake.version = "release 2.0"
    compile_(source)
    assert len(fake.compiled) == 3
    before = build.source_digest()
    monkeypatch.setattr(build, "FLAGS", [*build.FLAGS, "-DMORE"])
    compile_(source)
    assert len(fake.compiled) == 4 and build.source_digest() != before


def test_an_interrupted_compilation_leaves_no_object_behind(tree):
    fake, source = tree
    first = source.read_text()
    assert compile_(source) == first
    source.write_text(first + "int two = 2;\n")
    fake.kill = True
    with pytest.raises(KeyboardInterrupt):
        compile_(source)
    fake.kill = False
    source.write_text(first)
    assert compile_(source) == first
