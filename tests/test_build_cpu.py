"""Which changes make the library's objects be compiled anew (no compiler and no GPU needed)."""
import os

import pytest

from b200_sampler import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A tree of two sources; one.cu reaches deep.h through top.h alone.  Returns its folder and the list of compiled sources."""
    for name in ("csrc", "include", "obj"):
        (tmp_path / name).mkdir()
    files = {"csrc/one.cu": '#include "top.h"\n', "csrc/two.cu": '#include "deep.h"\n', "csrc/near.cuh": "",
             "include/top.h": '#include "deep.h"\n', "include/deep.h": "enum { A };\n", "build.py": "FLAGS = []\n"}
    for name, text in files.items():
        (tmp_path / name).write_text(text)
        os.utime(tmp_path / name, (1000, 1000))
    compiled = []

    def run(cmd, verbose=False):
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").write("object")
        os.utime(out, (2000, 2000))
        if "-c" in cmd:
            compiled.append(os.path.basename(cmd[-1]))
    monkeypatch.setattr(build, "CSRC", str(tmp_path / "csrc"))
    monkeypatch.setattr(build, "INCLUDE", str(tmp_path / "include"))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(build, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "__file__", str(tmp_path / "build.py"))
    monkeypatch.setattr(build, "build_histpack", lambda force=False: "")
    monkeypatch.setattr(build, "nvcc_path", lambda: "nvcc")
    monkeypatch.setattr(build, "_run", run)
    build.build()
    assert sorted(compiled) == ["one.cu", "two.cu"]
    compiled.clear()
    build.build()
    assert compiled == []
    return tmp_path, compiled


def test_a_changed_source_compiles_alone(tree):
    at, compiled = tree
    os.utime(at / "csrc/one.cu", (3000, 3000))
    build.build()
    assert compiled == ["one.cu"]


@pytest.mark.parametrize("name", ["include/deep.h", "include/top.h", "csrc/near.cuh"])
def test_a_changed_header_compiles_every_source(tree, name):
    """Also a source that names the header only through another one: constants must not differ between two objects."""
    at, compiled = tree
    os.utime(at / name, (3000, 3000))
    build.build()
    assert sorted(compiled) == ["one.cu", "two.cu"]


def test_changed_flags_compile_every_source(tree):
    at, compiled = tree
    os.utime(at / "build.py", (3000, 3000))
    build.build()
    assert sorted(compiled) == ["one.cu", "two.cu"]
