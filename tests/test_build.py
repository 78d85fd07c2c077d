"""What the build compiles again, with a compiler that only writes down what it was asked for."""
import stat
import sys

import pytest

from unet_amd import build as b


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of two files and a compiler that logs its command lines and creates the output."""
    csrc, lib = tmp_path / "csrc", tmp_path / "lib"
    csrc.mkdir()
    (tmp_path / "include").mkdir()
    for name in ("one.hip", "two.hip", "common.h"):
        (csrc / name).write_text("// nothing\n")
    (tmp_path / "include" / "unet_mi355.h").write_text("// nothing\n")
    log = tmp_path / "log"
    log.write_text("")
    cc = tmp_path / "cc"
    cc.write_text(f"#!{sys.executable}\nimport sys\na = sys.argv\nopen({str(log)!r}, 'a').write(' '.join(a[1:]) + '\\n')\nopen(a[a.index('-o') + 1], 'w').write('x')\n")
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    for name, value in (("HERE", tmp_path / "pkg"), ("CSRC", csrc), ("LIBDIR", lib), ("OBJDIR", lib / "obj"), ("SOURCES", ["one.hip", "two.hip"]),
                        ("FLAGS", ["-O3"]), ("_hipcc", lambda: str(cc))):
        monkeypatch.setattr(b, name, value)

    def compiled(**kw):
        log.write_text("")
        b.build(verbose=False, **kw)
        return sorted(line.split(" -c ")[1].split()[0].rsplit("/", 1)[1] for line in log.read_text().splitlines() if " -c " in line)

    return csrc, lib, compiled


def test_unchanged_sources_are_not_compiled_again(tree):
    csrc, lib, compiled = tree
    assert compiled() == ["one.hip", "two.hip"] and (lib / b.LIBNAME).exists()
    assert compiled() == []
    assert compiled(force=True) == ["one.hip", "two.hip"]


def test_other_flags_reach_objects_that_are_there(tree, monkeypatch):
    csrc, lib, compiled = tree
    compiled()
    monkeypatch.setattr(b, "FLAGS", ["-O3", "-packed-fp32-ops"])
    assert compiled() == ["one.hip", "two.hip"]
    assert compiled() == []


def test_objects_of_an_unknown_command_are_compiled_again(tree):
    csrc, lib, compiled = tree
    compiled()
    (lib / "obj" / "one.hip.o.cmd").unlink()
    assert compiled() == ["one.hip"]


def test_the_entry_point_compiles_everything(monkeypatch):
    import __graft_entry__ as entry

    asked = []
    monkeypatch.setattr(b, "build", lambda force=False, verbose=True: asked.append(force))
    entry.build()
    assert asked == [True]
