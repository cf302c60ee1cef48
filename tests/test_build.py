"""The build's own commands, with stand-ins for the compilers that write down how they were called (CPU only)."""
import os
import sys

import pytest

from htr_amd import build

# writes its arguments to a file of its own in $CALLS and makes the file that -o names
STAND_IN = """#!{python}
import os, sys, tempfile
fd, _ = tempfile.mkstemp(dir=os.environ["CALLS"])
os.write(fd, "\\n".join(sys.argv[1:]).encode())
os.close(fd)
with open(sys.argv[sys.argv.index("-o") + 1], "w") as f:
    f.write("made")
"""


@pytest.fixture
def calls(tmp_path, monkeypatch):
    """Runs the build with `extra`: the argument lists of its compile and link commands."""
    tool, kept = tmp_path / "tool", tmp_path / "calls"
    tool.write_text(STAND_IN.format(python=sys.executable))
    tool.chmod(0o755)
    kept.mkdir()
    monkeypatch.setenv("CALLS", str(kept))
    monkeypatch.setenv("HIPCC", str(tool))
    monkeypatch.setenv("CXX", str(tool))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "BINDING", str(tmp_path / "fast.so"))

    def run(extra=()):
        for f in kept.iterdir():
            f.unlink()
        assert build.build(extra=extra) == build.LIB and os.path.exists(build.LIB)
        told = [f.read_text().split("\n") for f in kept.iterdir()]
        hip = [t for t in told if build.BINDING not in t]
        return [t for t in hip if "-c" in t], [t for t in hip if "-c" not in t]
    return run


def test_extra_options_reach_the_linker_too(calls):
    compiles, links = calls(["--coverage", "-DX=1"])
    assert len(compiles) == len(build.SOURCES) and len(links) == 1
    for told in compiles + links:
        assert "--coverage" in told and "-DX=1" in told


def test_builds_at_once_have_objects_of_their_own(calls):
    objects = [{told[told.index("-o") + 1] for told in calls()[0]} for _ in range(2)]
    assert len(objects[0]) == len(objects[1]) == len(build.SOURCES)
    assert not objects[0] & objects[1]
    assert not any(os.path.exists(o) for o in objects[0] | objects[1])          # and leave none behind


def test_what_is_linked_is_what_was_compiled(calls):
    compiles, (link,) = calls()
    assert {told[told.index("-o") + 1] for told in compiles} == {a for a in link if a.endswith(".o")}
    assert link[link.index("-o") + 1] == build.LIB
    assert {told[told.index("-c") + 1] for told in compiles} == set(build.SOURCES)
