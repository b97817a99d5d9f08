"""Objects of the library are kept between builds as long as they were made from the text at hand."""
import subprocess

import pytest

from quintrit_b200 import build


@pytest.fixture
def source(tmp_path, monkeypatch):
    """One source of a build in a folder of its own; the compiler copies it to the object, or is stopped behind that."""
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    state = dict(path=tmp_path / "a.cu", runs=0, stop=False)

    def run(cmd, **kw):
        state["runs"] += 1
        (tmp_path / "a.cu.o").write_text(state["path"].read_text())
        if state["stop"]:
            raise KeyboardInterrupt
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    return state


def compile_it(source, text=None, **kw):
    if text is not None:
        source["path"].write_text(text)
    obj, _ = build._compile("a.cu", kw.get("force", False), False, [])
    return open(obj).read()


def test_an_object_is_used_again(source):
    assert compile_it(source, "one") == "one" and compile_it(source) == "one" and source["runs"] == 1
    assert compile_it(source, "two") == "two" and source["runs"] == 2
    assert compile_it(source, force=True) == "two" and source["runs"] == 3


def test_an_object_of_a_build_that_was_stopped_is_not(source):
    compile_it(source, "one")
    source["stop"] = True
    with pytest.raises(KeyboardInterrupt):
        compile_it(source, "two")
    source["stop"] = False
    assert compile_it(source, "one") == "one"
