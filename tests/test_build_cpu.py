"""When the native call path is rebuilt, and that a build replaces it whole (the compiler is a fake that writes its output file)."""
import os
import types

import pytest

from kb_nano_b200 import build


@pytest.fixture
def fake(monkeypatch, tmp_path):
    """The built files in a folder of their own; every compiler call is recorded and succeeds, or fails when told to."""
    state = types.SimpleNamespace(outputs=[], fail=False)

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        state.outputs.append(out)
        with open(out, "w") as f:
            f.write(f"build {len(state.outputs)}")
        return types.SimpleNamespace(returncode=int(state.fail), stdout="", stderr="no such header")

    monkeypatch.setattr(build, "CALLS_PATH", str(tmp_path / "_calls.so"))
    monkeypatch.setattr(build, "CALLS_STAMP", str(tmp_path / "build" / "_calls.stamp"), raising=False)
    monkeypatch.setattr(build, "_build_lib", lambda force, verbose: None)
    monkeypatch.setattr(build.subprocess, "run", run)
    return state


def content():
    with open(build.CALLS_PATH) as f:
        return f.read()


def test_built_once_and_again_after_another_torch_or_python(fake, monkeypatch):
    import torch
    build.build()
    build.build()
    assert len(fake.outputs) == 1 and content() == "build 1"
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    build.build()
    build.build()
    assert len(fake.outputs) == 2 and content() == "build 2"
    monkeypatch.setattr(build.sys, "version", "4.0")
    build.build()
    assert len(fake.outputs) == 3
    build.build(force=True)
    assert len(fake.outputs) == 4


def test_rebuilt_without_a_stamp_or_after_a_change_of_its_source(fake, monkeypatch, tmp_path):
    build.build()
    os.remove(build.CALLS_STAMP)
    build.build()
    assert len(fake.outputs) == 2
    src = tmp_path / "calls.cpp"
    src.write_text("")
    os.utime(src, (2**32, 2**32))
    monkeypatch.setattr(build, "CALLS_SRC", str(src))
    build.build()
    assert len(fake.outputs) == 3


def test_linked_beside_its_place_and_moved_there(fake, tmp_path):
    build.build()
    assert all(out != build.CALLS_PATH and os.path.dirname(out) == str(tmp_path) for out in fake.outputs)
    assert sorted(os.listdir(tmp_path)) == ["_calls.so", "build"]


def test_a_failed_build_leaves_the_old_file_and_is_tried_again(fake, tmp_path):
    build.build()
    fake.fail = True
    with pytest.raises(RuntimeError, match="no such header"):
        build.build(force=True)
    assert content() == "build 1" and sorted(os.listdir(tmp_path)) == ["_calls.so", "build"]
    fake.fail = False
    build.build()
    assert content() == "build 3"


def test_an_up_to_date_build_needs_no_compiler(fake, monkeypatch):
    build.build()

    def missing():
        raise RuntimeError("nvcc not found")

    monkeypatch.setattr(build, "_nvcc", missing)
    build.build()
    assert len(fake.outputs) == 1
