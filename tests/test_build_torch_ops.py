"""When the autograd nodes' library is built again: a newer source, another torch or Python
than the one it was built for, or a build that did not end."""

import os
import subprocess
import types

import pytest

from flash_hog_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    monkeypatch.setattr(build, "TORCH_OPS_LIB", str(tmp_path / "_torch_ops.so"))
    monkeypatch.setattr(build, "BUILD_DIR", str(tmp_path / "_build"))
    source = tmp_path / "torch_ops.cpp"
    source.write_text("// nodes")
    os.utime(source, (1000, 1000))
    monkeypatch.setattr(build, "TORCH_OPS_SOURCE", str(source))
    state = types.SimpleNamespace(runs=0, rc=0, source=source)

    def run(cmd, **_):
        state.runs += 1
        if state.rc == 0:
            with open(cmd[cmd.index("-o") + 1], "w") as f:
                f.write("library")
        return subprocess.CompletedProcess(cmd, state.rc, "", "no such file")

    monkeypatch.setattr(build.subprocess, "run", run)
    return state


def _builds(tree):
    before = tree.runs
    build.build_torch_ops()
    assert os.path.exists(build.TORCH_OPS_LIB)
    return tree.runs - before


def test_built_once(tree):
    assert [_builds(tree) for _ in range(3)] == [1, 0, 0]


def test_a_newer_source_builds_again(tree):
    _builds(tree)
    late = os.path.getmtime(build.TORCH_OPS_LIB) + 10
    os.utime(tree.source, (late, late))
    assert _builds(tree) == 1


@pytest.mark.parametrize("what", ["torch", "python"])
def test_another_torch_or_python_builds_again(tree, monkeypatch, what):
    _builds(tree)
    with monkeypatch.context() as m:
        if what == "torch":
            real = build.importlib.metadata.version
            m.setattr(build.importlib.metadata, "version", lambda n: "99.0" if n == "torch" else real(n))
        else:
            m.setattr(build.sys, "version", "3.99.0")
        assert [_builds(tree) for _ in range(2)] == [1, 0]
    assert _builds(tree) == 1  # and back


def test_a_library_of_unknown_origin_is_built_again(tree):
    with open(build.TORCH_OPS_LIB, "w") as f:
        f.write("from elsewhere")
    assert _builds(tree) == 1


def test_a_failed_build_raises_and_is_not_taken_for_done(tree):
    _builds(tree)
    late = os.path.getmtime(build.TORCH_OPS_LIB) + 10
    os.utime(tree.source, (late, late))
    tree.rc = 1
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no such file"):
            build.build_torch_ops()
    tree.rc = 0
    os.utime(tree.source, (1000, 1000))
    assert _builds(tree) == 1
