"""When the Python binding of the block-scaled FP8 operators is built again (CPU)."""
import os
import subprocess

import pytest

from recavsr_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source, a header and the paths of a binding, and the compiler calls made."""
    for name in ("BINDING_SOURCE", "INCLUDE"):
        path = tmp_path / name
        path.write_text("")
        os.utime(path, (1, 1))
        monkeypatch.setattr(build, name, str(path))
    monkeypatch.setattr(build, "BINDING", str(tmp_path / "binding.so"))
    monkeypatch.setattr(build, "BINDING_KEY", str(tmp_path / "binding.key"), raising=False)
    calls = []

    def compiler(cmd, **_):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    return calls


def test_binding_is_kept_while_nothing_changes(tree):
    build._build_binding(False)
    build._build_binding(False)
    assert len(tree) == 1
    build._build_binding(True)
    assert len(tree) == 2


def test_binding_follows_its_sources(tree):
    build._build_binding(False)
    os.utime(build.INCLUDE, (2 ** 32, 2 ** 32))
    build._build_binding(False)
    assert len(tree) == 2


def test_binding_follows_torch(tree, monkeypatch):
    """Its object layouts are those of the torch headers it was compiled with."""
    build._build_binding(False)
    version = build.importlib.metadata.version
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: version(name) + ".post1")
    build._build_binding(False)
    assert len(tree) == 2


def test_binding_follows_python(tree, monkeypatch):
    build._build_binding(False)
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399")
    build._build_binding(False)
    assert len(tree) == 2


def test_binding_has_its_name_only_when_whole(tree):
    build._build_binding(False)
    assert build.BINDING not in tree[0]
    assert os.path.exists(build.BINDING) and os.listdir(os.path.dirname(build.BINDING)).count("binding.so.part") == 0


def test_failed_compiler_leaves_the_old_binding(tree, monkeypatch):
    build._build_binding(False)
    monkeypatch.setattr(build.subprocess, "run",
                        lambda cmd, **_: subprocess.CompletedProcess(cmd, 1, "", "no such header"))
    with pytest.raises(RuntimeError, match="no such header"):
        build._build_binding(True)
    assert open(build.BINDING).read() == "built"
