"""When the torch binding of the device operators is built, and when not."""
import importlib.util
import os
import subprocess
import sys
import types

import pytest

from poorgrad_b200 import build


@pytest.fixture
def compiler(monkeypatch, tmp_path):
    """Builds into tmp_path by a compiler that only writes its output; its calls."""
    calls = []

    def run(cmd, **_):
        calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_operators.so"))
    monkeypatch.setattr(build, "BINDING_STAMP", str(tmp_path / "_operators.stamp"))
    monkeypatch.setattr(build, "subprocess", types.SimpleNamespace(run=run))
    return calls


def test_without_torch_the_library_is_built_alone(compiler, monkeypatch):
    monkeypatch.setattr(build, "build_library", lambda force: "library")
    find = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.build_binding() is None
    assert build.build() == "library"
    assert compiler == [] and not os.path.exists(build.BINDING)


def test_another_torch_gets_another_binding(compiler, monkeypatch):
    assert build.build_binding() == build.BINDING
    assert build.build_binding() == build.BINDING and len(compiler) == 1
    version = build.importlib.metadata.version
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: version(name) + ".other")
    build.build_binding()
    build.build_binding()
    assert len(compiler) == 2
    monkeypatch.undo()


def test_an_unmarked_binding_is_built_again(compiler):
    build.build_binding()
    os.remove(build.BINDING_STAMP)
    build.build_binding()
    assert len(compiler) == 2
    build.build_binding(force=True)
    assert len(compiler) == 3


def test_a_checkout_without_torch_imports_the_rest():
    """The package and its library load where torch cannot be imported; only the operators ask for it."""
    code = ("import sys; sys.modules['torch'] = None; sys.path[:0] = [%r]\n"
            "import poorgrad_b200\n"
            "from poorgrad_b200 import abi\n"
            "abi.load_library()\n"
            "try:\n    import poorgrad_b200.operators\n"
            "except ImportError:\n    print('no operators')\n") % build.ROOT
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.split() == ["no", "operators"], out.stderr[-2000:]
