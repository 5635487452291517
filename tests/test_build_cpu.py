"""What the build recipe compiles, without running a compiler on the kernels."""
import os
import subprocess
import sys

import pytest

from cuda_fused_attention_b200 import build as recipe


class Recorded:
    """In place of subprocess.Popen: a compiler that succeeds and writes nothing."""
    commands = []

    def __init__(self, command, **_):
        Recorded.commands.append(command)
        self.returncode = 0

    def communicate(self):
        return "", ""


@pytest.fixture
def recorded(monkeypatch):
    Recorded.commands = []
    monkeypatch.setattr(subprocess, "Popen", Recorded)
    return Recorded


def _outputs(recorded):
    return [os.path.basename(command[command.index("-o") + 1]) for command in recorded.commands]


def test_libraries_are_built_without_torch(recorded, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)         # as if it were not installed
    assert recipe.build(force=True) == recipe.LIB_PATH
    assert _outputs(recorded) == ["libfa_sm100.so", "libfa_sm100_debug.so"]
    assert "binding of the paged-cache operators is not built" in capsys.readouterr().out


def test_everything_is_built_with_torch(recorded):
    recipe.build(force=True, verbose=False)
    outputs = _outputs(recorded)
    assert outputs[:2] == ["libfa_sm100.so", "libfa_sm100_debug.so"] and len(outputs) == 3 and outputs[2].startswith("_paged")


def test_a_missing_binding_asks_for_a_build_only_with_torch(monkeypatch, tmp_path):
    for name in ("LIB_PATH", "DEBUG_LIB_PATH"):
        path = tmp_path / name
        path.write_text("")
        os.utime(path, (2 ** 32, 2 ** 32))
        monkeypatch.setattr(recipe, name, str(path))
    monkeypatch.setattr(recipe, "BINDING_PATH", str(tmp_path / "absent"))
    assert recipe.needs_build()
    monkeypatch.setitem(sys.modules, "torch", None)
    assert not recipe.needs_build()


def test_the_binding_is_named_after_what_it_was_compiled_for(monkeypatch):
    """Another torch or Python looks for another file, and asks for a build."""
    torch = pytest.importorskip("torch")
    import importlib.metadata
    name = os.path.basename(recipe.BINDING_PATH)
    assert name == recipe.binding_name() and torch.__version__ in name and sys.implementation.cache_tag in name
    assert recipe.binding_command()[-1] == recipe.BINDING_PATH
    with monkeypatch.context() as other:
        other.setattr(importlib.metadata, "version", lambda package: "0.1")
        assert recipe.binding_name() != name
    with monkeypatch.context() as other:
        other.setattr(sys.implementation, "cache_tag", "cpython-0")
        assert recipe.binding_name() != name


def test_the_dense_forward_links_without_the_paged_sources(tmp_path):
    """A target that lists the dense forward's four sources alone (front end only: no GPU code is assembled)."""
    import ctypes
    dense = [os.path.join(recipe.CSRC, name) for name in ("fa_sm100.cu", "fa_sm100_host.cu", "fa_sm100_api.cu", "fa_sm100_static.cu")]
    output = str(tmp_path / "dense.so")
    done = subprocess.run([recipe.nvcc_path(), "-std=c++17", "-gencode", "arch=compute_100a,code=compute_100a", "-shared",
                           "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "-Xlinker", "--no-undefined",
                           "-I", os.path.join(recipe.ROOT, "include"), "-I", recipe.CSRC, *dense, "-o", output],
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]
    lib = ctypes.CDLL(output, mode=os.RTLD_NOW)
    assert lib.fa_sm100_supported(128) == 1 and not hasattr(lib, "fa_sm100_paged_plan")
