"""The build's second part, the Python binding: left out where torch is not
there, built again for another torch or Python."""
import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

BUILD = Path(__file__).resolve().parents[1] / "random-things_b200" / "build.py"


@pytest.fixture
def build():
    spec = importlib.util.spec_from_file_location("xn_build", BUILD)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_the_library_alone_without_torch():
    """Callers of the C ABI need neither torch nor Python's headers: the command builds the library and says what it
    left out."""
    code = """if True:
        import importlib.util, sys
        spec = importlib.util.spec_from_file_location("xn_build", sys.argv[1])
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.build = lambda **kw: mod.LIB_PATH
        assert importlib.util.find_spec("torch") is None
        sys.exit(mod.main([]))
    """
    # -S: no site-packages.
    out = subprocess.run([sys.executable, "-I", "-S", "-c", code, str(BUILD)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr
    assert "libxn_fused.so" in out.stdout and "xn_torch.so" not in out.stdout
    assert "xn_torch.so" in out.stderr and "torch is not installed" in out.stderr


def test_the_binding_is_built_again_for_another_torch(build, monkeypatch, tmp_path):
    runs = []

    def run(cmd, check):
        runs.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("built")

    lib = tmp_path / "libxn_fused.so"
    lib.write_text("")
    monkeypatch.setattr(build, "LIB_PATH", lib)
    monkeypatch.setattr(build, "BINDING_PATH", tmp_path / "xn_torch.so")
    monkeypatch.setattr(build, "BUILD_DIR", tmp_path / "_build")
    monkeypatch.setattr(build.subprocess, "run", run)
    import torch

    build.build_binding()
    build.build_binding()
    assert len(runs) == 1
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    build.build_binding()
    build.build_binding()
    assert len(runs) == 2
    monkeypatch.setattr(build.sys, "version", "another Python")
    build.build_binding()
    build.build_binding()
    assert len(runs) == 3
    build.build_binding(force=True)
    assert len(runs) == 4
