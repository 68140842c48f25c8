"""The build's second part, the Python binding: left out where torch is not
there."""
import subprocess
import sys
from pathlib import Path

BUILD = Path(__file__).resolve().parents[1] / "random-things_b200" / "build.py"


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
