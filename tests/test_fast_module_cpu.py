"""a11spec._fast, the layer operators' compiled module: what needs it, and how it is built."""
import os
import subprocess
import sys

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "a11-llm-optimizer_b200")


def _package_without_fast(tmp_path):
    """A copy of the package (links) that has neither a11spec._fast nor what builds it."""
    os.makedirs(tmp_path / "a11spec")
    for f in sorted(os.listdir(os.path.join(PKG, "a11spec"))):
        if f.endswith(".py") or f == "liba11spec.so":
            os.symlink(os.path.join(PKG, "a11spec", f), tmp_path / "a11spec" / f)
    return str(tmp_path)


def _python(code, path, **env):
    return subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path, **env}, capture_output=True,
                          text=True, timeout=300)


def test_package_works_without_the_module(tmp_path):
    """Importing the package and its other operators does not need it; the layer operators say what is missing."""
    r = _python("""
import torch, a11spec
import a11spec.decoder, a11spec.generate, a11spec.tree_model, a11spec.kv_pages
assert a11spec.ngram_bucket(3, 4, 10) >= 0
t = torch.zeros(4, 64, dtype=torch.bfloat16)
for call in (lambda: a11spec.add_rms_norm(t, t[0]), lambda: a11spec.linear(t, t), lambda: a11spec.chunk_attention(t, t, t, t, t)):
    try:
        call()
    except ImportError as e:
        assert "_fast" in str(e)
    else:
        raise SystemExit("no error")
""", _package_without_fast(tmp_path))
    assert r.returncode == 0, r.stderr


def test_module_is_loaded_on_the_first_call():
    r = _python("""
import sys, a11spec
from a11spec import _lib
assert "a11spec._fast" not in sys.modules
f = _lib.fast
assert _lib.fast is f and "a11spec._fast" in sys.modules
try:
    _lib.no_such_name
except AttributeError as e:
    assert "no_such_name" in str(e)
else:
    raise SystemExit("no error")
""", PKG)
    assert r.returncode == 0, r.stderr
