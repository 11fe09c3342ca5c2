"""a11spec._fast, the layer operators' compiled module: what needs it, and how it is built."""
import os
import subprocess
import sys

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "a11-llm-optimizer_b200")


def _package_without_fast(tmp_path):
    """A copy of the package (links) that has neither a11spec._fast nor what builds it."""
    os.makedirs(tmp_path / "a11spec", exist_ok=True)
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


# --------------------------------------------------------------------------- the build
def _tree_with_compiler(tmp_path):
    """The package with its sources (links), no built module, and on PATH a g++ that takes
    its time, logs its runs and puts out the module that the real one made."""
    path = _package_without_fast(tmp_path / "pkg")
    os.symlink(os.path.join(PKG, "build.py"), os.path.join(path, "build.py"))
    os.symlink(os.path.join(PKG, "cpp"), os.path.join(path, "cpp"))
    os.symlink(os.path.join(os.path.dirname(PKG), "include"), tmp_path / "include")
    os.makedirs(tmp_path / "bin")
    gxx = tmp_path / "bin" / "g++"
    gxx.write_text("""#!/bin/sh
echo run >> "$LOG"
while [ "$1" != -o ]; do shift; done
head -c 1000 "$MODULE" > "$2"
sleep 2
cat "$MODULE" > "$2"
chmod +x "$2"
""")
    gxx.chmod(0o755)
    import a11spec._lib as lib
    env = dict(LOG=str(tmp_path / "log"), MODULE=sys.modules["a11spec._fast"].__file__ if lib.fast else "",
               PATH=str(tmp_path / "bin") + os.pathsep + os.environ["PATH"], PYTHONPATH=path)
    return path, env


USE = "import torch, a11spec; from a11spec import _lib; assert _lib.fast.row_stride(torch.zeros(2, 8), 8) == 8"


def test_a_module_of_another_build_is_not_loaded(tmp_path):
    path, env = _tree_with_compiler(tmp_path)
    for name in ("_fast.so", "_fast-0123456789-0123456789.so"):  # of another torch, or of other sources
        with open(os.path.join(path, "a11spec", name), "wb") as f:
            f.write(b"not this one")
    for _ in range(2):
        r = _python(USE, path, **{k: v for k, v in env.items() if k != "PYTHONPATH"})
        assert r.returncode == 0, r.stderr
    assert open(env["LOG"]).read() == "run\n"  # built once, found the second time


def test_the_name_follows_torch_and_the_sources(tmp_path):
    path, env = _tree_with_compiler(tmp_path)
    r = _python("""
import importlib.util, os, shutil, sys, torch
spec = importlib.util.spec_from_file_location("b", os.path.join(os.environ["TREE"], "build.py"))
b = importlib.util.module_from_spec(spec)
spec.loader.exec_module(b)
names = [b.fast_path()]
torch.__version__ += ".other"
names.append(b.fast_path())
copy = os.path.join(os.environ["TREE"], "changed.h")
shutil.copy(b.FAST_SOURCES[1], copy)
with open(copy, "a") as f:
    f.write("/* */")
b.FAST_SOURCES = (b.FAST_SOURCES[0], copy)
names.append(b.fast_path())
assert len(set(names)) == 3, names
""", path, TREE=path)
    assert r.returncode == 0, r.stderr


def test_processes_that_build_at_once(tmp_path):
    path, env = _tree_with_compiler(tmp_path)
    ranks = [subprocess.Popen([sys.executable, "-c", USE], env={**os.environ, **env}, stderr=subprocess.PIPE, text=True)
             for _ in range(3)]
    for r in ranks:
        err = r.communicate(timeout=300)[1]
        assert r.returncode == 0, err
    assert open(env["LOG"]).read() == "run\n"
    left = [f for f in os.listdir(os.path.join(path, "a11spec")) if "fast" in f]
    assert len(left) == 1, left


def test_missing_library_is_built_on_import(tmp_path):
    path, env = _tree_with_compiler(tmp_path)
    os.symlink(os.path.join(PKG, "csrc"), os.path.join(path, "csrc"))
    lib = os.path.join(path, "a11spec", "liba11spec.so")
    env.update(MODULE=os.path.realpath(lib), NVCC=str(tmp_path / "bin" / "g++"))
    os.unlink(lib)
    r = _python("import a11spec; a11spec.ngram_bucket(1, 2, 10)", path, **{k: v for k, v in env.items() if k != "PYTHONPATH"})
    assert r.returncode == 0, r.stderr
    assert open(env["LOG"]).read() == "run\n"


def test_processes_that_build_the_library_at_once(tmp_path):
    """The same for liba11spec.so, which the import builds where it is missing."""
    path, env = _tree_with_compiler(tmp_path)
    os.symlink(os.path.join(PKG, "csrc"), os.path.join(path, "csrc"))
    lib = os.path.join(path, "a11spec", "liba11spec.so")
    env.update(MODULE=os.path.realpath(lib), NVCC=str(tmp_path / "bin" / "g++"))
    os.unlink(lib)
    ranks = [subprocess.Popen([sys.executable, "-c", "import a11spec; a11spec.ngram_bucket(1, 2, 10)"], env={**os.environ, **env},
                              stderr=subprocess.PIPE, text=True) for _ in range(3)]
    for r in ranks:
        err = r.communicate(timeout=300)[1]
        assert r.returncode == 0, err
    assert open(env["LOG"]).read() == "run\n"
    assert [f for f in os.listdir(os.path.join(path, "a11spec")) if f.startswith((".", "liba11"))] == ["liba11spec.so"]


def test_a_folder_without_locks_still_builds(tmp_path):
    """Some network file systems refuse a lock on a folder."""
    path, env = _tree_with_compiler(tmp_path)
    r = _python("""
import fcntl
def refuse(*a):
    raise OSError(9, "Bad file descriptor")
fcntl.flock = refuse
""" + USE, path, **{k: v for k, v in env.items() if k != "PYTHONPATH"})
    assert r.returncode == 0, r.stderr
