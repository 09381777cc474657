"""What importing the package needs: libtiermm.so, and nothing that only the newer entry points use
(no GPU needed)."""
import os
import re
import shutil
import subprocess
import sys

import tier_amd

HERE = os.path.dirname(os.path.abspath(tier_amd.__file__))

CALLS = """
import tier_amd as t
A, L = 4096, t.lib()
for call, args in ((t.moe_plan, (A, -1, 2, 8, A, A, A)), (t.moe_sort, (A, 0, 15, A, A, A, 16, 4, 2, 16)),
                   (t.i8_quant, (None, 0, 300, A, 384, A, 2, 300)),
                   (t.i8_linear, (A, 0, 300, A, 384, A, None, A, 99, 20, 2, 20, 300))):
    try:
        call(*args)
    except t.TiermmError as e:
        print(call.__name__, e.code, t.last_error() in str(e))
t.i8_gemm(A, 384, A, A, 384, A, None, A, 0, 20, 0, 20, 300)
print(t.i8_row_bytes(129), t.q_row_bytes(t.Q4_K, 256))
"""


def _package(tmp_path, *libs):
    """A copy of the package's Python files with links to the named libraries."""
    d = tmp_path / "tier_amd"
    d.mkdir()
    for f in os.listdir(HERE):
        if f.endswith(".py"):
            shutil.copy(os.path.join(HERE, f), d)
    for f in libs:
        os.symlink(os.path.join(HERE, f), d / f)
    return d


def _python(cwd, code):
    return subprocess.run([sys.executable, "-c", code], cwd=cwd, text=True, stdout=subprocess.PIPE,
                          stderr=subprocess.PIPE, timeout=100)


def test_without_call_module(tmp_path):
    """No _call.so (no CPython headers where the library was built): every entry point answers as with it."""
    _package(tmp_path, "libtiermm.so")
    without = _python(tmp_path, CALLS)
    assert without.returncode == 0, without.stderr
    assert without.stdout.splitlines() == ["moe_plan 2 True", "moe_sort 2 True", "i8_quant 2 True", "i8_linear 1 True",
                                           "256 144"]
    other = tmp_path / "with"
    other.mkdir()
    _package(other, "libtiermm.so", "_call.so")
    assert _python(other, CALLS).stdout == without.stdout


def test_import_errors_name_a_command_that_works(tmp_path):
    """No library, or one without the newer functions: an ImportError whose command does not import the
    package first."""
    d = _package(tmp_path)
    for how in ("none", "older"):
        if how == "older":
            (d / "empty.c").write_text("int tiermm_nothing(void) { return 0; }\n")
            subprocess.run(["gcc", "-shared", "-fPIC", "-o", d / "libtiermm.so", d / "empty.c"], check=True)
        r = _python(tmp_path, "import tier_amd")
        assert r.returncode and "ImportError" in r.stderr.splitlines()[-1], r.stderr
        path = re.search(r"run `python (\S+)`", r.stderr)[1]
        assert os.path.samefile(path, d / "build.py")
        # as `python path` runs it, up to the build itself
        r = _python(tmp_path, f"import runpy; b = runpy.run_path({path!r}); print(callable(b['build']))")
        assert r.stdout == "True\n", r.stderr


def test_build_without_python_headers(tmp_path, monkeypatch):
    """build() without CPython's headers leaves out _call.so, an older one too, and builds the rest."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("build_copy", os.path.join(HERE, "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    for name in ("OUT_DIR", "LIB", "PROBE_LIB", "CALL_LIB"):
        monkeypatch.setattr(b, name, str(tmp_path / name))
    (tmp_path / "CALL_LIB").write_text("older")
    made = []

    def run(cmd):
        made.append(cmd[cmd.index("-o") + 1])
        open(made[-1], "w").close()
        return ""

    monkeypatch.setattr(b, "_run", run)
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert b.build() == b.LIB
    assert os.path.exists(b.LIB) and os.path.exists(b.PROBE_LIB) and not os.path.exists(b.CALL_LIB)
    open(tmp_path / "Python.h", "w").close()
    b.build()
    assert os.path.exists(b.CALL_LIB)
