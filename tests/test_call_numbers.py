"""None is a null address for the entry points called through tier_amd._call, and not a size, a stride
or a type: there it raises, as the ctypes functions do (no GPU needed)."""
import ctypes

import pytest

import tier_amd

A = 4096  # an address that no call follows
V = ctypes.c_void_p
# wrapper -> arguments that it refuses or answers before any device work
CALLS = {
    "moe_plan": (A, 0, 2, 8, None, A, A, None, 0),
    "moe_sort": (A, 0, 16, A, A, A, 16, 0, 2, 16),
    "moe_sort_grad": (A, 0, 16, A, A, 16, 0, 2, 16),
    "moe_unsort": (A, 0, 16, A, A, A, 16, 0, 2, 16),
    "moe_unsort_grad": (A, 0, 16, A, 16, A, A, A, A, 16, A, 0, 2, 16),
    "i8_quant": (A, 0, 300, A, 384, A, 0, 300),
    "i8_gemm": (A, 384, A, A, 384, A, None, A, 0, 20, 0, 20, 300),
    "i8_linear": (A, 0, 300, A, 384, A, None, A, 0, 20, 0, 20, 300, None, 0),
    "i8_gemm_grouped": (A, 384, A, None, 4, 2, A, 4, A, 384, A, A, 0, 20, 0, 20, 300),
}


def _call(name, args):
    """The status: 0, or the code of what it raised."""
    try:
        getattr(tier_amd, name)(*args)
    except tier_amd.TiermmError as e:
        return e.code
    return 0


@pytest.mark.parametrize("name", CALLS)
def test_none_is_no_number(name):
    args, types = CALLS[name], getattr(tier_amd.lib(), "tiermm_" + name).argtypes
    assert len(types) == len(args) + 1  # the stream
    assert _call(name, args) in (tier_amd.OK, tier_amd.EINVAL)
    for i, t in enumerate(types[:-1]):
        with_none = args[:i] + (None,) + args[i + 1:]
        if t is V:
            assert _call(name, with_none) in (tier_amd.OK, tier_amd.EINVAL)
        else:
            with pytest.raises((TypeError, ctypes.ArgumentError)):
                _call(name, with_none)


def test_call_module_of_older_sources(tmp_path):
    """A _call whose Call takes no third argument: the functions are called through ctypes."""
    import os
    import shutil
    import subprocess
    import sys
    here, d = os.path.dirname(os.path.abspath(tier_amd.__file__)), tmp_path / "tier_amd"
    d.mkdir()
    for f in os.listdir(here):
        if f.endswith(".py"):
            shutil.copy(os.path.join(here, f), d)
    os.symlink(os.path.join(here, "libtiermm.so"), d / "libtiermm.so")
    (d / "_call.py").write_text("class Call:\n    def __init__(self, address, n):\n        pass\n")
    code = ("import tier_amd as t\n"
            "try:\n    t.moe_plan(4096, -1, 2, 8, 4096, 4096, 4096)\n"
            "except t.TiermmError as e:\n    print(e.code)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, text=True, stdout=subprocess.PIPE,
                       stderr=subprocess.PIPE, timeout=100)
    assert r.stdout == "2\n", r.stderr
