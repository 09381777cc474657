"""The routed int8 layer of examples/: plan, gathered and sorted expert products, the way back, and the
backward pass, together, against the unquantized layer in 64 bits.

Codes are steps of max / 127 of a row.  For normal rows of some hundred values the largest is 3 to 3.5
times the rms, so a side is off by 3.5 / 127 / sqrt(12) = 0.8 % of its rms and a product by 1.1 %.
The output passes two products, the second on an activation that carries the first's error (its gradient
and the product with `up` at most double it): 1.1 + 2 * 1.1 = 3.3 %, dweights as the output (of
|dout| |y|, whose product it is), dx four products at most: 6.6 %.  bf16 adds 0.4 % at each of some steps.  The bars are twice that.
"""
import os
import re
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BARS = {"out": 0.07, "dweights": 0.07, "dx": 0.14}


def test_layer(gpu):
    """The example in a process of its own (torch brings its own HIP runtime)."""
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "routed_int8_layer.py")], cwd=ROOT, text=True,
                       stdout=subprocess.PIPE, stderr=subprocess.PIPE, timeout=110)
    assert r.returncode == 0, r.stderr[-2000:]
    found = re.findall(r"(\d+) tokens, (\S+): (\w+) (\S+) off", r.stdout)
    assert len(found) == 3 * 2 * len(BARS), r.stdout
    for T, dtype, name, err in found:
        assert float(err) <= BARS[name], (T, dtype, name, err)
