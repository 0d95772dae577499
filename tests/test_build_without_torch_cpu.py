"""The library serves hosts without Python or torch: what builds it needs nvcc alone."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = """
import sys
sys.modules["torch"] = None                  # what an import finds where there is none
from nestquant_b200 import build
build.OPS = sys.argv[1]
print(build.build())
from nestquant_b200 import capi
assert capi.lib().nq_build_arch() == 100
"""


@pytest.mark.parametrize("stale", [False, True])
def test_the_library_builds_without_torch(tmp_path, stale):
    """the torch module is left out, and the build says so"""
    from nestquant_b200 import build
    build.build()
    ops = tmp_path / "_torch_ops.so"
    if stale:
        ops.write_text("of an older source")
        os.utime(ops, (1, 1))
    r = subprocess.run([sys.executable, "-c", CODE, str(ops)], capture_output=True, text=True, cwd=ROOT, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.strip() == build.LIB and "torch" in r.stderr and "routing" in r.stderr
    assert not ops.exists()                  # an older module does not stay beside a newer library


def test_a_module_that_is_up_to_date_stays(tmp_path):
    ops = tmp_path / "_torch_ops.so"
    ops.write_text("of this source")
    code = CODE.replace("build.build()", "build._torch_ops(build.LIB, force=True)")
    r = subprocess.run([sys.executable, "-c", code, str(ops)], capture_output=True, text=True, cwd=ROOT, timeout=600)
    assert r.returncode == 0 and r.stdout.strip() == "None" and ops.exists(), r.stderr[-2000:]
