"""Importing the package maps none of its native code: host-only users need no build, and load none."""

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

CODE = """
import sys
from pathlib import Path
import nano_vllm_ascend_b200 as pkg
from nano_vllm_ascend_b200 import PagedKVCacheFp4, ops_fp4
own = str(Path(pkg.__file__).parent)
mapped = lambda: sorted({line.split()[-1] for line in open("/proc/self/maps") if own in line and ".so" in line})
assert not mapped(), mapped()
assert not any(name.endswith("_fp4_calls") for name in sys.modules)
ops_fp4.pool_shape(4, 16, 2)
PagedKVCacheFp4(1, 4, 16, 2, 128, "cpu")
assert not mapped(), mapped()
binding = ops_fp4._calls  # asked for: loaded (None where it is not built)
assert any("_fp4_calls" in m for m in mapped()) == (binding is not None)
assert ops_fp4._calls is binding
"""


def test_the_package_is_imported_without_native_code():
    res = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
