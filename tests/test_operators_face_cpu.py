"""The operators' entry points with what a caller may hand them by mistake:
configs that no call takes, tensors of another element type, calls from two
threads.  Without a GPU, like test_operators_cpu.py."""
import subprocess
import sys
from pathlib import Path

import pytest


@pytest.fixture(scope="module")
def L(pkg):
    import moe_b200.build as build
    import moe_b200.lib as lib
    build.build()
    lib.load()
    return lib


QUERY = """
import sys
sys.path.insert(0, sys.argv[1])
import conftest
conftest.load_pkg()
import moe_b200.lib as L
make, size = L.Engine.residual_norm_cfg, L.Engine.residual_norm_workspace_bytes
bad = [make(h, 16) for h in (0, 32769, 2 ** 32 - 255, 2 ** 32 - 1)]
bad += [make(64, 1 << 31), make(64, 16, gate=4), make(64, 16, y_type=2), make(64, 16, y_stride=63)]
print([size(c) for c in bad], size(None))
print(size(make(1, 16)), size(make(32768, 200)))
"""


def test_workspace_query_of_configs_that_no_call_takes(L):
    """The query comes before the call that refuses the config: it answers 0 and
    lives.  In a process of its own, which a division by zero would end."""
    r = subprocess.run([sys.executable, "-c", QUERY, str(Path(__file__).parent)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    assert r.stdout.splitlines() == [f"{[0] * 8} 0", f"{16 * 2 * 4} {148 * 2 * 32768 * 4}"]
