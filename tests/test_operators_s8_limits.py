"""What a grid holds where operands of an int8 product are not aligned.  No GPU."""
import os
import subprocess
import sys

import test_operators_host as host
from cldnn_amd import hip, ops_s8
from test_operators_host import AT, launches, runtime  # noqa: F401


def operands_that_are_not_aligned():
    """The largest product whose result's tiles of 64 x 64 a grid holds, and the next: refused where the operands are, before a launch."""
    e = hip.Engine()
    most = (1 << 24) - 1
    for m, n, fits in ((64 * most, 64, True), (64 * most + 1, 64, False), (64, 64 * most, True), (1, 64 * most + 1, False)):
        op = ops_s8.MatmulS8(e, ops_s8.matmul_s8_desc(m, n, 16))
        assert op._enqueue(op.h, *[AT] * 7) == 0
        for a, w in ((AT + 1, AT), (AT, AT + 8)):
            before = len(launches())
            status = op._enqueue(op.h, a, w, *[AT] * 5)
            found = launches()[before:]
            if fits:
                assert status == 0 and len(found) == 1 and found[0][2] == most
            else:
                assert status == -5 and not found and b"not aligned to 16 bytes: too large" in hip.lib().cldnn_hip_last_error()


@host.pytestmark
def test_operands_that_are_not_aligned(runtime):  # noqa: F811
    code = "import sys; sys.path[:0] = %r; import test_operators_s8_limits as t; t.operands_that_are_not_aligned()" % [host.ROOT, host.HERE]
    env = dict(os.environ, LD_PRELOAD=":".join(x for x in (runtime, os.environ.get("LD_PRELOAD")) if x))
    p = subprocess.run([sys.executable, "-c", code], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert p.returncode == 0, p.stdout
