"""A process that Nsight tools run launches plainly instead of cooperatively (as CFB200_COOPERATIVE=0 does): the same results."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("env", [{"NV_NSIGHT_INJECTION_TRANSPORT_TYPE": "uds"}, {"CFB200_COOPERATIVE": "0"}, {"NV_NSIGHT_INJECTION_TRANSPORT_TYPE": "uds", "CFB200_COOPERATIVE": "1"}])
def test_layer_and_decoder_in_a_process_of_their_own(cuda_device, env):
    """The last: a variable of its own decides."""
    r = subprocess.run([sys.executable, "-c", "import __graft_entry__ as g; g.smoke()"], capture_output=True, text=True, timeout=300, cwd=ROOT, env=os.environ | env)
    assert r.returncode == 0 and "== oracle" in r.stdout, r.stdout + r.stderr
