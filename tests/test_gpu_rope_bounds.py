"""Every access of the query / key kernels stays inside its operand: a child process runs
tests/_rope_bounds_battery.py on the bounds-checked library, in which no check may fail,
and whose outputs are those of the release library."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from dslperfgap_amd import _lib
from dslperfgap_amd.build import DEBUG_LIB_PATH

sys.path.insert(0, str(Path(__file__).parent))
import _rope_bounds_battery  # noqa: E402

pytestmark = pytest.mark.gpu


def test_no_access_leaves_its_operand(tmp_path):
    if _lib.LIB_PATH.resolve() == DEBUG_LIB_PATH.resolve():
        pytest.skip("this session runs on the debug library itself (VBH_CHECK_BOUNDS run)")
    assert DEBUG_LIB_PATH.exists(), f"{DEBUG_LIB_PATH} is missing: run the build"
    print("[gpu] rope bounds: release battery", flush=True)
    want = _rope_bounds_battery.run()
    print("[gpu] rope bounds: debug battery in a child process", flush=True)
    out = tmp_path / "debug.pt"
    res = subprocess.run(
        [sys.executable, "-u", str(Path(__file__).parent / "_rope_bounds_battery.py"), str(out)],
        env=dict(os.environ, VBHIP_LIB=str(DEBUG_LIB_PATH)), capture_output=True, text=True,
        timeout=100)
    assert res.returncode == 0, res.stderr[-4000:]
    got = torch.load(out, weights_only=True)
    assert got["failed"] == 0, f"{got['failed']} failed bounds checks, first at {got['where']}"
    assert set(got["outs"]) == set(want)
    differ = [k for k in want if int(got["outs"][k]) != int(want[k])]
    assert not differ, differ[:5]
