"""The query / key operators on the bounds-checked library, in a child process: no check
fails, and fp32 and bf16 outputs are those of the release library, value by value."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from dslperfgap_amd import _lib
from dslperfgap_amd.build import DEBUG_LIB_PATH

sys.path.insert(0, str(Path(__file__).parent))
import _rope_order_battery  # noqa: E402

pytestmark = pytest.mark.gpu


def test_checksums_see_values_in_each_others_places():
    t = torch.arange(40, dtype=torch.float32, device="cuda:0")
    want = _rope_order_battery.checksums(t)
    for i, j in ((0, 1), (7, 23), (38, 39)):
        other = t.clone()
        other[[i, j]] = t[[j, i]]
        assert all(a != b for a, b in zip(_rope_order_battery.checksums(other), want))


def test_values_lie_where_the_release_library_has_them(tmp_path):
    if _lib.LIB_PATH.resolve() == DEBUG_LIB_PATH.resolve():
        pytest.skip("this session runs on the debug library itself (VBH_CHECK_BOUNDS run)")
    assert DEBUG_LIB_PATH.exists(), f"{DEBUG_LIB_PATH} is missing: run the build"
    print("[gpu] rope order: release battery", flush=True)
    want = _rope_order_battery.run()
    print("[gpu] rope order: debug battery in a child process", flush=True)
    out = tmp_path / "debug.pt"
    res = subprocess.run(
        [sys.executable, "-u", str(Path(__file__).parent / "_rope_order_battery.py"), str(out)],
        env=dict(os.environ, VBHIP_LIB=str(DEBUG_LIB_PATH)), capture_output=True, text=True,
        timeout=100)
    assert res.returncode == 0, res.stderr[-4000:]
    got = torch.load(out, weights_only=True)
    assert got["failed"] == 0, f"{got['failed']} failed bounds checks, first at {got['where']}"
    differ = [k for k in want if got["outs"].get(k) != want[k]]
    assert set(got["outs"]) == set(want) and not differ, differ[:5]
