"""The host side of mDeepFRI.batch (packing, planning) with no torch, or one whose libraries do not load; what needs torch says why it is not there."""
import subprocess
import sys

import pytest

from conftest import ROOT

SCRIPT = """
import sys
sys.path[:0] = [%r, %r + '/metagenomic-deepfri_amd']
from mDeepFRI import batch
packed = batch.PackedProteins.pack(["ACDEF", "GHIKLMN"])
assert packed.B == 2
try:
    batch._torch()
except ImportError as e:
    assert type(e.__cause__).__name__ == %r and %r in str(e) and %r in str(e.__cause__), (e, e.__cause__)
else:
    raise SystemExit("torch was found")
"""


@pytest.mark.parametrize("error, text", [("OSError", "libsomething.so.1: cannot open shared object file"), ("ImportError", "a part of it is missing")])
def test_batch_planner_without_a_working_torch(tmp_path, error, text):
    (tmp_path / "torch.py").write_text("raise %s(%r)\n" % (error, text))
    out = subprocess.run([sys.executable, "-c", SCRIPT % (str(tmp_path), ROOT, error, text, text)], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr[-1500:]
