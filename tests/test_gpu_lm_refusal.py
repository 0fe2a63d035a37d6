"""What becomes of an error that the one-launch LSTM's cooperative launch returns: a refusal (the grid cannot be resident now) falls back to the per-step form
and says so once, anything else reaches the caller.  The error comes from a function of the runtime's name that is loaded in front of it and launches nothing."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

STAND_IN = r"""
#include <stdlib.h>
struct dim3_ { unsigned x, y, z; };
int hipLaunchCooperativeKernel(const void *f, struct dim3_ g, struct dim3_ b, void **args, unsigned lds, void *stream) { return atoi(getenv("TEST_COOPERATIVE_ERROR")); }
"""

CHILD = r"""
import ctypes, os, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import numpy as np
from mdfri_testkit import synthetic
from mDeepFRI.batch import HotPathEngine, PackedProteins
from mDeepFRI.predict import Predictor
w = synthetic.glorot_gcn_weights(seed=3, n_terms=20, embed=256, gc_dims=(256,), fc_dim=256)
w.update(synthetic.glorot_lm_weights(seed=1000, hidden=64, embed=256))
rng = np.random.default_rng(11)
packed = PackedProteins.pack([synthetic.random_sequence(rng, n) for n in (1, 7, 33, 20)])
engine = HotPathEngine({"mf": Predictor("synthetic", weights=w)})
features = lambda: np.concatenate([np.asarray(f) for f in engine.lm_features(packed)])
os.environ["MDFRI_LM_PERSISTENT_MAX_B"] = "0"
want = features()
del os.environ["MDFRI_LM_PERSISTENT_MAX_B"]
for code in (720, 701, 401, 720):       # hipErrorCooperativeLaunchTooLarge, hipErrorLaunchOutOfResources, hipErrorIllegalState
    os.environ["TEST_COOPERATIVE_ERROR"] = str(code)
    print("refused", code, np.array_equal(features(), want), flush=True)
for code in (98, 719, 1):               # hipErrorInvalidDeviceFunction, hipErrorLaunchFailure, hipErrorInvalidValue
    os.environ["TEST_COOPERATIVE_ERROR"] = str(code)
    try:
        features()
        print("swallowed", code, flush=True)
    except RuntimeError as e:
        print("raised", code, "failed" in str(e), flush=True)
"""


def test_only_refusals_of_the_cooperative_launch_fall_back(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("needs gcc")
    (tmp_path / "stand_in.c").write_text(STAND_IN)
    subprocess.check_call(["gcc", "-shared", "-fPIC", str(tmp_path / "stand_in.c"), "-o", str(tmp_path / "stand_in.so")])
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "metagenomic-deepfri_amd")]))
    env.pop("MDFRI_LM_PERSISTENT_MAX_B", None)
    r = subprocess.run([sys.executable, "-c", CHILD, str(tmp_path / "stand_in.so")], env=env, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split("\n")[:7] == ["refused 720 True", "refused 701 True", "refused 401 True", "refused 720 True", "raised 98 True", "raised 719 True", "raised 1 True"], r.stdout
    assert r.stderr.count("launch refused (hipErrorCooperativeLaunchTooLarge)") == 1 and r.stderr.count("launch refused") == 1, r.stderr[-2000:]
