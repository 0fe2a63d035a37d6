"""mDeepFRI.batch brings torch in when it is imported: a process that imports the batch layer, builds a Predictor (the library's first HIP
call) and then an engine must not import torch on top of a running HIP runtime (see the comment at the import in mDeepFRI/batch.py)."""
import subprocess
import sys

from conftest import ROOT


def test_batch_layer_imports_torch_before_the_library_is_loaded():
    script = ("import sys; sys.path.insert(0, %r + '/metagenomic-deepfri_amd')\n"
              "import mDeepFRI.batch\n"
              "from mDeepFRI import _hip\n"
              "assert 'torch' in sys.modules and _hip._lib is None\n" % ROOT)
    out = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
