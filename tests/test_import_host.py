"""The package imports with a torch that was built without CUDA: scenes, readers and settings need no device."""
import os
import subprocess
import sys

import pytest

pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_import_with_a_torch_without_cuda():
    code = ("import torch; del torch._C._cuda_getCurrentRawStream\n"
            "import ds_splat_b200 as ds, ds_splat_b200.scenes, ds_splat_b200.scene_io\n"
            "try: ds.gated_recurrence(torch.zeros(1, 2, 4), torch.zeros(1, 2, 4))\n"
            "except RuntimeError as e: assert 'CUDA tensor' in str(e)\n"
            "else: raise AssertionError('not refused')")
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
