"""CPU: the largest score of a row (matcoredsl_b200/csrc/common.cuh, max_of), compiled for the host: it
is found at every place, and nothing behind the row is read."""
import subprocess

from tests.native_util import compile_native


def test_max_of(tmp_path):
    r = subprocess.run([compile_native("max_of", tmp_path)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout)  # below 0: ended by a signal
