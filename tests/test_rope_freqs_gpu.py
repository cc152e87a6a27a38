"""The C++ mirror's rotary frequencies: the defaults of Python's rope_freqs."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_cpp_defaults(gpu):
    exe, src = (os.path.join(HERE, "cpp", "rope_freqs_test" + x) for x in ("", ".cpp"))
    if not os.path.exists(exe) or os.path.getmtime(exe) < os.path.getmtime(src):
        subprocess.run(["bash", os.path.join(HERE, "cpp", "build.sh")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    print(r.stdout, r.stderr, flush=True)
    assert r.returncode == 0, r.stdout + r.stderr
