"""Host side of the operators beside the softmax at the edges of what they accept."""
import os
import subprocess

import causal_softmax as cs

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_of_a_group_up_to_the_largest_matrix(tmp_path):
    """The kernels' own cursor, compiled as C++: a signed one passes 2^31 - 1 and never ends."""
    exe = str(tmp_path / "turns_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(cs.PKG_DIR, "csrc"), "-o", exe, os.path.join(ROOT, "tests", "turns_check.cpp")],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr
