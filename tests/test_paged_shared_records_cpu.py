"""Where the attention over shared prefixes keeps the sums that its join puts together, on the host."""
import os
import subprocess

from yalm_b200 import _lib


def test_places_of_records_against_wide_arithmetic(tmp_path):
    here, csrc = os.path.dirname(os.path.abspath(__file__)), os.path.join(os.path.dirname(_lib.__file__), "csrc")
    exe = str(tmp_path / "records")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I" + csrc, "-o", exe,
                    os.path.join(here, "paged_shared_records_check.cpp")], check=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
