"""The hand-over of the paged attention's query buffers (yb_paged_attention_dev, yb_paged_attention_shared_dev) in every order
of its warps' steps, on the host."""
import os
import re
import subprocess

from yalm_b200 import _lib

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")


def test_no_query_buffer_is_written_while_it_is_read(tmp_path):
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "buffers")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I" + CSRC, "-o", exe, os.path.join(here, "paged_query_buffers_check.cpp")],
                   check=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


def test_the_kernel_releases_what_it_has_read():
    """What the model above is of: a product warp arrives on the barrier of the buffer that it reads and on no other."""
    src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "paged_attn.cu")).read())
    assert "const int qb = query_buffer(two, p, buf);" in src
    assert re.findall(r"umma_commit_if\(e, &q_empty\[([^;]*)\]\);", src) == ["qb", "qb"]
    assert "if (query_releases(two) == 2) umma_commit_if(e, &q_empty[qb]);" in src
