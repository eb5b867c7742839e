"""What of the sampler for rows of logits (yb_sample_rows_dev) can be shown without a GPU."""
import os
import re
import subprocess

from yalm_b200 import _lib

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")


def _body(src, head):
    """The text between the braces that follow `head`."""
    at = src.index("{", src.index(head) + len(head))
    depth = 0
    for i in range(at, len(src)):
        depth += {"{": 1, "}": -1}.get(src[i], 0)
        if not depth:
            return src[at + 1: i]
    raise AssertionError(head)


def _written(text):
    """Words of a block's shared memory that a text writes."""
    words = set(re.findall(r"\bs\.(\w+)(?:\[[^\]]*\])?\s*(?:[-+*|&^]|<<|>>)?=(?!=)", text))
    return words | set(re.findall(r"atomic\w+\(&s\.(\w+)", text))


def test_what_other_blocks_read_stays_while_the_first_works_alone():
    """Between cluster_arrive and cluster_wait the first block finishes a row by itself, and nothing keeps the others from
    being late with what they read from it behind the last barrier: that must be words which it does not write there."""
    src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "sample_rows.cu")).read())
    alone = [_body(src, h) for h in ("u64 select(Shared& s", "Pair block_scan(Shared& s", "u64 block_sum(Shared& s",
                                     "void clear_bins(Shared& s", "auto take_list = [&]", "auto finish = [&](bool by_rank")]
    written = set().union(*(_written(t) for t in alone))
    assert {"told", "found", "mine", "warps", "sums", "count"} <= written  # (the patterns find what they should)
    parts = src.split("cluster_arrive();")
    assert len(parts) > 2
    for before, after in zip(parts, parts[1:]):
        assert re.match(r"\s*if \(rank == 0\) finish\([^;]*;\s*cluster_wait\(\);", after)
        behind = re.split(r"cluster_sync_all\(\);|\bpick\([^;]*;|\bfind\([^;]*;", before)[-1]
        read = set(re.findall(r"dsmem_ptr\(&s\.(\w+)", behind))
        assert read and not read & written, read & written
    # the row's limit, which all read behind a barrier after the first block's select: the next one must not reach it
    read = set(re.findall(r"(?:set_limit\(|at = )\*dsmem_ptr\(&s\.(\w+)", src))
    assert read and not read & written, read & written


SHARES = r"""
#include <cstdio>
#include <cstring>
#include <random>
#define __device__
#define __forceinline__ inline
typedef unsigned long long u64;
typedef unsigned __int128 wide;
static u64 __umul64hi(u64 a, u64 b) { return (u64)((wide)a * b >> 64); }
static unsigned __float_as_uint(float f) { unsigned u; memcpy(&u, &f, 4); return u; }
#include "share.inc"
int main() {
  std::mt19937_64 r(1);
  for (int i = 0; i < 3000000; ++i) {
    unsigned u = (unsigned)(r() % 0x3f800000u);                  // every number from 0 to below 1
    if (i % 3 == 0) u = (unsigned)(126 - r() % 126) << 23;       // powers of two
    if (i < 3000) u = (unsigned)i;                               // the smallest
    float x;
    memcpy(&x, &u, 4);
    u64 sum = 1 + (r() >> (1 + r() % 63));
    if (i % 5 == 0) sum = 1ull << (r() % 64);
    const unsigned e = u >> 23, d = 150 - (e ? e : 1);
    const wide p = (wide)(e ? (u & 0x7fffff) | 0x800000 : u) * sum;  // x * sum = p / 2^d
    u64 want = d >= 100 ? 1 : (u64)((p + (((wide)1 << d) - 1)) >> d);
    if (!want) want = 1;
    if (share_of(x, sum) != want || want > sum) return printf("%a of %llu: %llu, not %llu\n", x, sum, share_of(x, sum), want), 1;
  }
  const float odd[] = {-0.f, 0.f, -1.f, 1.f, 2.f, 1.f / 0.f, -1.f / 0.f, 0.f / 0.f};
  const u64 of[] = {1, 1, 1, 77, 77, 77, 1, 1};
  for (int i = 0; i < 8; ++i)
    if (share_of(odd[i], 77) != of[i]) return printf("%a\n", odd[i]), 1;
  puts("ok");
}
"""


def test_shares_of_sums_are_whole_numbers_rounded_up(tmp_path):
    """The kernel's own function, cut out of its source, against 128 bits."""
    src = open(os.path.join(CSRC, "sample_rows.cu")).read()
    head = "__device__ __forceinline__ u64 share_of(float x, u64 sum)"
    (tmp_path / "share.inc").write_text(head + " {" + _body(src, head) + "}\n")
    (tmp_path / "share.cpp").write_text(SHARES)
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(tmp_path / "share"), str(tmp_path / "share.cpp")], check=True, timeout=300)
    r = subprocess.run([str(tmp_path / "share")], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
