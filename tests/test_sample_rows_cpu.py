"""What of the sampler for rows of logits (yb_sample_rows_dev) can be shown without a GPU."""
import os
import re

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
