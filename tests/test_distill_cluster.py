"""Order of the distillation kernel's accesses to other blocks' shared memory, read from the source: a block sends nothing before all blocks
of the cluster have started and made their barriers, and none leaves before the last has sent; named barriers are arrived at and
waited for by the same number of threads."""
import os
import re

from tests.conftest import ROOT


def kernel():
    text = open(os.path.join(ROOT, "aeon_b200", "csrc", "distill.cu")).read()
    text = re.sub(r"//[^\n]*", "", text)
    at = text.index("distill_block_kernel(const distill_launch L)")
    depth, i = 1, text.index("{", at) + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
    return text[at:i]


def test_remote_stores_lie_between_waits():
    order = re.findall(r"\b(cluster_wait|cluster_send|barrier_init|cluster_arrive)\(", kernel())
    assert order[0] == "barrier_init" and order.index("cluster_arrive") < order.index("cluster_wait") < order.index("cluster_send")
    assert order[-2:] == ["cluster_arrive", "cluster_wait"]


def test_every_wait_is_bounded_or_the_hardware_s():
    text = open(os.path.join(ROOT, "aeon_b200", "csrc", "distill.cu")).read()
    wait = text[text.index("bool barrier_wait("):]
    assert re.search(r"for \(int i = 0; i < 1 << 20; \+\+i\)", wait[:600])
    assert "while (true)" not in text and "for (;;)" not in text


def test_named_barriers_have_one_count():
    body = kernel()
    assert set(re.findall(r"bar_(?:sync|arrive)\((?:\w+), (\w+)\)", body)) == {"ALL"}
    for name in ("SUMS", "RESULT", "WRITTEN"):
        assert len(re.findall(r"bar_\w+\(%s," % name, body)) >= 2, name
    assert "__syncthreads" not in body


def test_all_lanes_reach_the_warp_s_votes():
    """No vote or match of a whole warp stands behind a short-circuit or a choice in the same expression."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "aeon_b200", "csrc", "distill.cu")).read())
    for m in re.finditer(r"[^;{}]*__(?:match_any|any|shfl_xor|reduce_max)_sync\(0xffffffffu", text):
        before = m.group(0).rsplit("__", 1)[0]
        assert "&&" not in before and "||" not in before, m.group(0)[-120:]
