"""The order of barriers in the paged-cache kernels, read from their source: what a
kernel must pass before it touches another CTA's memory, and which barriers have no
limit.  A wrong order shows on a GPU only as a rare fault or a hang, so it is looked
for here instead of being run."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "not-cute-zig_b200", "csrc")


def body(path, name):
    """The text of function `name` between its outer braces, without comments."""
    with open(os.path.join(CSRC, path)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    start = text.index("{", re.search(r"\b%s\(const DecodeParams &?p\)|\b%s\(const PlanParams p\)" % (name, name), text).end())
    depth, i = 0, start
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            return text[start:i]


def test_cluster_memory_is_touched_after_a_cluster_barrier():
    """A CTA's shared memory may be reached by the others of its cluster only once it has
    started, which a cluster barrier alone says."""
    for path, name in (("paged_sm100.cuh", "paged_plan"), ("paged_sm100.cuh", "decode_body")):
        text = body(path, name)
        touch = re.search(r"\bcluster_(store|load)\w*\(", text)
        passed = re.search(r"\bcluster_(wait|sync_all)\(\)", text)
        assert touch and passed and passed.start() < touch.start(), name
        if passed.group(1) == "wait":
            assert re.search(r"\bcluster_arrive\(\)", text[:passed.start()]), name


def test_softmax_warps_leave_a_hardware_barrier_together():
    """bar.sync has no limit, so no softmax warp of paged_decode_wide may stand at one that
    another has left: they enter the merge by a vote that all four take part in, also those
    that stopped at a limited wait, and nothing between the vote and the end of the item leaves."""
    text = body("paged_wide_sm100.cuh", "paged_decode_wide")
    softmax = text[text.index("const int copy = warp"):]
    assert "softmax_sync" not in text[:len(text) - len(softmax)]
    enter = softmax.index("if (!softmax_together(true)) break;")
    last = softmax.rindex("softmax_sync();")
    assert enter < softmax.index("softmax_sync();")
    assert not re.search(r"\bbreak\b|\breturn\b|paged_wait", softmax[enter + len("if (!softmax_together(true)) break;"):last])
    # every other way out of the loop says so first, and votes once behind it
    exits = [m.start() for m in re.finditer(r"\bbreak;", softmax)]
    assert len(exits) == 4
    for at in exits:
        assert softmax[:at].endswith(("if (gave_up) ", "if (!softmax_together(true)) "))
    assert re.search(r"if \(kCopies > 1 && gave_up\) softmax_together\(false\);", softmax[max(last, exits[-1]):])
