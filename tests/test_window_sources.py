"""What the source of attention's windowed forward kernel promises and no run can show, as tests/test_kernel_sources.py has it of the
others: a wait that runs out ends lane by lane, but instructions of whole warps stand behind it."""
import os
import re

from tests.test_kernel_sources import CSRC, _blocks_around

FILE = os.path.join(CSRC, "rmn_attention_window.cu")


def _text():
    with open(FILE) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _span(text, at):
    """From a place in front of a bracket to the bracket's end."""
    depth, i = 0, text.index("(", at)
    for j in range(i, len(text)):
        depth += {"(": 1, ")": -1}.get(text[j], 0)
        if depth == 0:
            return at, j
    raise AssertionError(text[at:at + 80])


def test_only_one_lane_waits_alone():
    text = _text()
    fetch = _span(text, text.index("hand_out(a, tail, numbers"))
    calls = [m.start() for m in re.finditer(r"\b(?:mbar|lane)_wait\(", text)]
    assert calls
    for at in calls:
        after_time = any(re.search(r"if \(timed_out && lane == 0\)", head) for head in _blocks_around(text, at))
        assert fetch[0] < at < fetch[1] or after_time, text[at:at + 80]
    # who calls what was handed to hand_out: one lane, and all hear how it went
    body = text[text.index("void hand_out("):text.index("struct Shape")]
    assert len(re.findall(r"\bfetch\(", body)) == 1
    assert re.search(r"if \(lane == 0\) ok = fetch\(item\);\s*timed_out = __any_sync\(0xffffffffu, !ok\);", body)


def test_a_wait_that_ran_out_is_heard():
    """Every warp_wait's answer is looked at."""
    text = _text()
    calls = [m.start() for m in re.finditer(r"\bwarp_wait\(", text)]
    assert len(calls) >= 5
    for at in calls:
        assert re.search(r"if \((?:!timed_out && )?!$", text[:at]), text[at - 40:at + 60]
        assert "timed_out = true" in text[at:at + 120], text[at:at + 120]
