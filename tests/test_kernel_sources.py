"""What the kernels' sources promise and no run can show: an order whose violation would hang a GPU is looked for in the text."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "riemannengine_b200", "csrc")


def _kernels():
    """(file, kernel name, text from its head to the next kernel) of every __global__ function."""
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        starts = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
        for a, b in zip(starts, starts[1:]):
            yield name, re.search(r"\b(k_\w+)", text[a:b]).group(1), text[a:b]


@pytest.mark.parametrize("file,kernel,text", [pytest.param(*k, id=k[1]) for k in _kernels() if "tcgen05.alloc" in k[2]])
def test_the_next_kernel_is_released_behind_the_allocation_of_tensor_memory(file, kernel, text):
    """A block of the next kernel that came onto the SM first and took the tensor memory would hold it while it waits for
    this kernel, which waits for the memory."""
    alloc = text.index("tcgen05.alloc")
    barrier = text.index("__syncthreads()", alloc)
    for release in ("after_previous_kernel()", "release_next_kernel()", "griddepcontrol.launch_dependents"):
        for m in re.finditer(re.escape(release), text):
            assert m.start() > barrier, (file, kernel, release)


@pytest.mark.parametrize("file,kernel,text", [pytest.param(*k, id=k[1]) for k in _kernels() if "setmaxnreg" in k[2]])
def test_register_splits_are_executed_by_whole_warpgroups(file, kernel, text):
    """setmaxnreg is one instruction for the four warps of a warpgroup: the branch it opens has to hold for all or none."""
    with open(os.path.join(CSRC, file)) as f:
        constants = dict(re.findall(r"\b(k\w+) = (\d+)\b", f.read()))
    for m in re.finditer("setmaxnreg", text):
        branch = text[text.rindex("if (", 0, m.start()):m.start()]
        limit = re.match(r"if \(warp < (\w+)\) \{", branch)
        assert limit and int(constants[limit.group(1)]) % 4 == 0, (file, kernel, branch)


def _blocks_around(text, at):
    """What stands in front of every brace that is open at a place of a text, the innermost last."""
    heads, last = [], 0
    for m in re.finditer(r"[{};]", text[:at]):
        if m.group() == "{":
            heads.append(text[last:m.start()])
        elif m.group() == "}" and heads:
            heads.pop()
        last = m.end()
    return heads


@pytest.mark.parametrize("file", ["rmn_attention_fwd.cu", "rmn_attention_bwd.cu", "rmn_attention_rows.cu"])
def test_warps_leave_the_waits_of_attention_together(file):
    """A wait that runs out ends lane by lane. Behind it stand instructions of whole warps (tcgen05, elect, barriers), so either one lane
    alone waits, or the lanes vote: in warp_wait, or right behind the wait."""
    with open(os.path.join(CSRC, file)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    calls = list(re.finditer(r"\b(mbar_wait|lane_wait)\(", text))
    assert calls
    for m in calls:
        around = _blocks_around(text, m.start())
        one_lane = any(re.search(r"if \(lane == 0\b", head) for head in around)
        own = any("auto lane_wait = " in head for head in around)
        voted = re.search(r"__(all|any)_sync\(0xffffffffu, (here|timed_out)\)", text[m.start():m.start() + 200])
        assert one_lane or own or voted, text[m.start():m.start() + 80]


def _passes_early(slots, groups, loads=24):
    """Whether some order of events lets a wait by parity pass before its load has landed: `groups` of warps take the loads of a ring in
    turn, each load goes into its slot once the one before there has been released, and lands late. Every slot's barrier counts the
    landings; a wait for its n-th passes when the count is n + 1, or any other number of that parity."""
    done = [0] * groups  # loads that a group is through with

    def landed_first(late):  # all that may land without `late` does, then every group goes as far as it can
        landed, released = set(), set()
        for _ in range(loads * 2):
            for i in range(loads):
                if i != late and (i < slots or i - slots in released):
                    landed.add(i)
            for g in range(groups):
                i = g + done[g] * groups
                if i >= loads:
                    continue
                count = sum(1 for j in landed if j % slots == i % slots and j <= i)
                if (count - (i // slots + 1)) % 2 == 0:  # the wait passes
                    if i not in landed:
                        return True
                    released.add(i)
                    done[g] += 1
        return False

    for late in range(loads):
        done[:] = [0] * groups
        if landed_first(late):
            return True
    return False


def test_rings_are_waited_for_phase_by_phase():
    """Warps that take a ring's slots in turn skip phases of its barriers unless the turns divide the slots; a wait by parity then passes
    for a load that has not landed. The kernel of few query rows has one group of warps that waits for every load."""
    assert _passes_early(3, 2) and not any(_passes_early(n, 1) for n in (2, 3, 6)) and not _passes_early(4, 2)
    with open(os.path.join(CSRC, "rmn_attention_rows.cu")) as f:
        text = f.read()
    loops = re.findall(r"for \(int t64 = ([^;]*); t64 < last_tile; ([^)]*)\)", text)
    assert loops and all(loop == ("first_tile", "++t64") for loop in loops)
    assert "mbar_init(&empty[i], WARPS)" in text
