"""The order in which a row's workgroups of sample's last launch hand their results over, in the code that the
compiler makes of it (no GPU): a barrier waits for no store to memory, so every wave has to wait for its own
before the L2 is written back and the workgroup's ticket taken, or the last workgroup, on another XCD, reads what
was there before."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "swarmllm_amd", "csrc")
STORE = re.compile(r"\s+(global|flat)_(store|atomic)")
TICKET = re.compile(r"\s+(global|flat)_atomic_add\w* v\d+, .*offset:12 sc0")  # SampleState::ticket, its old value wanted


def assembly(tmp_path):
    """sample.hip as the Makefile builds it, as assembly of the device's code."""
    rule = subprocess.run(["make", "-n", "-W", "sample.hip", "_build/sample.o"], cwd=CSRC, capture_output=True, text=True,
                          check=True).stdout
    line = next(li for li in rule.splitlines() if "-c sample.hip" in li)
    words = shlex.split(line.split("2>&1")[0])
    out = str(tmp_path / "sample.s")
    words[words.index("-c")] = "-S"
    words[words.index("-o") + 1] = out
    subprocess.run(words + ["--cuda-device-only"], cwd=CSRC, check=True, capture_output=True)
    with open(out) as f:
        return f.read().splitlines()


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"), reason="no compiler")
def test_stores_are_written_back_before_the_ticket(tmp_path):
    kernels, name = {}, None
    for line in assembly(tmp_path):
        start = re.match(r"(_ZN\w*sample_finish_kernel\w*):", line)
        if start:
            name = start.group(1)
            kernels[name] = []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name:
            kernels[name].append(line)
    assert len(kernels) == 6  # three types, two alignments
    for name, lines in kernels.items():
        tickets = [i for i, line in enumerate(lines) if TICKET.match(line)]
        assert len(tickets) == 1, name
        barrier = max(i for i in range(tickets[0]) if "s_barrier" in lines[i])
        # back from the barrier to the wait, without a branch or a store between
        i = barrier - 1
        while not re.search(r"s_waitcnt.*vmcnt\(0\)", lines[i]):
            assert not STORE.match(lines[i]) and "branch" not in lines[i] and not lines[i].startswith(".LBB"), (name, lines[i])
            i -= 1
        # behind which the L2 is written back, and nothing else written, before the ticket is taken
        after = lines[barrier:tickets[0]]
        assert not any(STORE.match(line) for line in after), name
        back = [j for j, line in enumerate(after) if "buffer_wbl2 sc1" in line]
        assert back and any(re.search(r"s_waitcnt.*vmcnt\(0\)", line) for line in after[back[-1]:]), name
