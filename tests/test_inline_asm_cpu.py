"""Reads written as inline assembly: the compiler takes such a statement's outputs as written when it ends, and does not
count what is in flight.  So each statement that reads into registers has to wait for its own reads, in the code that is built."""
import re
import subprocess

import pytest

from masters_thesis_amd.ops import build as B

READ = re.compile(r"\b(ds_read|ds_load|global_load|buffer_load|flat_load|scratch_load|s_load)\w*")
WITH_READS = [s for s in B.sources() if re.search(r"asm volatile\((?:[^;]|;(?=[^;]*\"))*(?:ds_read|_load)", s.read_text()) or "ds_read_b64_tr_b16 %" in s.read_text()]


def statements(src):
    """Inline assembly of the device code: lists of instructions."""
    flags = B.kernel_flags(src, [f"--offload-arch={B.ARCH}", "-std=c++17", "-O3", "-munsafe-fp-atomics", f"-I{B.CSRC}"])
    r = subprocess.run([B._hipcc(), *flags, "--cuda-device-only", "-S", str(src), "-o", "-"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    found, at = [], None
    for line in r.stdout.splitlines():
        if "#ASMSTART" in line:
            at = []
        elif "#ASMEND" in line:
            found.append(at)
            at = None
        elif at is not None:
            at.append(line.strip())
    return found


def test_sources_with_reads_are_known():
    assert [s.stem for s in WITH_READS] == ["gemm"]


@pytest.mark.parametrize("src", WITH_READS, ids=lambda s: s.stem)
def test_reads_are_waited_for_in_their_statement(src):
    reads = 0
    for lines in statements(src):
        asked = [i for i, x in enumerate(lines) if READ.match(x)]
        if not asked:
            continue
        reads += len(asked)
        waits = [i for i, x in enumerate(lines) if x.startswith("s_waitcnt") and ("lgkmcnt(0)" if lines[asked[0]].startswith(("ds_", "s_")) else "vmcnt(0)") in x]
        assert waits and waits[-1] > asked[-1], lines
        # no read's registers hold the address of a later one
        regs = lambda x: {n for a, b in re.findall(r"\bv\[?(\d+)(?::(\d+))?", x) for n in range(int(a), int(b or a) + 1)}  # noqa: E731
        for k, i in enumerate(asked):
            out, _, rest = lines[i].partition(",")
            for j in asked[k + 1:]:
                assert not regs(out) & regs(lines[j].partition(",")[2].split("offset")[0]), lines
    assert reads
