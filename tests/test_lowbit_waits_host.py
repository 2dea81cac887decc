"""CPU check of the low-bit kernels' assembly: nothing reads LDS while a copy into it by the same wave may be under way.  A wait counts only where it is for all
loads (vmcnt(0)): a number of younger loads is the compiler's to change."""
import os
import re
import subprocess

import pytest

from physicedit_amd import build

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def early_reads(lines):
    """-> lines that read LDS with a copy pending, on any path (depth first over the instructions, with whether a copy is pending)"""
    labels = {line[:-1]: k for k, line in enumerate(lines) if line.endswith(":")}
    seen, found, paths = set(), set(), [(0, False)]
    while paths:
        k, pending = paths.pop()
        while k < len(lines) and (k, pending) not in seen:
            seen.add((k, pending))
            op, _, rest = lines[k].partition(" ")
            if op.startswith(("global_load_lds", "buffer_load_lds")) or (op.startswith("buffer_load") and rest.endswith(" lds")):
                pending = True
            elif op == "s_waitcnt" and "vmcnt(0)" in rest:
                pending = False
            elif op.startswith("ds_read") and pending:
                found.add(k)
            elif op == "s_endpgm":
                break
            if op == "s_branch":
                k = labels[rest.strip()]
                continue
            if op.startswith("s_cbranch"):
                paths.append((labels[rest.strip()], pending))
            k += 1
    return [lines[k] for k in sorted(found)]


def test_the_check_itself():
    copy, read, loop = "global_load_lds_dwordx4 v1, s[0:1]", "ds_read_b128 v[0:3], v4", ".LBB0_1:"
    assert early_reads([copy, read, "s_endpgm"]) == [read]
    assert early_reads([copy, "s_waitcnt vmcnt(3)", read, "s_endpgm"]) == [read]
    assert early_reads([copy, "s_waitcnt vmcnt(0) lgkmcnt(0)", read, "s_endpgm"]) == []
    assert early_reads([loop, read, copy, "s_cbranch_scc1 .LBB0_1", "s_endpgm"]) == [read]
    assert early_reads([loop, "s_waitcnt vmcnt(0)", read, copy, "s_cbranch_scc1 .LBB0_1", "s_endpgm"]) == []


@pytest.mark.parametrize("source,kernels", [("w4.hip", 132), ("kv_e4m3.hip", 8)])
def test_copies_into_lds_are_waited_for(tmp_path, source, kernels):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    out = tmp_path / "a.s"
    subprocess.run([HIPCC, *build.FLAGS, *build.EXTRA_FLAGS.get(source, []), "--offload-device-only", "-S", "-o", str(out), os.path.join(build.CSRC, source)],
                   check=True, capture_output=True)
    text, n, copies = out.read_text(), 0, 0
    for m in re.finditer(r"\n(_ZN2pe\w+):", text):
        body = text[m.start():text.index(".Lfunc_end", m.start())]
        lines = [x for x in (line.split(";")[0].strip() for line in body.splitlines()) if x and not (x.startswith(".") and not x.endswith(":"))]
        n, copies = n + 1, copies + any(x.startswith("global_load_lds") for x in lines)
        assert not early_reads(lines), m.group(1)
    assert n >= kernels and copies >= 4
