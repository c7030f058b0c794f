"""Loads that go straight to LDS are awaited before the barrier that hands their tile over: neither a barrier nor LDS reads
wait for them.  Checked on the gfx950 assembly of every source that has such loads, as it is built."""
import glob
import os
import re
import subprocess

import pytest

from memvanta_amd import build

SOURCES = [p for p in sorted(glob.glob(os.path.join(build.HERE, "csrc", "*.hip"))) if "load_lds" in open(p).read()]


def _unawaited(lines):
    """(loads to LDS, lines of barriers and ends that one can reach without a wait for all vector loads since) of a function's
    assembly, by a walk over its blocks until nothing changes."""
    blocks, at = [[]], {}
    for line in lines:
        label = re.match(r"(\S+):", line)
        if label:
            blocks.append([])
            at[label[1]] = len(blocks) - 1
        op = line.split(";")[0].split()
        if not line.startswith("\t") or not op or op[0].startswith("."):
            continue
        blocks[-1].append((op[0], line.split(";")[0].strip()))
        if op[0].startswith(("s_cbranch", "s_branch", "s_endpgm")):
            blocks.append([])
    loads, bad = 0, set()
    open_at = [False] * (len(blocks) + 1)  # a load may be under way when the block starts
    work = list(range(len(blocks)))
    for b in blocks:
        for op, text in b:
            assert op not in ("s_setpc_b64", "s_swappc_b64"), text  # no calls: the walk stays within the function
            loads += bool(re.match(r"(global|buffer)_load", op) and ("_lds_" in op or text.endswith(" lds")))
    while work:
        i = work.pop()
        pending, to = open_at[i], [i + 1] if i + 1 < len(blocks) else []
        for op, text in blocks[i]:
            if re.match(r"(global|buffer)_load", op) and ("_lds_" in op or text.endswith(" lds")):
                pending = True
            elif op == "s_waitcnt" and "vmcnt(0)" in text:
                pending = False
            elif op in ("s_barrier", "s_endpgm") and pending:
                bad.add((i, text))
            if op.startswith(("s_cbranch", "s_branch")):
                target = at[text.split()[1]]
                to = [target] if op == "s_branch" else to + [target]
            elif op == "s_endpgm":
                to = []
        for t in to:
            if pending and not open_at[t]:
                open_at[t] = True
                work.append(t)
    return loads, bad


def test_the_walk():
    """A loop whose head's barrier is awaited on the way in but not on the way back."""
    load, wait, barrier, end = "\tglobal_load_lds_dwordx4 v[2:3], off", "\ts_waitcnt vmcnt(0) lgkmcnt(0)", "\ts_barrier", "\ts_endpgm"
    back = "\ts_cbranch_scc1 .L0"
    assert _unawaited([load, wait, ".L0:", barrier, load, back, wait, end]) == (2, {(1, "s_barrier")})
    assert _unawaited([load, ".L0:", wait, barrier, load, back, wait, end]) == (2, set())
    assert _unawaited([load, "\ts_waitcnt lgkmcnt(0)", barrier, wait, end])[1]
    assert _unawaited(["\tbuffer_load_dwordx4 v1, s[4:7], s16 offen lds", end])[1]


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no compiler here")
@pytest.mark.parametrize("source", [os.path.basename(p) for p in SOURCES])
def test_sources(source, tmp_path):
    out = tmp_path / "a.s"
    flags = [f for f in build.HIP_FLAGS if f != "-shared"]
    subprocess.run([build.HIPCC, *flags, f"-I{build.ROOT}/include", f"-I{build.HERE}/csrc", "--cuda-device-only", "-S", "-o", str(out),
                    "-x", "hip", os.path.join(build.HERE, "csrc", source)], check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    text, kernels, bad = out.read_text(), 0, {}
    for body in re.split(r"\n(?=_Z\w+:)", text)[1:]:
        name = body.split(":")[0]
        loads, found = _unawaited(body.split(".Lfunc_end")[0].splitlines()[1:])
        kernels += loads > 0
        if found:
            bad[name] = len(found)
    assert kernels and not bad, bad


def test_there_are_sources():
    assert {"mvh_attn_shared.hip", "mvh_fp8.hip"} <= {os.path.basename(p) for p in SOURCES}
