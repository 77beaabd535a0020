"""Properties of the serving operators' compiled gfx950 code (CPU only: hipcc cross-compiles).

The rules of the history kernels' code, for the same reasons: no vector
register goes to memory, no LDS read writes a register that an MFMA is still
to write, and m0 belongs to the LDS-DMA helpers.
"""

from __future__ import annotations

import os
import re
import subprocess

import pytest

from aws_training_study_amd import build_native
from test_device_code import _m0_misuse, _pending_destination_reads, _scratch_ops

KERNELS = re.compile(r"(attend_few|attend_many|token|cache_read|merge_few_ranges|merge_many_ranges)_kernel")


@pytest.fixture(scope="module")
def device_code(tmp_path_factory):
    out = tmp_path_factory.mktemp("devcode") / "serving.s"
    cmd = [build_native.hipcc(), f"--offload-arch={build_native.OFFLOAD_ARCH}", "-O3", "-std=c++17",
           f"-I{build_native.INCLUDE_DIR}", *build_native.DEVICE_FLAGS, "--cuda-device-only", "-S",
           "-Rpass-analysis=kernel-resource-usage", *[os.fspath(s) for s in build_native.SERVING_SOURCES], "-o",
           os.fspath(out)]
    result = subprocess.run(cmd, capture_output=True, text=True)
    assert result.returncode == 0, result.stderr[-2000:]
    usage, current = {}, None
    for line in result.stderr.splitlines():
        m = re.search(r"Function Name: (\S+)", line)
        if m:
            current = usage.setdefault(m.group(1), {})
            continue
        m = re.search(r"remark:.*?\s+([A-Za-z ]+?)(?: \[[^\]]*\])?: (\d+) \[", line)
        if m and current is not None:
            current[m.group(1).strip()] = int(m.group(2))
    asm = out.read_text()
    bodies = {}
    for m in re.finditer(r"^(_Z\S+):", asm, re.M):
        bodies[m.group(1)] = asm[m.end():asm.find(".Lfunc_end", m.end())].splitlines()
    # (without the kernels of the shared headers that this object does not launch)
    return tuple({n: x for n, x in of.items() if KERNELS.search(n)} for of in (usage, bodies))


def test_every_kernel_is_looked_at(device_code):
    usage, bodies = device_code
    assert set(usage) == set(bodies)
    counts = {}
    for n in usage:
        kind = KERNELS.search(n).group(1)
        counts[kind] = counts.get(kind, 0) + 1
    # head dims x (scaled e4m3, e4m3, bf16) x row tiles; x 1 for many rows; x
    # rotations, pages and types x groups of a wave; x types; x 1
    assert counts == {"attend_few": 18, "attend_many": 9, "token": 30, "cache_read": 6, "merge_few_ranges": 3,
                      "merge_many_ranges": 3}


def test_no_vector_register_goes_to_memory(device_code):
    usage, bodies = device_code
    for name, used in usage.items():
        assert used["VGPRs Spill"] == 0 and used["ScratchSize"] == 0, (name, used)
        assert _scratch_ops(bodies[name]) == (0, 0), name


def test_no_lds_read_into_a_pending_mfma_destination(device_code):
    _, bodies = device_code
    for name, lines in bodies.items():
        hits = _pending_destination_reads(lines)
        assert not hits, f"{name}: {hits[:3]}"


def test_m0_belongs_to_the_lds_dma_helpers(device_code):
    _, bodies = device_code
    dma = 0
    for name, lines in bodies.items():
        hits = _m0_misuse(lines)
        assert not hits, f"{name}: {hits[:3]}"
        dma += sum(1 for l in lines if l.strip().startswith("global_load_lds_dwordx4"))
    assert dma > 0
