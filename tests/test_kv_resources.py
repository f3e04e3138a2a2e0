"""Registers of the attention kernels, checked at compile time (no GPU): of the forms that a short call
waits for, those of single tokens and those of few rows of up to 128 channels keep none in scratch memory,
few rows of 256 channels no more than a dozen, and two workgroups fit a CU."""
import os
import re
import shutil
import subprocess

import pytest

from tuckmill_amd import build as B


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """(registers, spilled, waves per SIMD) of every kernel over the cache, by its mangled name."""
    hipcc = shutil.which(B.HIPCC) or (B.HIPCC if os.path.exists(B.HIPCC) else None)
    if hipcc is None:
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("resources") / "device.o"
    cmd = [hipcc, "-x", "hip", "-std=c++17", "-O3", *B.DEVICE_FLAGS, "--cuda-device-only",
           "-I", os.path.join(B.ROOT, "include"), "-I", B.CSRC,
           "-Rpass-analysis=kernel-resource-usage", "-c", os.path.join(B.CSRC, "tm_kv.cpp"), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    found = {}
    for block in res.stderr.split("Function Name: ")[1:]:
        number = lambda what: int(re.search(re.escape(what) + r": (\d+)", block).group(1))
        found[block.split()[0]] = (number(" VGPRs"), number("VGPRs Spill"), number("Occupancy [waves/SIMD]"))
    return found


def of(kernels, pattern):
    some = [v for name, v in kernels.items() if re.search(pattern, name)]
    assert some, f"no kernel {pattern}"
    return some


def test_single_tokens_keep_their_registers(kernels):
    for registers, spilled, waves in of(kernels, r"attn_decode_kernelI(DF16_|f)Li\d+ELb[01]ELb0E"):
        assert spilled == 0 and waves >= 2, registers


def test_few_rows_keep_their_registers(kernels):
    for registers, spilled, waves in of(kernels, r"attn_decode_kernelI(DF16_|f)Li(64|128)ELb[01]ELb1E"):
        assert spilled == 0 and waves >= 3, registers


def test_tiles_of_rows_fit_two_workgroups_per_cu(kernels):
    for registers, spilled, waves in of(kernels, r"attn_prefill_kernelILi64E"):
        assert spilled == 0 and waves >= 2, registers
    for registers, spilled, waves in of(kernels, r"attn_prefill_kernelILi128E"):
        assert waves >= 2, registers


def test_few_rows_of_256_channels_keep_all_but_a_dozen_registers(kernels):
    for registers, spilled, waves in of(kernels, r"attn_decode_kernelI(DF16_|f)Li256ELb[01]ELb1E"):
        assert spilled <= 12 and waves >= 2, (registers, spilled)


def test_tiles_of_rows_of_256_channels_fit_a_cu(kernels):
    for registers, spilled, waves in of(kernels, r"attn_prefill_kernelILi256E"):
        assert spilled <= 24 and waves >= 1, (registers, spilled)


def test_tiles_of_rows_of_64_channels_fit_three_workgroups_per_cu(kernels):
    for registers, spilled, waves in of(kernels, r"attn_prefill_kernelILi64E"):
        assert spilled == 0 and waves >= 3, registers
