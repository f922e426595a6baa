"""CPU: attention over parts of a cache (first tokens kept beside a window, log-sum-exps, shared prefixes,
joined states), the unchanged kernel sources built for the host against a HIP emulator under
AddressSanitizer + UBSan on exact-size buffers, against the C oracle; and the refusals of their C entry
points, before any launch."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

EMU = Path(__file__).resolve().parent / "hostemu"

pytestmark = pytest.mark.skipif(not Path("/opt/rocm/llvm/bin/clang++").exists(), reason="needs ROCm clang++")


@pytest.fixture(scope="module")
def program():
    subprocess.run(["make", "-s", "-C", str(EMU), "_build/emu_states"], check=True, timeout=600, capture_output=True)
    return EMU / "_build" / "emu_states"


@pytest.mark.parametrize("case", ["plan", "merge", "decode", "prefill", "shared"])
def test_kernels_under_host_emulation_and_asan(program, case):
    res = subprocess.run([str(program), case], capture_output=True, text=True, timeout=600)
    tail = "\n".join((res.stdout + res.stderr).splitlines()[-40:])
    assert res.returncode == 0, tail
    assert "all ok" in res.stdout, tail
