"""What the setup of a device may fail for (no GPU needed): every launcher of the library returns -2 where it fails, so it fails for errors of the CUDA runtime
alone, and a kernel that cannot run as it was compiled keeps only its own calls from it."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "drama_rs_b200", "csrc")


def configure(name: str) -> str:
    with open(os.path.join(CSRC, name)) as f:
        s = re.sub(r"//[^\n]*", "", f.read())
    s = s[s.rindex("static cudaError_t configure_all() {") :]
    return s[: s.index("\n}\n")]


@pytest.mark.parametrize("name", ["block_norms.cuh", "gemv.cuh", "moe_decode.cuh", "moe_decode_fp8.cuh", "moe_few.cuh", "moe_prefill.cuh", "moe_prefill_tc.cuh",
                                  "proj_lora.cuh", "proj_rows.cuh", "router.cuh", "stack_decode.cuh"])
def test_setup_fails_for_runtime_errors_alone(name):
    own = set(re.findall(r"return (cudaError\w+);", configure(name)))
    assert own <= {"cudaErrorInvalidDevice"}, own  # beside those that a runtime call returned


def test_too_few_registers_keep_only_the_kernel_itself_off():
    with open(os.path.join(CSRC, "proj_rows.cuh")) as f:
        s = f.read()
    assert "g_fits[d] = a.numRegs >= LAUNCH_REGS && b.numRegs >= LAUNCH_REGS;" in configure("proj_rows.cuh")
    (decision,) = re.findall(r"if \((.*)\) return launch<F16>\(p, dev, st\);", s)
    assert decision.startswith("g_fits[d] && many(")
