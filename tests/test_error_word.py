"""The device's error word is kept by the one translation unit that reads it: a kernel of another unit whose wait can
give up would report to nobody, and does not build."""
import os
import subprocess

import pytest

from aiwn_b200.csrc import build

SOURCE = """
#define %s
#include "il_sm100.cuh"
extern "C" __global__ void waits(int* done) {
    __shared__ uint64_t bar;
    *done = %s;
}
"""


def _compiles(tmp_path, define, value):
    src = tmp_path / "unit.cu"
    src.write_text(SOURCE % (define, value))
    run = subprocess.run([build.NVCC, *build.FLAGS, "-I", build.HERE, "-c", "-o", str(tmp_path / "unit.o"), str(src)],
                         capture_output=True, text=True)
    return run.returncode == 0, run.stderr


@pytest.mark.skipif(not os.path.exists(build.NVCC), reason="needs nvcc")
def test_only_the_unit_with_the_error_word_may_wait(tmp_path):
    wait = "il::mbar_wait_bounded(il::smem_addr(&bar), 0)"
    ok, log = _compiles(tmp_path, "IL_ERROR_WORD", wait)
    assert ok, log
    ok, log = _compiles(tmp_path, "NO_ERROR_WORD", "(int)il::smem_addr(&bar)")
    assert ok, log
    ok, log = _compiles(tmp_path, "NO_ERROR_WORD", wait)
    assert not ok and "report_error" in log
