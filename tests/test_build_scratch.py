"""The build refuses kernels that keep values in scratch memory where none may (compiles, no GPU)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SPILLS = """
#include <hip/hip_runtime.h>
__global__ void turned(float* p, const int* at) {
  float x[64];
  for (int i = 0; i < 64; ++i) x[i] = p[64 * threadIdx.x + i];
  for (int i = 0; i < 64; ++i) x[at[i] & 63] += x[at[64 + i] & 63];
  for (int i = 0; i < 64; ++i) p[64 * threadIdx.x + i] = x[i];
}
"""
FITS = """
#include <hip/hip_runtime.h>
__global__ void twice(float* p) { p[threadIdx.x] *= 2.f; }
"""


@pytest.fixture(scope="module")
def build():
    spec = importlib.util.spec_from_file_location("tagi_build", ROOT / "triton-tagi_amd" / "build.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_the_attention_units_are_held_to_it(build):
    names = {src.name for src, _, _ in build.compile_units()}
    assert {"tagi_remax_attention.hip", "tagi_remax_step.hip"} <= set(build.NO_SCRATCH) <= names


def test_a_kernel_in_scratch_memory_ends_the_build(build, tmp_path):
    src = tmp_path / build.NO_SCRATCH[0]
    src.write_text(SPILLS)
    with pytest.raises(RuntimeError, match="scratch memory(.|\n)*turned.*bytes a lane"):
        build.compile_unit(build._hipcc(), src, tmp_path / "x.o", [])
    src.write_text(FITS)
    build.compile_unit(build._hipcc(), src, tmp_path / "x.o", [])
    assert (tmp_path / "x.o").exists()


def test_a_report_without_kernels_is_not_taken_for_a_good_one(build, tmp_path):
    src = tmp_path / build.NO_SCRATCH[0]
    src.write_text("int nothing() { return 0; }\n")
    with pytest.raises(RuntimeError, match="no kernel"):
        build.compile_unit(build._hipcc(), src, tmp_path / "x.o", [])
    other = tmp_path / "other.hip"  # any other unit may use it
    other.write_text(SPILLS)
    build.compile_unit(build._hipcc(), other, tmp_path / "x.o", [])
