"""The chunks that the input-gradient GEMMs load, checked on the CPU for every lane: csrc/qgemm_chunks.h is plain C++, and the kernels take
their addresses from it.  (What a lane reads outside a row is masked before it reaches a product, so values alone would not show it;
tests/test_gemm_bounds_gpu.py shows the wide kernel's reads of the first operand only.)"""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <initializer_list>
#include "qgemm_chunks.h"
// an operand of `rows` rows of K elements, `ld` apart: the reads of a lane, row * ld + offset ... + width, must end inside it
static int bad = 0;
static void look(const char* what, int rows, int K, long ld, long at, int width) {
  const long end = (long)(rows - 1) * ld + K;
  if (at < 0 || at + width > end || at % ld + width > K) { ++bad; std::printf("%s K %d rows %d at %ld\n", what, K, rows, at); }
}
int main() {
  const int Ks[] = {8, 16, 24, 32, 40, 64, 72, 104};
  for (int K : Ks) for (int rows : {1, 5, 127, 128, 129, 300}) for (int pad : {0, 8}) {
    const long ld = K + pad;
    const int nkt = (K + 31) / 32;
    for (int first = 0; first < rows; first += 128)
      for (int k0 = 0; k0 <= (nkt + 2) * 32; k0 += 32)
        for (int tid = 0; tid < 512; ++tid) {
          const int ca = (tid & 7) * 4, cb = (tid & 3) * 8;
          for (int i = 0; i < 4; ++i) {
            const long ra = (long)qbs_row(first, (tid + 512 * i) >> 3, rows) * ld, rb = (long)qbs_row(first, (tid + 512 * i) >> 2, rows) * ld;
            look("wide A", rows, K, ld, ra + qbs_chunk0(ca, K) + OFFSET(ca, k0, K), 4);
            look("wide B", rows, K, ld, rb + qbs_chunk0(cb, K) + OFFSET(cb, k0, K), 8);
            look("narrow A", rows, K, ld, ra + ca + qbs_chunk_from_c(ca, k0, K), 4);
            look("narrow B", rows, K, ld, rb + cb + qbs_chunk_from_c(cb, k0, K), 8);
            look("narrow A, no scale", rows, K, ld, ra + ca - ca, 4);
          }
          look("wide scale", 1, K, K, OFFSET(ca, k0, K) + qbs_chunk0(ca, K), 4);
          look("wide A, no scale", 1, K, K, qbs_chunk0(ca, K), 4);
          look("narrow scale", 1, K, K, qbs_chunk(ca, k0, K), 4);
          // what is inside is where it belongs
          if (k0 + ca < K && qbs_chunk0(ca, K) + OFFSET(ca, k0, K) != k0 + ca) ++bad;
          if (k0 + cb < K && cb + qbs_chunk_from_c(cb, k0, K) != k0 + cb) ++bad;
          if (bad > 5) return 1;
        }
  }
  return bad != 0;
}
"""


def run(tmp_path, program):
    cxx = shutil.which("g++") or shutil.which("c++") or shutil.which("clang++")
    assert cxx, "a C++ compiler"
    (tmp_path / "t.cpp").write_text(program)
    exe = str(tmp_path / "t")
    subprocess.run([cxx, "-O1", "-std=c++17", "-I", os.path.join(ROOT, "ofq_amd", "csrc"), str(tmp_path / "t.cpp"), "-o", exe], check=True)
    return subprocess.run([exe], capture_output=True, text=True)


def test_every_lane_reads_inside_its_operand(tmp_path):
    r = run(tmp_path, PROGRAM.replace("OFFSET", "qbs_step"))
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("mistake", [("qbs_chunk0(ca, K)", "ca"), ("qbs_chunk0(cb, K)", "cb"), ("ra + ca - ca", "ra + ca"), ("OFFSET(ca, k0, K)", "k0")])
def test_the_check_sees_a_read_behind_the_row(tmp_path, mistake):
    """A lane's chunk left where it is in a row shorter than a step, a placeholder load from it, a step past the row's end."""
    r = run(tmp_path, PROGRAM.replace(*mistake).replace("OFFSET", "qbs_step"))
    assert r.returncode != 0
