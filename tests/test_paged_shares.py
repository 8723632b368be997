"""How a paged attention call is cut between its two kernels (paged_work.cuh),
compiled for the host and swept over sizes up to the entry's limits (no GPU
needed): the shares are positive numbers and the grids fit the workspace, also for
the calls that are too large to run."""
from __future__ import annotations

import subprocess

import pytest

import __graft_entry__ as ge
from test_kernel_resources import CSRC

PROGRAM = r"""
#include <cstdio>

#include "paged_work.cuh"

int main() {
  int bad = 0, cases = 0;
  for (int sms : {2, 16, 132, 148})
    for (int rows : {1, 128, 129, 1 << 21, 1 << 30})          // query rows per KV head
      for (long long units : {1ll, 7ll, 300ll, 8192ll, 1ll << 22, 1ll << 30})
        for (long long keys : {1ll, 4096ll, 33ll << 20, 1ll << 30})  // of the prefix
          for (float own : {1.0f, 1e3f, 1e7f, 1.1e12f, 3e20f}) {
            hxb::PagedArgs a{};
            a.ctas[0] = sms;
            a.ctas[1] = 2 * sms;
            a.group = 1;
            a.total_q = rows;
            const int work = (int)((keys + hxb::kBN - 1) / hxb::kBN) + 2;
            const hxb::WideShare w = hxb::wide_share(a, (int)units, work, own);
            const int ctas = hxb::ctas_beside(a, (int)units, w);
            const bool fits = (double)units * work < (double)hxb::kMostWork;
            ++cases;
            if (w.per < 1 || w.work < work || ctas < 2 || ctas > a.ctas[1] ||
                (fits && (double)units * w.work > (double)sms * w.per * (1 + 1e-6))) {
              if (bad++ < 5)
                printf("sms %d rows %d units %lld work %d own %g: per %d, work %d, ctas %d\n", sms,
                       rows, units, work, own, w.per, w.work, ctas);
            }
          }
  printf("%d of %d\n", bad, cases);
  return bad != 0;
}
"""


def test_shares_of_the_two_kernels_are_numbers_at_every_size(tmp_path):
    build = ge._load_build_module()
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("nvcc not available")
    src, exe = tmp_path / "shares.cu", tmp_path / "shares"
    src.write_text(PROGRAM)
    r = subprocess.run([nvcc, *build.NVCC_FLAGS, "-I", str(CSRC), str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, f"status {r.returncode}: {r.stdout}"
