"""How a paged attention call is cut between its two kernels (paged_work.cuh),
compiled for the host and swept over sizes up to the entry's limits (no GPU
needed): the shares are positive numbers and the grids fit the workspace, also for
the calls that are too large to run. And the order of the launch dependencies that
lets the two run at once, read from the source."""
from __future__ import annotations

import re
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


def kernel_body(name):
    """The kernel's source behind its signature, without comments."""
    text = (CSRC / f"attention_paged_{name}.cuh").read_text()
    body = text[text.index(f"attention_paged_{name}_kernel("):]
    return re.sub(r"//.*", "", body)


def test_the_narrow_kernel_starts_when_all_before_the_wide_one_has_ended():
    """Beside the wide kernel the narrow one reads the inputs without a wait: it starts
    when every CTA of the wide one has triggered, which each does behind its own wait
    for all that came before. No path may trigger, or end, ahead of that wait."""
    wide = kernel_body("wide")
    assert wide.count("pdl_wait();") == wide.count("pdl_trigger();") == 1
    before, after = wide.split("pdl_wait();")
    assert "return" not in before and "pdl_trigger" not in before
    assert re.match(r"\s*pdl_trigger\(\);", after)  # at the top level, for all threads
    assert before.count("{") - before.count("}") == 1


def test_the_narrow_kernel_ends_behind_the_wide_one():
    """The combine kernel waits for the narrow one only, so no path of that one may let
    it start early or end without having waited for the wide one."""
    narrow = kernel_body("narrow")
    assert "pdl_trigger" not in narrow
    first, second, rest = narrow.split("pdl_wait();")
    assert re.search(r"if \(args\.beside\) \{[^{}]*\} else \{\s*$", first)
    assert re.search(r"if \(args\.beside\) $", second) and re.match(r"\s*\}\s*\}", rest)
    roles = second[second.index("if (warp == 0) {"):]
    assert not re.search(r"^  return", roles, re.M)  # (returns of the roles' lambdas only)
