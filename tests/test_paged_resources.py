"""Resource assumptions of the paged attention kernels, read from ptxas's report
at build time (no GPU needed): the wide kernel launches with the registers its
split names and does not spill; two CTAs of the narrow kernel fit an SM, and its
instances for decode rows (at most 8 per KV head) do not spill."""
from __future__ import annotations

import re

import pytest

from test_kernel_resources import CSRC, _kernels, _ptxas_report


@pytest.fixture(scope="module")
def report():
    return _ptxas_report(CSRC / "attention_paged.cu")


def test_wide_kernel_matches_its_register_split_without_spills(report):
    text = (CSRC / "attention_paged_wide.cuh").read_text()
    launch = int(re.search(r"constexpr int kPagedRegsLaunch = (\d+);", text).group(1))
    found = _kernels(report, "attention_paged_wide_kernel")
    assert len(found) == 2  # D = 64, 128
    for name, used in found.items():
        assert used == (launch, 0, 0), f"{name}: (registers, spill stores, loads) = {used}"


def test_narrow_kernel_fits_twice_on_an_sm(report):
    found = _kernels(report, "attention_paged_narrow_kernel")
    assert len(found) == 6  # 4, 8 and 16 rows of D = 64, 128
    for name, (regs, st, ld) in found.items():
        rows = int(re.search(r"ILi\d+ELi(\d+)E", name).group(1))
        assert -(-regs // 8) * 8 * 256 * 2 <= 65536, f"{name}: {regs} registers"
        assert rows == 16 or st == ld == 0, f"{name}: {st} B spill stores, {ld} B spill loads"


def test_combine_kernel_does_not_spill(report):
    for name, (regs, st, ld) in _kernels(report, "attention_paged_combine_kernel").items():
        assert st == ld == 0, f"{name}: {st} B spill stores, {ld} B spill loads"
