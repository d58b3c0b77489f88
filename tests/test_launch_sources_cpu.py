"""What the host side of the kernels keeps between calls: one process may use several devices, from several threads."""

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "himuon_b200" / "csrc"
LAUNCHERS = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("*.cu")) if "cudaFuncSetAttribute" in p.read_text() or "allow_smem" in p.read_text()}


def _kept(code):
    """Types of the variables that functions keep."""
    return re.findall(r"^[ \t]+static (?!__device__|constexpr|const |_assert|_cast)([^;(={]*)[;={]", code, re.M)


@pytest.mark.parametrize("name", ["gemm_sm100.cu", "gemm2_sm100.cu"])
def test_products_are_set_up_on_every_device(name):
    """Shared memory is allowed to a kernel for one device, and how many pairs fit is that device's: neither may be remembered for all of them."""
    code = LAUNCHERS[name]
    assert "cudaFuncSetAttribute" not in code and re.search(r"\ballow_smem\(", code)
    kept = [k for k in _kept(code) if not re.search(r"\[64\]", k)]
    assert kept and all(k.startswith("std::atomic<uint64_t>") for k in kept), kept


@pytest.mark.parametrize("name", LAUNCHERS)
def test_what_launches_keep_is_atomic_and_belongs_to_a_device(name):
    code = LAUNCHERS[name]
    kept = _kept(code)
    assert all(k.startswith("std::atomic<") for k in kept), kept
    for k in kept:                                       # a bit, or a place, for each device
        assert k.startswith("std::atomic<uint64_t>") or "[64]" in k, k
