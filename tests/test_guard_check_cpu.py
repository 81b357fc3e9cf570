"""tools/guard_check.py without a device: its operands end (start) exactly where their mapping ends (starts), whatever their size, and an
option it does not know -- the retired ones that used to make a launch run out of bounds among them -- ends it before the runtime is touched."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "tools"))
import guard_check  # noqa: E402

GRAN, BASE = 1 << 21, 1 << 40


class FakeHip:
    """The virtual-memory calls, remembering what was mapped."""

    def __init__(self):
        self.reserved, self.mapped, self.unmapped = [], [], []

    def hipMemAddressReserve(self, out, span, align, *_):
        assert align.value == GRAN and span.value % GRAN == 0
        out._obj.value = BASE
        self.reserved.append(span.value)
        return 0

    def hipMemCreate(self, out, nbytes, *_):
        out._obj.value = 1
        assert nbytes.value % GRAN == 0
        return 0

    def hipMemMap(self, at, nbytes, *_):
        self.mapped.append((at.value, nbytes.value))
        return 0

    def hipMemSetAccess(self, at, nbytes, *_):
        assert (at.value, nbytes.value) == self.mapped[-1]
        return 0

    hipMemset = lambda self, at, fill, nbytes: 0 if (at.value, nbytes.value) == self.mapped[-1] else 1      # noqa: E731


@pytest.mark.parametrize("nbytes", [1, 2, 64, GRAN - 1, GRAN, GRAN + 1, 3 * GRAN, 5 * GRAN + 12346])
@pytest.mark.parametrize("front", [False, True])
def test_an_operand_touches_the_unmapped_page_on_the_asked_side(monkeypatch, nbytes, front):
    hip = FakeHip()
    monkeypatch.setattr(guard_check.Guarded, "hip", hip)
    monkeypatch.setattr(guard_check.Guarded, "gran", GRAN)
    monkeypatch.setattr(guard_check.Guarded, "prop", guard_check.MemAllocationProp(), raising=False)
    g = guard_check.Guarded(nbytes, front)
    (at, mapped), = hip.mapped
    assert at <= g.ptr and g.ptr + nbytes <= at + mapped                      # the whole operand is mapped
    assert g.ptr == at if front else g.ptr + nbytes == at + mapped            # and flush with the mapping's first / last byte
    assert at - BASE >= GRAN and BASE + hip.reserved[0] - (at + mapped) >= GRAN      # a reserved, unmapped granule on both sides


def test_extents_end_with_the_last_element():
    for case in guard_check.cases():
        m, n, k, _, _, tb, lda, ldb, ldc, batch, bcast = case
        rows_b, cols_b = (n, k) if tb else (k, n)
        last = lambda rows, cols, ld, entries: int(np.ravel_multi_index((entries - 1, rows - 1, cols - 1), (entries, rows, ld)))      # noqa: E731
        assert guard_check.gemm_extents(case) == (last(m, k, lda, batch) + 1, last(rows_b, cols_b, ldb, 1 if bcast else batch) + 1, last(m, n, ldc, batch) + 1)


def test_a_tensor_is_as_long_as_its_last_element(monkeypatch):
    seen = []
    monkeypatch.setattr(guard_check, "Guarded", lambda nbytes, front: seen.append(nbytes) or C.c_int())
    from cubecl_amd import ElemType
    guard_check.guarded_tensor((3, 5), (11, 2), ElemType.F32, False, [])
    guard_check.guarded_tensor((0, 5), (5, 1), ElemType.F32, False, [])
    assert seen == [4 * (2 * 11 + 4 * 2 + 1), 1]


@pytest.mark.parametrize("option", [["--selftest"], ["--resume-after", "3:auto"], ["--self"], ["--resume", "0:auto"]])
def test_retired_options_end_it_before_the_device_is_touched(option):
    r = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, 'tools'); import guard_check as g\n"
                        "def no(*a, **k): raise SystemExit('the device was touched')\n"
                        "g.Mi355Runtime.client = g.Guarded.init = no\nsys.argv[1:] = " + repr(option) + "\ng.main()"],
                       cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 2 and "unrecognized arguments" in r.stderr and "touched" not in r.stderr, r.stderr[-500:]
