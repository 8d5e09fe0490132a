"""The products with 4-bit weights against 64 bits where a NaN counts as wrong: a comparison of the form |a - b| > bound is false
for NaN, which a kernel writes where a wait ran out or a row does not exist. The cases are those of test_gpu_q4, run once more."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_q4 as q4  # noqa: E402
from test_gpu_q4 import (  # noqa: E402, F401
    test_dense, test_glu, test_groups, test_ids, test_long_rows, test_one_matrix_in_an_order, test_short_groups_among_long_ones,
    test_strides, test_strides_of_many_rows, test_sums_of_one_sign)

compared = q4.check


def strict(got, y, tol, skip=None, rms=6 * 4 * 2.0 ** -23):
    """test_gpu_q4.check, and every value that it compares is a finite number."""
    finite = torch.isfinite(got)
    if skip is not None:
        finite[skip] = True
    assert bool(finite.all()), f"{int((~finite).sum())} of {finite.numel()} not finite, at {(~finite).nonzero()[:4].tolist()}"
    compared(got, y, tol, skip, rms)


@pytest.fixture(autouse=True)
def checked(monkeypatch):
    monkeypatch.setattr(q4, "check", strict)


def test_strict_rejects_one_nan():
    y = torch.ones((9, 9), dtype=torch.float64)
    for dtype in (q4.F16, q4.BF16, q4.F32):
        good, bad = y.to(dtype), y.to(dtype)
        bad[3, 4] = float("nan")
        q4.check(good, y, 0.0 * y, rms=None)
        q4.check(bad, y, 0.0 * y, torch.tensor([3]), rms=None)
        with pytest.raises(AssertionError):
            q4.check(bad, y, 0.0 * y, rms=None)


for _test in (test_dense, test_glu, test_groups, test_ids, test_long_rows, test_one_matrix_in_an_order, test_short_groups_among_long_ones,
              test_strides, test_strides_of_many_rows, test_sums_of_one_sign):
    pytest.mark.gpu(_test)
