"""The norm's C entries refuse what their kernels do not take before any launch (no GPU)."""
import pytest

from maloq_amd import _lib


def test_normed_row_entries():
    one = 16  # (no pointer is read)
    for name, args, what in [
            ("maloq_rms_norm_unit_fwd", (7, one, 8, None, 0, one, 4, 64, 1e-6, None, one, None, one, None), "dtype"),
            ("maloq_rms_norm_unit_fwd", (2, one, 8, None, 0, one, 4, 16385, 1e-6, None, one, None, one, None), "16384"),
            ("maloq_rms_norm_unit_fwd", (2, one, 8, None, 0, one, 1 << 31, 64, 1e-6, None, one, None, one, None), "out of range"),
            ("maloq_rms_norm_unit_bwd", (2, one, 8, None, 0, one, 8, one, one, 4, 64, None, one, one, None), "partial"),
            ("maloq_rms_norm_unit_bwd", (3, one, 8, None, 0, one, 8, one, one, 4, 64, one, one, None, None), "dtype")]:
        with pytest.raises(_lib.MaloqHipError, match=what):
            _lib.call(name, *args)
    _lib.call("maloq_rms_norm_unit_fwd", 2, None, 64, None, 0, None, 0, 64, 1e-6, None, None, None, None, None)  # no rows
