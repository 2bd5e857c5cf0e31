"""Sizes of the workspaces around the experts, without a GPU."""

import ctypes

import pytest

from calibration_free_moe.reader import _ext


@pytest.mark.parametrize("hidden,splits", [
    (8, 1), (256, 1), (264, 2), (4096, 16), (4104, 9), (4608, 9), (4616, 10), (5120, 10), (8192, 16),
    (8200, 11), (65536, 16),
])
def test_no_split_of_the_hidden_dimension_is_empty(hidden, splits):
    """Up to 16 workgroups share it in whole turns of 256 values: as many as have any."""
    size = _ext.library().cfmoe_apply_adapters_scratch_bytes
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_int32] * 6
    assert size(hidden, 64, 40, 4, 3, 0) == splits * 3 * 40 * 4


@pytest.mark.parametrize("hidden,splits", [(256, 1), (264, 2), (4104, 2), (65536, 2)])
def test_splits_of_many_tokens(hidden, splits):
    size = _ext.library().cfmoe_apply_adapters_scratch_bytes
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_int32] * 6
    sort = size(hidden, 64, 40, 4, 5000, 0) - splits * 5000 * 40 * 4
    assert sort == size(hidden, 64, 48, 4, 5000, 0) - splits * 5000 * 48 * 4
    assert 0 < sort <= 2 * 5000 * 4 + 65536
