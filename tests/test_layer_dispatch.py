"""Every kernel of routed_experts in the built library has a case that runs it.

The rules are those of tests/layer_dispatch.py; the library's own list of kernels says
whether they have kept up with the source.
"""

import re

from calibration_free_moe.reader import _ext
from tests import layer_dispatch as dispatch


def compiled():
    with open(_ext.LIBRARY_PATH, "rb") as f:
        found = re.findall(rb"_ZN5cfmoe12_GLOBAL__N_1\d\d(experts_[a-z0-9_]*_kernel(?:IL\w*?EE)?)Ev?NS", f.read())
    return {name.decode() for name in found}


def reached():
    found = set()
    for hidden, width, experts, pairs, fp4, counts in dispatch.CASES:
        found |= dispatch.launches(hidden, width, experts, 1, pairs, fp4, counts)
    return found


def test_every_kernel_has_a_case_and_every_case_a_kernel():
    assert {name for name, _, _ in reached()} == compiled()


def test_every_column_pass_has_a_case():
    """A rows kernel of up to four column tiles multiplies four, two or one at a time."""
    passes = {(name, tiles) for name, tiles, _ in reached()}
    for name in compiled():
        rows = re.fullmatch(r"experts_rows_kernel\w*ELb[01]ELi(\d)ELi\dEE", name)
        for tiles in (4, 2, 1) if rows else ():
            assert tiles > int(rows[1]) or (name, tiles) in passes, (name, tiles)


def test_kernels_of_one_round_have_cases_of_several_passes():
    several = {name for name, _, many in reached() if many}
    for name in compiled():
        if re.fullmatch(r"experts_rows_kernel\w*ELb[01]ELi[12]ELi1EE", name) or "down" in name:
            assert name in several, name


def test_cuts_leave_no_wave_without_a_load():
    for fp4, down, lengths in ((False, False, range(128, 4097, 128)), (True, False, range(128, 4097, 128)),
                               (True, True, range(32, 4097, 32))):
        for length in lengths:
            units = (length + 127) // 128 if fp4 else length // 32
            splits, loads = dispatch.cut_of(units, fp4, down)
            for wave in range(splits):
                steps = units * (wave + 1) // splits - units * wave // splits
                assert 1 <= steps <= loads <= (4 if fp4 else 16)
