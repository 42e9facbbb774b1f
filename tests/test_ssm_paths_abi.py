"""Further refusals and sizes of the selective scan and the product with its epilogue (include/fhc_seq.h), without a GPU: every
refusal is an error status with a message before any device work; the pointers are never followed."""
import pytest

import fhtest  # noqa: F401
from test_seq_abi import P, mod, refused
from test_ssm_abi import linear_call, ssm_call


@pytest.mark.parametrize("act,text", [(0x103, "act 259"), (0x203, "act 515"), (0x200, "act 512"), (0x1100, "act 4352")])
def test_linear_takes_one_flag_beside_the_activation(act, text):
    for back in (False, True):
        refused(linear_call(back, act=act), text)


def test_linear_workspace_of_a_rounded_dv_is_the_smaller():
    m = mod()
    L = m._lib()
    for rows, c, f in ((20, 64, 48), (300, 65, 47), (2500, 130, 4100)):
        for act in m.LINEAR_ACTS.values():
            full, rounded = (m.LinearDesc(1, act + flag, rows, c, f) for flag in (0, m.ROUND_DV))
            assert L.fhc_linear_saved_bytes(full) == L.fhc_linear_saved_bytes(rounded)
            assert L.fhc_linear_workspace_bytes(full, 0) == L.fhc_linear_workspace_bytes(rounded, 0)
            sizes = [L.fhc_linear_workspace_bytes(d, 1) for d in (full, rounded)]
            assert sizes[0] == sizes[1] if act == 2 else sizes[0] > sizes[1]


def test_ssm_groups_of_states_fit_an_index():
    """groups * n is a row of B and C, in 31 bits."""
    wide = (P, 1 << 40, 1 << 40)
    s = {n: wide for n in ("x", "dt", "bm", "cm", "z", "y", "dy", "dx", "ddt", "dbm", "dcm", "dz")}
    for d in (0, 1 << 26, 1 << 27):
        for back in (False, True):
            refused(ssm_call(back, b=1, t=1, d=d, n=64, groups=1 << 26, **s), "groups of 64 states")
    L = mod()._lib()
    assert L.fhc_ssm_workspace_bytes(mod().SsmDesc(1, 1, 1, 1 << 26, 64, 1 << 26, P, None, None, None), 1) == 0
