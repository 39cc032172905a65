"""CPU tests: further calls that the attention operators refuse, and what their host side answers.  None of these calls
reaches a kernel launch."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def g():
    import gptoss_moe
    return gptoss_moe


A = 1 << 20  # an aligned address that no call here reads


@pytest.mark.parametrize("change", [dict(beta_fast=float("inf")), dict(beta_fast=1e308),
                                    dict(beta_fast=1e300, original_positions=1e-30),
                                    dict(beta_fast=float("inf"), original_positions=float("inf"))])
def test_rope_ramp_without_a_beginning_refused(g, change):
    """Frequencies would be NaN: the ramp begins infinitely far away."""
    cfg = g.default_rope_config()
    for k, v in change.items():
        setattr(cfg, k, v)
    assert g.lib.gptoss_rope_table(ctypes.byref(cfg), A + 4, None) == g.GPTOSS_ERR_INVALID
    assert b"beta_fast" in g.lib.gptoss_last_error()
    cfg.scaling_factor = 1.0  # unused then: what is refused is the table's alignment
    assert g.lib.gptoss_rope_table(ctypes.byref(cfg), A + 4, None) == g.GPTOSS_ERR_INVALID
    assert b"aligned" in g.lib.gptoss_last_error()
