"""Attention over the paged cache without a GPU: arguments of its self-test."""
import ti_b200 as ti


def test_selftest_stop_takes_steps_and_minus_one():
    try:
        assert ti.lib().ti_selftest_paged_stop(-2) == ti.TI_ERR_INVALID
        assert "step" in ti.lib().ti_last_error().decode()
        assert ti.lib().ti_selftest_paged_stop(3) == 0
    finally:
        assert ti.lib().ti_selftest_paged_stop(-1) == 0
