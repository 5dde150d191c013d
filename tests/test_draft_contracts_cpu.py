"""Promises of the operators for drafted tokens that need no GPU."""
from conftest import nb


def test_wait_error_refusals():
    for name in ("nd_take_wait_error", "nd_wait_flag"):
        assert getattr(nb.lib(), name)(None) == 1  # cudaErrorInvalidValue
        assert nb.lib().nd_last_error().decode() == name + ": null pointer"
