"""Statistics that the C++ adapter's residual norm must not use: those of an earlier training step after a forward in
evaluation mode, or after one that was refused (no device is touched)."""
from tests.test_cpp_adapter import driver


def test_backward_needs_the_last_forward_to_be_a_training_one():
    assert driver().drv_stale_statistics() == 0
