"""What the paged operators refuse or report, without a GPU."""

import pytest

from light_b200 import _lib, ops


@pytest.mark.parametrize("device", [63, 64, -1])
def test_status_of_a_device_that_is_not_there_is_an_error_and_no_bits(device):
    """CUDA's error codes are positive: 100, as bits, would say that a slot was outside the cache."""
    assert _lib.lib().light_b200_paged_status(device) < 0
    with pytest.raises(_lib.Light200Error, match="light_b200"):
        ops.paged_status(device)
    assert _lib.lib().light_b200_paged_status_clear(device) < 0
    with pytest.raises(_lib.Light200Error, match="light_b200"):
        ops.paged_status(device, clear=True)
