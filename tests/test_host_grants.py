"""What the library remembers of the shared memory it was granted: every (kernel, device) pair, however many kernels and devices."""
import pytest

from ferro_kittens_b200._lib import library


@pytest.mark.parametrize("pairs", [0, 1, 63, 64, 65, 128, 500, 5000])
def test_every_grant_is_remembered(pairs):
    assert library().fk_selftest_grants(pairs) == pairs
