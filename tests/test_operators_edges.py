"""Operators of the quantized layers at the ends of what they take: what needs no device.  Refusals are decided on the host, before any launch."""
import pytest

from tests.test_operators import P, _status


@pytest.mark.parametrize("K", [2 ** 30 + 1, 2 ** 31 - 16384, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
def test_rows_longer_than_the_kernel_counts_are_refused(K):
    """Columns are counted in 32 bits in steps of up to 16384, and looked at up to as many behind the last step: near 2^31 the count would wrap."""
    status, message = _status("mq_quantize_tokens", P, 1, 1, K, K, P, K, P, None)
    assert status == 3 and b"2^30" in message
