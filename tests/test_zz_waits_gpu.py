"""GPU: after all other tests of the process."""
import pytest

from flexkv_b200 import fp4_cache


@pytest.mark.gpu
def test_no_wait_ran_out_in_any_test():
    assert fp4_cache.fp4_wait_timeouts() == 0
