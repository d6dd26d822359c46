"""Block tables at the sizes where their launch changes."""

import pytest

from test_block_tables_gpu import mixed, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [4083, 4084, 4085, 4095, 4096, 4097])
def test_requests_whose_sums_take_about_64_KiB(count):
    """Four words a request in LDS beside what every workgroup has there: from 4084 requests on more than a launch has unasked."""
    step(mixed(count, count, most=40), 16, seed=count)
