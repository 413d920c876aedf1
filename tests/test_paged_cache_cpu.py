"""The buffers of the paged 4-bit cache, on the host."""
import pytest

from dynaflow_b200 import ops
from dynaflow_b200.paged import PagedKVCache4


@pytest.mark.parametrize("max_len,page", [(100, 64), (128, 64), (1, 16), (17, 16), (300, 48)])
def test_every_position_that_can_have_a_slot_has_its_angles(max_len, page):
    """A request may grow to the end of its last page."""
    cache = PagedKVCache4(1, 1, num_pages=8, page_size=page, max_requests=1, max_len=max_len, max_rows=4, rope_theta=500.0, device="cpu")
    room = cache.page_table.shape[1] * page
    assert room >= max_len and cache.angles.shape == (room, 128)
    assert (cache.angles == ops.rope_angles(room, 500.0, "cpu")).all()
