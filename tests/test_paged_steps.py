"""CPU checks of PagedCache's steps over a fake device: what they hand to the kernels, and what is left when one of them fails."""
import numpy as np
import pytest

from test_paged import FakeBuffer, FakeDevice, check, state  # noqa: F401
from webgpt_b200.paged import PagedCache


def test_starts_has_a_number_for_every_sequence():
    """The kernels read n_seq + 1 numbers: a number of tokens stands for all sequences, as in advance(), and nothing else fits."""
    c = PagedCache(FakeDevice(), 3, 1, 8, n_pages=12, page_size=4)
    for new in (2, np.int64(2), [2, 2, 2], np.array([2, 2, 2], np.int32)):
        assert list(c.starts(new).data.view(np.int32)) == [0, 2, 4, 6]
    assert list(c.starts([2]).data.view(np.int32)) == [0, 2, 4, 6]
    assert list(c.starts(0).data.view(np.int32)) == [0, 0, 0, 0]
    for new in ([1, 2], [1, 2, 3, 4], [[1, 2, 3], [1, 2, 3]], [1, -1, 1], -1):
        with pytest.raises(ValueError):
            c.starts(new)
