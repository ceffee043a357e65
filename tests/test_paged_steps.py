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


class Failing(FakeDevice):
    """A device whose n-th allocation or write from now on fails."""
    left = None

    def step(self):
        if self.left is not None:
            self.left -= 1
            if self.left < 0:
                raise OSError("no")

    def buffer(self, nbytes, dims=None):
        self.step()
        device = self

        class Buffer(FakeBuffer):
            def write(self, array, offset=0):
                device.step()
                return super().write(array, offset)

            def read(self, dtype, count, offset=0):
                return self.data[offset:offset + count * np.dtype(dtype).itemsize].view(dtype).copy()

        b = Buffer(nbytes)
        self.made = getattr(self, "made", []) + [b]
        return b


def attempts(c, call, untouched):
    """Lets each allocation and write of the call fail in turn: the cache stays what it was. Then the call is made."""
    for n in range(100):
        before = list(c.free), [list(p) for p in c.pages], list(c.lengths)
        c.device.left = n
        try:
            call()
        except OSError:
            c.device.left = None
            assert (list(c.free), c.pages, list(c.lengths)) == before
            check(c)
            untouched()
            continue
        c.device.left = None
        check(c)
        return n
    raise AssertionError("too many steps")


def test_steps_that_fail_change_nothing():
    c = PagedCache(Failing(), 3, 1, 8, n_pages=20, page_size=4, max_length=30, weights=True)
    assert attempts(c, lambda: c.advance([9, 1, 17]), lambda: None) >= 2
    assert attempts(c, lambda: c.retreat([0, 1, 9]), lambda: None) >= 2
    assert attempts(c, lambda: c.release(0), lambda: None) >= 2
    assert list(c.lengths) == [0, 0, 8]
