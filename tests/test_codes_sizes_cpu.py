"""CPU: sizes that do not fit the 32 bits in which the library takes them, and shapes at their ends, are refused before it is called."""
import pytest
import torch

from test_codes_cpu import bare


def handle():
    """A handle that takes tensors without storage as its own."""
    c = bare()
    c.device = torch.empty(1, device="meta").get_device()
    return c


def empty(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("size", [1 << 32, (1 << 32) + 5, (1 << 33) + 1])
def test_tables_and_rows_beyond_32_bits_are_refused(size):
    c, idx, u = handle(), empty(2, dtype=torch.int32), empty(2)
    with pytest.raises(ValueError, match="rows"):
        c.lookup(idx, table=empty(size, 4))
    with pytest.raises(ValueError, match="2\\^32"):
        c.lookup(idx, table=empty(3, size))
    with pytest.raises(ValueError, match="2\\^32"):
        c.sample(empty(2, size), u)
    with pytest.raises(ValueError, match="rows"):
        c.lookup_gradient(empty(2, 4), idx, K=size)
    with pytest.raises(ValueError, match="2\\^32"):
        c.lookup_gradient(empty(2, size), idx, K=4)


def test_negative_tables_are_refused():
    with pytest.raises(ValueError):
        handle().lookup_gradient(empty(2, 4), empty(2, dtype=torch.int32), K=-1)


def test_results_without_dimensions_are_refused():
    """One index has no dimension; its result has one."""
    c, one = handle(), empty(dtype=torch.int32)
    for out in (empty(), empty(5), empty(1, 4)):
        with pytest.raises(ValueError):
            c.lookup(one, table=empty(3, 4), out=out)
    with pytest.raises(ValueError):
        c.lookup_gradient(empty(), one, K=3)
