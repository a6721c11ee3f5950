"""Workspaces and refusals of the training operators at the limits of their sizes, at the C ABI on the CPU."""
import pytest

F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    from vector_hip import training  # declares the signatures

    return training._lib


@pytest.mark.parametrize("dtype,longest", [(F32, 1 << 22), (F16, 1 << 23), (BF16, 1 << 23)])
@pytest.mark.parametrize("table", [65, 100, 190])
def test_gradients_take_rows_in_pieces_that_a_product_can_read(lib, dtype, longest, table):
    """The rows are K of the table's gradient: past the longest that a product reads, what grows with their number
    is at most a float's worth (a power of two) a row, beside the sum over pieces."""
    size = lib.vhip_softmax_xent_workspace
    at, past = size(dtype, longest, table, 16, 1), size(dtype, 4 * longest, table, 16, 1)
    assert past - at <= 4 * 3 * longest + 4 * table * 16 + 4096
