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


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("gradients", [0, 1])
@pytest.mark.parametrize("rows,table,dim", [(1 << 25, 1000, 1024), (1 << 22, 100, 65_536), (1 << 20, 1, 65_536), (1 << 29, 300, 64)])
def test_packed_rows_count_in_a_piece(lib, dtype, gradients, rows, table, dim):
    """Rows are packed a piece at a time: 4 GiB hold what a piece needs, beside the table's operands, the parts of
    one product (at most 512 of them), the sum over pieces and a power of two a row."""
    got = lib.vhip_softmax_xent_workspace(dtype, rows, table, dim, gradients)
    size = 4 if dtype == F32 else 2
    beside = table * (dim + 64) * (size + 4) + 512 * 256 * (dim + 4) * 4 + 4 * rows
    assert got <= (4 << 30) + (1 << 28) + beside


@pytest.mark.parametrize("a,b,c,steps,refused", [
    (3.4445, -4.7750, 2.0315, 100, False), (25.0, -0.04, 0.0, 2, False), (25.0, -0.04, 0.0, 3, False), (25.0, -0.04, 0.0, 4, True), (2.0, 0.0, 0.0, 30, False),
    (2.0, 0.0, 0.0, 31, True), (25.0, 0.0, 0.0, 7, True), (1e20, 0.0, 0.0, 1, True), (3.0, 40.0, 0.0, 5, True),
    (0.0, 0.0, 1.5e9, 1, True), (1.0, -4e9, 3e9, 1, True), (-2.0, 1.5, -0.5, 50, False), (0.0, 0.0, 0.0, 3, False),
])
def test_coefficients_without_a_bound_are_refused(lib, a, b, c, steps, refused):
    """All other checks are passed: what is not refused gets as far as looking for its GPU."""
    missing = lib.vhip_device_count() + 100
    got = lib.vhip_orthogonalize(missing, F32, 4096, 1, 4, 8, 8, 32, steps, a, b, c, 1e-7, 4096, 8, 32, 4096, 1 << 30, None)
    assert got != 0 and (got == -5) == refused
