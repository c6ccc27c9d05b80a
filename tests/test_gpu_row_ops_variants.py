"""Row operators on the MI355X: the residual norm's remaining type pairs, and row counts that reach the kernels of many rows and
walk their grids more than once, against the definitions in 64 bits."""
import pytest

from test_gpu_row_ops import B, BF16, F16, F32, SIZES, check_layer_norm, check_residual_norm, data, params  # noqa: F401

pytestmark = pytest.mark.gpu

# both sides of the switch at 2048 rows, widths at both ends of its variants; rows that walk each grid's loop more than once
# with a ragged last turn
LONG = [(2048, 1000), (2049, 1000), (2049, 1024), (2051, 2047), (2049, 2048), (8195, 520), (9001, 1100), (12001, 300)]


@pytest.mark.parametrize("rows,width", LONG)
@pytest.mark.parametrize("dtype,ptype", [(F32, F32), (BF16, F32), (F16, F16)])
def test_layer_norm_of_many_rows(B, rows, width, dtype, ptype):
    w, b = params(width, ptype, 5)
    check_layer_norm(B, data(rows, width, dtype, 1), w, b, data(rows, width, dtype, 2))


@pytest.mark.parametrize("rows,width", LONG)
@pytest.mark.parametrize("dtype,rtype,p", [(F32, F32, 0.5), (BF16, F32, 0.1), (BF16, BF16, 0.0), (F16, F16, 0.25), (F16, F32, 0.2)])
def test_residual_norm_of_many_rows(B, rows, width, dtype, rtype, p):
    w, b = params(width, F32, 5)
    check_residual_norm(B, data(rows, width, dtype, 1), data(rows, width, rtype, 2), w, b, data(rows, width, dtype, 3),
                        data(rows, width, rtype, 4), p)


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("dtype,rtype,p", [(BF16, BF16, 0.1), (F16, F32, 0.25)])
def test_residual_norm_of_the_other_type_pairs(B, rows, width, dtype, rtype, p):
    w, b = params(width, dtype, 5)
    check_residual_norm(B, data(rows, width, dtype, 1), data(rows, width, rtype, 2), w, b, data(rows, width, dtype, 3),
                        data(rows, width, rtype, 4), p)
