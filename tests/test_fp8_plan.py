"""What the block-scaled e4m3 products plan from their sizes, on the CPU: the scratch queries refuse what the
calls refuse."""
import pytest

from eredu_amd import _native

L = _native.lib()
P = 4096  # an address; nothing here gets as far as a launch
BF16, E4M3 = 2, 4


def grouped(x_rows, experts, routes, n, k, x_dtype):
    coded = x_dtype == E4M3
    return L.eq_fp8_grouped_matmul(P, P, k, P if coded else None, x_rows if coded else 0, x_rows, P, P, experts, P, P, routes, n, k,
                                   x_dtype, BF16, P + 16, 0, None)  # (scratch that no call takes)


@pytest.mark.parametrize("routes", [1, 64, 65, 5000])
@pytest.mark.parametrize("x_rows,k,x_dtype,words", [
    (0, 128, E4M3, "x must have a row"), (0, 128, BF16, "x must have a row"),
    (1 << 20, 3200, E4M3, "3 * 2^30"), (1 << 20, 3200, BF16, "3 * 2^30"), (1 << 12, 1 << 20, BF16, "3 * 2^30")])
def test_scratch_of_routes_is_refused_where_the_call_is(x_rows, k, x_dtype, words, routes):
    assert grouped(x_rows, 4, routes, 64, k, x_dtype) != 0
    assert words in L.eq_last_error().decode()
    assert L.eq_fp8_grouped_matmul_scratch(x_rows, 4, routes, 64, k, x_dtype, BF16) == -1
    assert words in L.eq_last_error().decode()


def test_scratch_of_routes_up_to_the_limit():
    """One row below 3 * 2^30 bytes is taken, and nothing is refused for an x that no route reads."""
    rows = (3 << 30) // 3200
    assert rows * 3200 < 3 << 30 <= (rows + 1) * 3200
    assert L.eq_fp8_grouped_matmul_scratch(rows, 4, 100, 64, 3200, BF16, BF16) >= rows * 3200
    assert L.eq_fp8_grouped_matmul_scratch(rows + 1, 4, 100, 64, 3200, BF16, BF16) == -1
    for routes, n in ((0, 64), (100, 0)):
        assert L.eq_fp8_grouped_matmul_scratch(0, 4, routes, n, 128, E4M3, BF16) >= 0
        assert grouped(0, 4, routes, n, 128, E4M3) == 0
