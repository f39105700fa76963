"""What the paged cache hands its entry points of an operand: rows at the stride that
they lie at where the kernels can read them so, a copy where not."""
import pytest
import torch

from eredu_amd import EreduError, PagedKVCache

D, HEADS = 128, 4


def rows(t):
    c = PagedKVCache.__new__(PagedKVCache)
    c.head_dim, c._index, c.device = D, t.get_device(), t.device
    return c._rows(t, "q")


def filled(*shape):
    return torch.arange(torch.Size(shape).numel(), dtype=torch.float32).remainder_(251).view(shape).to(torch.bfloat16)


def aligned(t):
    """t's values where 16-byte alignment of what follows is by the offset alone."""
    assert t.data_ptr() % 16 == 0
    return t


ONE_ROW = [
    lambda: filled(HEADS, 1, D).transpose(0, 1),                     # kept by head
    lambda: filled(HEADS * D).as_strided((1, HEADS, D), (0, D, 1)),  # a row given to many
    lambda: filled(HEADS * D).as_strided((1, HEADS, D), (3, D, 1)),
    lambda: filled(HEADS, 1, D).transpose(0, 1)[:, :1],              # one head
    lambda: filled(1, HEADS, 3, D)[:, :, 1],                         # heads apart
    lambda: filled(1, HEADS * D + 4)[:, : HEADS * D],                # in a row of odd width
    lambda: filled(5, 3 * HEADS * D)[2:3, HEADS * D : 2 * HEADS * D],
    lambda: filled(HEADS, D).expand(1, HEADS, D),
]


@pytest.mark.parametrize("i", range(len(ONE_ROW)))
def test_one_row_at_any_stride(i):
    t = aligned(ONE_ROW[i]())
    got = rows(t)
    heads = t.numel() // D
    assert got.shape == (1, heads, D) and torch.equal(got.reshape(-1), t.reshape(-1))
    assert got.stride(0) >= heads * D and got.stride(0) % 8 == 0
    assert got.stride(2) == 1 and (heads == 1 or got.stride(1) == D) and got.data_ptr() % 16 == 0


@pytest.mark.parametrize("n", [2, 5])
def test_rows_at_their_stride_are_not_copied(n):
    x = filled(n, 3 * HEADS * D)
    part = x[:, HEADS * D : 2 * HEADS * D]
    got = rows(part)
    assert got.data_ptr() == part.data_ptr() and got.stride(0) == 3 * HEADS * D
    assert rows(x.view(n, -1, D)).data_ptr() == x.data_ptr()


@pytest.mark.parametrize("make", [lambda: filled(HEADS, 3, D).transpose(0, 1), lambda: filled(1, HEADS, D).expand(3, HEADS, D),
                                  lambda: filled(3, HEADS * D + 4)[:, : HEADS * D], lambda: filled(3, HEADS, 2 * D)[..., ::2],
                                  lambda: filled(3, HEADS * D + 8)[:, 1 : HEADS * D + 1]])
def test_other_layouts_are_copied(make):
    t = make()
    got = rows(t)
    assert got.is_contiguous() and got.stride(0) == HEADS * D and torch.equal(got, t.reshape(3, HEADS, D))


def test_refusals():
    for bad in (filled(2, HEADS, D + 8), filled(2, D + 8), filled(D), filled(2, 2, 2, D)):
        with pytest.raises(EreduError, match="rows, heads"):
            rows(bad)
    with pytest.raises(EreduError, match="bfloat16"):
        rows(torch.zeros(2, HEADS, D))


@pytest.mark.parametrize("make", [lambda: filled(HEADS * D, 3).t(), lambda: filled(HEADS * D, 1).t(),
                                  lambda: filled(3, 2 * HEADS * D)[:, ::2], lambda: filled(D, 3).t(),
                                  lambda: filled(1, 1).expand(3, HEADS * D)])
def test_flat_rows_with_their_values_apart(make):
    t = make()
    got = rows(t)
    assert got.is_contiguous() and got.stride(0) == t.shape[1] and torch.equal(got, t.reshape(t.shape[0], -1, D))
