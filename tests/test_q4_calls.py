"""The Python layer of the 4-bit operators without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("shape,rows", [((0,), 1), ((3, 0), 3), ((2, 3, 0), 6), ((2, 0, 3, 0), 0), ((2, 3, 5), 6), ((5,), 1), ((0, 4, 8), 0)])
def test_rows_of_any_shape(shape, rows):
    """(..., n) as rows, with no columns too: the gradient of a product with a matrix that has no rows."""
    from ultraquant_b200 import q4
    assert tuple(q4._rows(torch.ones(shape)).shape) == (rows, shape[-1])


def test_overlap_is_that_of_the_bytes():
    """Against the sets of bytes, for views of one buffer: all that share are found, and columns, rows in turn and parts that
    do not share are told apart where the row strides agree or one of them is in one piece."""
    import random
    from ultraquant_b200 import q4
    rng = random.Random(3)
    buf = torch.zeros(240, dtype=torch.int16)

    def view():
        rows, n = rng.randint(0, 6), rng.randint(1, 9)
        step = rng.choice([n, n + rng.randint(1, 12), 12, 24])
        if step < n or (rows and (rows - 1) * step + n > 240):
            return view()
        at = rng.randint(0, 240 - ((rows - 1) * step + n if rows else 0))
        return torch.as_strided(buf, (rows, n), (step, 1), at)

    def members(t):
        return {t.storage_offset() + i * t.stride(0) + j for i in range(t.shape[0]) for j in range(t.shape[1])}

    seen = [0, 0]
    for _ in range(20000):
        a, b = view(), view()
        share = bool(members(a) & members(b))
        got = q4._overlap(a, b)
        if a.stride(0) == b.stride(0) or min(a.shape[0], b.shape[0]) <= 1 or a.is_contiguous() or b.is_contiguous():
            assert got == share, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
            seen[share] += 1
        else:
            assert got or not share
    assert min(seen) > 2000
    flat = buf[10:50]
    assert q4._overlap(flat, buf[49:]) and not q4._overlap(flat, buf[50:]) and not q4._overlap(buf[:10], flat)
