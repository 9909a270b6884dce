"""In-place calls of group norm: `out` is the input wherever it is the same memory, however the strides of axes of one element were written.  No GPU."""
import pytest
import torch

from elektronn3_amd import ops

VIEWS = [      # shape, strides of two views of the same elements
    ((1, 3, 4, 5, 8), (480, 160, 40, 8, 1), (7, 160, 40, 8, 1)),
    ((1, 1, 4, 5, 8), (160, 160, 40, 8, 1), (160, 9, 40, 8, 1)),
    ((1, 1, 1, 1, 8), (8, 8, 8, 8, 1), (1, 1, 1, 1, 1)),
    ((2, 1, 1, 5, 8), (80, 80, 80, 16, 1), (80, 3, 3, 16, 1)),
    ((2, 3, 4, 5, 1), (60, 20, 5, 1, 1), (60, 20, 5, 1, 60)),
]


@pytest.mark.parametrize('shape,a,b', VIEWS)
def test_same_view(shape, a, b):
    buf = torch.zeros(1000)
    x, out = buf.as_strided(shape, a), buf.as_strided(shape, b)
    assert ops._ldc(x) == ops._ldc(out)
    ops._chk_out(out, x)
    ops._chk_out(x, out)
    # one element further on it is another view, which overlaps
    if x.numel() > 1 and shape[4] > 1:
        with pytest.raises(ValueError, match='overlaps'):
            ops._chk_out(buf[1:].as_strided(shape, b), x)
    # rows of another length, from the same address
    if shape[3] > 1 and shape[4] > 1:
        wide = torch.zeros(2000)
        with pytest.raises(ValueError, match='overlaps'):
            ops._chk_out(wide.as_strided(shape, [s * 2 for s in a[:4]] + [1]), wide.as_strided(shape, a))
