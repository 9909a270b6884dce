"""How far a norm's input is from what its 8-bit checkpoint stands for: half a step of the block, a whole one where an element keeps its side of a ReLU's border."""
import pytest
import torch

from test_group_norm_gpu import DTYPES, HALF, U, make, ops      # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('act', ['relu', 'leaky', 'lin', 'silu'])
def test_error_in_steps(ops, act, dtype):      # noqa: F811
    x, _, w, b = make((2, 8, 16, 17, 64, 8), dtype, seed=71)
    ck = ops.group_norm_act(x, 8, w, b, activation=act, checkpoint=True)[3]
    val = ck.q.double().view(-1, 64) * ck.scale.double()[:, None]
    amax = x.double().reshape(-1, 64).abs().amax(1, keepdim=True)
    off = (val - x.double().reshape(-1, 64)).abs() / amax
    # the roundings of 127 / amax, the product and the scale: 127 steps off by 3 u each, as for checkpoint8()
    half, whole = 0.5 / 127 + 6 * U, 1 / 127 + 6 * U
    if act in ('lin', 'silu'):
        assert bool((off <= half).all())
    else:
        moved = off > half
        assert bool((off <= whole).all()) and bool(moved.any()) and float(moved.double().mean()) < 0.01
