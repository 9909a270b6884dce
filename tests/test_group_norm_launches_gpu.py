"""Group norms of many small groups, which take one launch or two by the lines that their groups share, against the formulas in 64 bits: element by element, with
the bounds of test_group_norm_gpu.py."""
import numpy as np
import pytest
import torch

from test_group_norm_gpu import DTYPES, HALF, check_stats, make, ops, ref_bwd, ref_fwd, ref_keep, ref_side, ref_stats, within      # noqa: F401

pytestmark = pytest.mark.gpu

SIZES = [
    (2, 16, 16, 16, 64, 64),       # instance norm of 4096 voxels
    (1, 13, 17, 12, 32, 32),
    (4, 16, 16, 16, 128, 128),
    (40, 8, 8, 8, 512, 64),        # groups of 8 channels, two launches in every type
    (8, 8, 8, 8, 512, 64),         # one
    (700, 4, 8, 8, 32, 8),         # groups of 4
    (600, 3, 5, 7, 96, 8),         # groups of 12
    (100, 3, 5, 7, 96, 8),
    (200, 5, 7, 9, 33, 33),        # rows of single elements
    (700, 2, 6, 10, 66, 2),
    (1700, 1, 10, 10, 80, 2),      # groups of 80 bytes in 16 bits, 160 in 32
]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', SIZES)
def test_whole_pass(ops, size, dtype):     # noqa: F811
    for act in ('relu', 'silu'):
        x, dy, w, b = make(size, dtype, seed=41)
        y, mean, rstd, ck = ops.group_norm_act(x, size[5], w, b, activation=act, checkpoint=True)
        check_stats(x, mean, rstd, size[5], 1e-5)
        want, err = ref_fwd(x, *ref_stats(x, size[5], 1e-5), w, b, act)
        within(y, want, err, dtype, f'{act} y')
        assert torch.equal(ops.group_norm_act(x, size[5], w, b, activation=act)[0], y)
        q, scale, _ = ref_keep(x)
        q = ref_side(x, q, scale, mean, rstd, w, b, act)
        assert np.array_equal(ck.q.cpu().numpy(), q) and np.array_equal(ck.scale.cpu().numpy(), scale)
        xin = x.clone()
        y2, _, _, ck2 = ops.group_norm_act(xin, size[5], w, b, activation=act, checkpoint=True, out=xin)
        assert torch.equal(ck2.q, ck.q) and torch.equal(ck2.scale, ck.scale)
        torch.testing.assert_close(y2, y, rtol=2 * HALF[dtype] + 1e-5, atol=1e-5)        # (the statistics' sums may have another order)
        val = torch.from_numpy((q.astype(np.float64) * np.repeat(scale.astype(np.float64), 64)[:q.size]).astype(np.float32)).cuda().reshape(x.shape)
        for src, at in ((x, x), (ck, val)):
            got = ops.group_norm_act_bwd(src, mean, rstd, dy, w, b, activation=act)
            want, err = ref_bwd(at, mean, rstd, dy, w, b, act)
            for g, r, e, name in zip(got, want, err, ('dx', 'dweight', 'dbias')):
                within(g, r, e, dtype if name == 'dx' else torch.float32, f'{act} {name}')
