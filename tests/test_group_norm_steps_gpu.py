"""Group norm on tensors that take every workgroup several steps with a ragged last one (the sizes of test_group_norm_gpu.py take one), and the forms that only large tensors reach: doubled
workgroup counts, finalising launches over group records, more groups than an apply pass merges.  Element by element against the formulas in 64 bits, with the bounds of that file."""
import numpy as np
import pytest
import torch

from test_group_norm_gpu import HALF, check_stats, make, ops, ref_bwd, ref_fwd, ref_keep, ref_side, ref_stats, within      # noqa: F401

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CASES = [
    ((1, 40, 64, 65, 64, 8), F32), ((1, 40, 64, 65, 64, 8), BF16), ((1, 40, 64, 65, 64, 8), F16),         # 2.6 steps of the forward's passes, 5.3 of the backward's
    ((3, 17, 45, 51, 40, 8), BF16), ((3, 17, 45, 51, 60, 5), F32),                                        # groups that pieces cut
    ((1, 41, 64, 65, 33, 3), F32), ((1, 41, 64, 65, 33, 3), BF16), ((1, 41, 64, 65, 33, 33), F16),        # rows of single elements
    ((1, 17, 16, 17, 512, 256), F32), ((1, 17, 16, 17, 512, 256), BF16),                                  # more than 128 groups in one tile
    ((1, 40, 63, 65, 64, 32), F32), ((1, 40, 63, 65, 64, 32), BF16),                                      # more than 8192 records to a sample
    ((1, 3, 33, 65, 1032, 4), F32), ((2, 2, 17, 31, 4104, 3), BF16),                                      # several tiles
    ((2, 33, 128, 129, 32, 8), F32), ((2, 33, 128, 129, 32, 8), BF16),                                    # twice the workgroups in the backward
    ((5, 37, 64, 65, 32, 4), F16),
]


@pytest.mark.parametrize('size,dtype', CASES)
def test_whole_pass(ops, size, dtype):     # noqa: F811
    G = size[5]
    for act, seed in (('relu', 51), ('silu', 52)):
        x, dy, w, b = make(size, dtype, seed=seed)
        y, mean, rstd, ck = ops.group_norm_act(x, G, w, b, activation=act, checkpoint=True)
        check_stats(x, mean, rstd, G, 1e-5)
        want, err = ref_fwd(x, *ref_stats(x, G, 1e-5), w, b, act)
        within(y, want, err, dtype, f'{act} y')
        y2, mean2, rstd2 = ops.group_norm_act(x, G, w, b, activation=act)
        assert torch.equal(y2, y) and torch.equal(mean2, mean) and torch.equal(rstd2, rstd)
        assert torch.equal(ops.group_norm_act_apply(x, mean, rstd, w, b, activation=act), y)
        del y2, want, err
        q, scale, _ = ref_keep(x)
        q = ref_side(x, q, scale, mean, rstd, w, b, act)
        assert np.array_equal(ck.q.cpu().numpy(), q) and np.array_equal(ck.scale.cpu().numpy(), scale)
        xin = x.clone()
        y3, mean3, _, ck3 = ops.group_norm_act(xin, G, w, b, activation=act, checkpoint=True, out=xin)
        torch.testing.assert_close(mean3, mean, rtol=2 ** -22, atol=1e-7)       # (their sums may have another order)
        torch.testing.assert_close(y3, y, rtol=2 * HALF[dtype] + 1e-5, atol=1e-5)
        assert torch.equal(ck3.scale, ck.scale) and float((ck3.q != ck.q).float().mean()) < 1e-6
        val = torch.from_numpy((q.astype(np.float64) * np.repeat(scale.astype(np.float64), 64)[:q.size]).astype(np.float32)).cuda().reshape(x.shape)
        within(ops.group_norm_act_apply(ck, mean, rstd, w, b, activation=act), *ref_fwd(val, mean, rstd, w, b, act), dtype, f'{act} recomputed y')
        for src, at in ((x, x), (ck, val)):
            got = ops.group_norm_act_bwd(src, mean, rstd, dy, w, b, activation=act)
            want, err = ref_bwd(at, mean, rstd, dy, w, b, act)
            for g, r, e, name in zip(got, want, err, ('dx', 'dweight', 'dbias')):
                within(g, r, e, dtype if name == 'dx' else torch.float32, f'{act} {name}')


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('shape,ldc', [((2, 33, 64, 65, 32), None), ((2, 33, 64, 65, 32), 64), ((1, 21, 65, 67, 33), 40)])
def test_checkpoints_of_several_steps(ops, shape, ldc, dtype):     # noqa: F811
    x, _, _, _ = make((*shape, 1), dtype, seed=61, ldc=ldc)
    ck = ops.checkpoint8(x)
    q, scale, val = ref_keep(x)
    assert np.array_equal(ck.q.cpu().numpy(), q) and np.array_equal(ck.scale.cpu().numpy(), scale)
    want = torch.from_numpy(val).to(dtype).reshape(shape)
    assert torch.equal(ops.checkpoint8_restore(ck).cpu(), want)
    buf = torch.full((*shape[:4], shape[4] + 8), 3.0, dtype=dtype, device='cuda')
    assert torch.equal(ops.checkpoint8_restore(ck, out=buf[..., :shape[4]]).cpu(), want) and bool((buf[..., shape[4]:] == 3).all())
