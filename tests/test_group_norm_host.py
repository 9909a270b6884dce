"""Refusals of the group-norm and 8-bit-checkpoint entry points, without a GPU: the checks of arguments come before any device work, in Python and behind the C ABI."""
import ctypes

import pytest
import torch

from elektronn3_amd import _lib, ops
from elektronn3_amd.norm import GroupNormAct


def call(name, *args):
    return getattr(_lib.load(), name)(*args)


FAKE = ctypes.c_void_p(1 << 20)     # (never dereferenced: every call below is refused on the host)


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(1, 2, 2, 2, 8)
    with pytest.raises(ValueError, match='CUDA'):
        ops.checkpoint8(x)
    with pytest.raises(ValueError, match='CUDA'):
        ops.group_norm_act(x, 2)
    with pytest.raises(ValueError, match='CUDA'):
        ops.group_norm_act_bwd(x, torch.zeros(1, 2), torch.zeros(1, 2), x)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        GroupNormAct(2, 8)(x.movedim(-1, 1))
    with pytest.raises(ValueError, match='Checkpoint8'):
        ops.checkpoint8_restore(x)
    with pytest.raises(ValueError, match='CUDA'):
        ops.Checkpoint8(torch.zeros(64, dtype=torch.int8), torch.zeros(1), (1, 1, 1, 8, 8), torch.float32)


@pytest.mark.parametrize('q,scale,shape,dtype', [
    (torch.zeros(63, dtype=torch.int8), torch.zeros(1), (1, 1, 1, 8, 8), torch.float32),
    (torch.zeros(64, dtype=torch.uint8), torch.zeros(1), (1, 1, 1, 8, 8), torch.float32),
    (torch.zeros(64, dtype=torch.int8), torch.zeros(2), (1, 1, 1, 8, 8), torch.float32),
    (torch.zeros(64, dtype=torch.int8), torch.zeros(1, dtype=torch.float64), (1, 1, 1, 8, 8), torch.float32),
    (torch.zeros(64, dtype=torch.int8), torch.zeros(1), (8, 8), torch.float32),
    (torch.zeros(64, dtype=torch.int8), torch.zeros(1), (1, 1, 1, 8, 8), torch.float64),
    (torch.zeros(128, dtype=torch.int8)[::2], torch.zeros(1), (1, 1, 1, 8, 8), torch.float32),
])
def test_checkpoints_that_do_not_fit_their_tensor(q, scale, shape, dtype):
    with pytest.raises(ValueError, match='Checkpoint8'):
        ops.Checkpoint8(q, scale, shape, dtype)


@pytest.mark.parametrize('act', ['prelu', 'rrelu', 'tanh', torch.nn.PReLU(), torch.nn.RReLU(), torch.nn.Tanh(), torch.nn.LeakyReLU(2.0)])
def test_activations_outside_the_kernels(act):
    with pytest.raises(NotImplementedError):
        ops._act_slope(act)
    with pytest.raises(NotImplementedError):
        GroupNormAct(2, 8, activation=act)


def test_module_arguments():
    with pytest.raises(ValueError):
        GroupNormAct(3, 8)
    m = GroupNormAct(2, 8)
    with pytest.raises(ValueError):
        m(torch.zeros(2, 8))
    with pytest.raises(ValueError):
        m(torch.zeros(2, 4, 3))
    assert 'checkpoint=False' in repr(m)


# the C ABI: (N, D, H, W, C, G) that are no sizes, types, slopes, rows, workspaces
GOOD = (2, 30, 40, 50, 16, 4)        # (large enough to need a workspace)


def fwd(dtype=0, x=FAKE, x_ldc=16, eps=1e-5, slope=0.0, y=FAKE, y_ldc=16, mean=FAKE, q=None, qs=None, dims=GOOD, ws=FAKE, nbytes=0):
    return call('e3_group_norm_act_fwd', None, dtype, x, x_ldc, None, None, eps, slope, y, y_ldc, mean, FAKE, q, qs, *dims, ws, ctypes.c_size_t(nbytes))


@pytest.mark.parametrize('kw,code', [
    (dict(dtype=3), 1), (dict(dtype=-1), 1), (dict(x=None), 1), (dict(y=None), 1), (dict(mean=None), 1), (dict(ws=None, nbytes=1 << 30), 4), (dict(x_ldc=15), 1), (dict(y_ldc=8), 1),
    (dict(eps=-1.0), 1), (dict(eps=float('nan')), 1), (dict(slope=3.0), 3), (dict(slope=-0.5), 3), (dict(slope=float('nan')), 3), (dict(q=FAKE), 1), (dict(qs=FAKE), 1),
    (dict(dims=(2, 3, 4, 5, 16, 3)), 1), (dict(dims=(2, 3, 4, 5, 16, 0)), 1), (dict(dims=(0, 3, 4, 5, 16, 4)), 1), (dict(dims=(2, 0, 4, 5, 16, 4)), 1),
    (dict(dims=(2, 3, 4, 5, 0, 4)), 1), (dict(), 4), (dict(nbytes=64), 4)])
def test_forward_refusals(kw, code):
    assert fwd(**kw) == code
    assert _lib.load().e3_last_error()


def test_backward_and_apply_refusals():
    b = lambda dims=GOOD, x=FAKE, q=None, qs=None, dy=FAKE, dx=FAKE, ldc=16, ws=FAKE, nbytes=0, slope=0.0: call(      # noqa: E731
        'e3_group_norm_act_bwd', None, 0, x, ldc, q, qs, FAKE, FAKE, None, None, slope, dy, 16, dx, 16, FAKE, FAKE, *dims, ws, ctypes.c_size_t(nbytes))
    assert b() == 4 and b(x=None) == 1 and b(x=None, q=FAKE) == 1 and b(dy=None) == 1 and b(dx=None) == 1 and b(ldc=9) == 1 and b(ws=None) == 1 and b(slope=2.5) == 3
    assert b(dims=(1, 1, 1, 1, 16, 5)) == 1
    a = lambda x=FAKE, q=None, qs=None, y=FAKE, ldc=16, dims=GOOD: call(      # noqa: E731
        'e3_group_norm_act_apply', None, 0, x, ldc, q, qs, FAKE, FAKE, None, None, 0.0, y, ldc, *dims)
    assert a(x=None) == 1 and a(y=None) == 1 and a(ldc=4) == 1 and a(dims=(1, 1, 1, 1, 16, 7)) == 1


def test_checkpoint_refusals():
    assert call('e3_checkpoint8_pack', None, 7, FAKE, 8, 4, 8, FAKE, FAKE) == 1
    assert call('e3_checkpoint8_pack', None, 0, None, 8, 4, 8, FAKE, FAKE) == 1
    assert call('e3_checkpoint8_pack', None, 0, FAKE, 7, 4, 8, FAKE, FAKE) == 1
    assert call('e3_checkpoint8_pack', None, 0, FAKE, 8, -1, 8, FAKE, FAKE) == 1
    assert call('e3_checkpoint8_pack', None, 0, FAKE, 8, 4, 0, FAKE, FAKE) == 1
    assert call('e3_checkpoint8_unpack', None, 1, FAKE, None, 4, 8, FAKE, 8) == 1
    assert call('e3_checkpoint8_unpack', None, 1, FAKE, FAKE, 4, 8, FAKE, 2) == 1
    assert call('e3_checkpoint8_pack', None, 0, None, 8, 0, 8, None, None) == 0        # nothing to do


@pytest.mark.parametrize('dims', [GOOD, (1, 1, 1, 1, 8, 1), (3, 17, 45, 51, 20, 5), (2, 64, 128, 128, 32, 8), (1, 1, 1, 1, 8192, 8192), (100000, 1, 1, 1, 8, 8), (1, 2048, 2048, 2048, 8, 8)])
def test_workspace_sizes(dims):
    assert 0 <= call('e3_group_norm_workspace_bytes', *dims, 0) < 1 << 31
    assert 0 <= call('e3_group_norm_workspace_bytes', *dims, 1) < 1 << 31
    assert call('e3_group_norm_workspace_bytes', *dims[:5], dims[5] + dims[4] + 1, 1) == 0
    # small groups need none: the forward, and the backward of one or two samples
    assert call('e3_group_norm_workspace_bytes', 1, 4, 8, 8, 128, 8, 1) == 0 < call('e3_group_norm_workspace_bytes', 3, 4, 8, 8, 128, 8, 1)
    assert call('e3_group_norm_workspace_bytes', 1, 4, 8, 8, 128, 8, 0) == 0 < call('e3_group_norm_workspace_bytes', 1, 64, 64, 64, 128, 8, 0)


def test_workspaces_off_their_alignment():
    odd = ctypes.c_void_p((1 << 20) + 8)
    for backward, name, args in ((0, 'fwd', (None, 0, FAKE, 32, None, None, 1e-5, 0.0, FAKE, 32, FAKE, FAKE, None, None)),
                                 (1, 'bwd', (None, 0, FAKE, 32, None, None, FAKE, FAKE, None, None, 0.0, FAKE, 32, FAKE, 32, FAKE, FAKE))):
        dims = (3, 64, 64, 64, 32, 8)
        need = call('e3_group_norm_workspace_bytes', *dims, backward)
        assert need > 0 and call(f'e3_group_norm_act_{name}', *args, *dims, odd, ctypes.c_size_t(need)) == 1
        assert b'aligned' in _lib.load().e3_last_error()


def test_sums_of_long_samples_are_cut():
    """A thread's fp32 sums of the backward have at most 512 terms: 256 threads to a workgroup, one (sum, sum) record of doubles per workgroup and channel."""
    voxels = 16384 * 16384
    assert call('e3_group_norm_workspace_bytes', 1, 1, 16384, 16384, 1, 1, 1) >= voxels // (512 * 256) * 16
    assert call('e3_group_norm_workspace_bytes', 1, 1, 16384, 16384, 32, 8, 1) >= voxels // (512 * 64) * 32 * 16


def test_rows_and_groups_beyond_the_kernels():
    t = torch.empty(8, device='meta').as_strided((2, 1, 1, 1, 8), (1 << 31, 8, 8, 8, 1))
    with pytest.raises(ValueError, match='rows of'):
        ops._ldc(t)
    lib = _lib.load()
    rc = lib.e3_group_norm_act_fwd(None, 0, FAKE, 32, None, None, 1e-5, 0.0, FAKE, 32, FAKE, FAKE, None, None, 1 << 20, 1, 1, 1, 32, 8, None, 0)
    assert rc == 3 and b'groups' in lib.e3_last_error()
