"""Calls at the limits of the group-norm and 8-bit-checkpoint entry points, without a GPU: tensors without memory (device 'meta') that pass for ones on a GPU."""
import pytest
import torch

from elektronn3_amd import ops

LONG = 1 << 32          # the C ABI's axes are 32-bit integers: one of LONG + n elements would be taken for one of n


class OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


def fake(shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device='meta').as_subclass(OnGpu)


@pytest.mark.parametrize('n', [1 << 31, LONG - 8, LONG, LONG + 40000])
@pytest.mark.parametrize('axis', range(4))
def test_axes_that_do_not_fit_the_c_abi(monkeypatch, axis, n):
    shape = [1, 1, 1, 1, 8]
    shape[axis] = n
    x = fake(shape)
    vec = torch.zeros(1, 2)
    monkeypatch.setattr(ops, '_call', lambda *a: pytest.fail('reached the library'))
    with pytest.raises(ValueError, match='2\\^31'):
        ops.group_norm_act(x, 2)
    monkeypatch.setattr(ops, '_stats', lambda *a: (vec, vec, 2))
    with pytest.raises(ValueError, match='2\\^31'):
        ops.group_norm_act_apply(x, vec, vec)
    with pytest.raises(ValueError, match='2\\^31'):
        ops.group_norm_act_bwd(x, vec, vec, x)


@pytest.mark.parametrize('n', [1 << 31, LONG, LONG + 5])
def test_channels_that_do_not_fit_the_c_abi(monkeypatch, n):
    monkeypatch.setattr(ops, '_call', lambda *a: pytest.fail('reached the library'))
    x = fake((1, 1, 1, 1, n))
    with pytest.raises(ValueError, match='longer than the kernels address'):
        ops.checkpoint8(x)
    with pytest.raises(ValueError, match='longer than the kernels address'):
        ops.group_norm_act(x, 1)
    with pytest.raises(ValueError, match='longer than the kernels address'):
        ops.Checkpoint8(fake((n,), torch.int8), fake((-(-n // 64),), torch.float32), (1, 1, 1, 1, n), torch.bfloat16)


def test_long_axes_that_the_checkpoints_take(monkeypatch):
    """Their voxels are counted in 64 bits: any axis but the channels may be long."""
    seen = []
    monkeypatch.setattr(ops, '_call', lambda device, fn, *args: seen.append(args))
    monkeypatch.setattr(ops, '_new_checkpoint', lambda x: ops.Checkpoint8(fake((x.numel(),), torch.int8), fake((-(-x.numel() // 64),), torch.float32), x.shape, x.dtype))
    x = fake((1, 1, 1, LONG + 40000, 2))
    ck = ops.checkpoint8(x)
    assert seen[-1][3:5] == (LONG + 40000, 2) and ck.shape == x.shape
    ops.checkpoint8_restore(ck, out=x)
    assert seen[-1][3:5] == (LONG + 40000, 2)
