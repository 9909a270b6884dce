"""Which group norms run in one launch, told by the size of the workspace that they ask for (none).  Groups narrower than a 128-byte line move every line once per group in it: with many
samples or channels two launches read less, however few voxels a group has.  No GPU."""
import pytest

from elektronn3_amd import _lib


def need(N, D, H, W, C, G, backward=0):
    return _lib.load().e3_group_norm_workspace_bytes(N, D, H, W, C, G, backward)


@pytest.mark.parametrize('dims', [
    (64, 8, 8, 8, 512, 64),         # many samples of 16-byte groups
    (1000, 4, 8, 8, 32, 8),         # groups of 4 channels
    (8, 16, 16, 16, 256, 256),      # instance norm: one 16-bit element of a 128-byte line
    (4, 16, 16, 16, 128, 128),
    (600, 3, 5, 7, 96, 8),          # groups of 12 channels
    (256, 5, 7, 9, 33, 33),
])
def test_forwards_in_two_launches(dims):
    assert need(*dims) > 0


@pytest.mark.parametrize('dims', [
    (1, 4, 8, 8, 128, 8), (4, 1, 5, 7, 24, 3), (1, 16, 16, 16, 8, 8), (1, 16, 16, 16, 64, 64), (16, 3, 5, 7, 1200, 100), (64, 8, 8, 8, 64, 8), (100, 5, 7, 9, 60, 5),
    (1024, 1, 7, 9, 512, 8),        # whole lines: no limit
])
def test_forwards_in_one_launch(dims):
    assert need(*dims) == 0


def test_backwards_element_by_element():
    """One-channel groups of more voxels than 16-byte pieces of 16-bit types can hold: one launch for one sample only."""
    assert need(1, 16, 16, 16, 64, 64, 1) == 0 < need(2, 16, 16, 16, 64, 64, 1)
    assert need(2, 13, 17, 12, 128, 128, 1) > 0
    assert need(2, 5, 7, 9, 24, 2, 1) == 0         # (groups of 12 in pieces of 8)
