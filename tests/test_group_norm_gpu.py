"""Group norm with activation, its gradients and the 8-bit activation checkpoints (elektronn3_amd/ops.py, elektronn3_amd/norm.py) against plain formulas in 64
bits, element by element.  The tolerances count roundings (u = 2^-24, half a step of fp32; `half` the same of the stored type):

  z       x - mean, rstd * weight, the product and the sum are one rounding each, mean and rstd one each: 8 u |p| + 2 u |mean rstd weight| + 2 u |z|, p = z - bias
  act     slope <= 1.1; SiLU: exp2's argument is rounded (u |z| 1.45), exp2 and rcp are good to 1 ulp (4 u): 1.1 * err(z) + u (2 |z| + 8) |y|
  sums    a thread adds at most 512 terms in fp32 before they go on in fp64: (512 + 12) u * sum |term|; terms' own errors are inside the 12
  storage half |y|, and half of the smallest step near 0
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -9 * 2, torch.float16: 2.0 ** -11}     # eps / 2 (bf16: 2^-8)
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # smallest step
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SLOPE = {'relu': 0.0, 'leaky': 0.1, 'lin': 1.0}

# N, D, H, W, C, G
SIZES = [
    (1, 1, 1, 1, 8, 1),            # one voxel
    (2, 1, 1, 1, 8, 8),            # one element per group: variance 0
    (1, 1, 1, 3, 1, 1),            # one channel
    (2, 3, 5, 7, 24, 3),
    (3, 2, 4, 4, 20, 5),           # channels no multiple of 8
    (1, 4, 8, 8, 256, 32),
    (2, 5, 9, 13, 40, 8),          # groups of 5 channels in pieces of 8
    (2, 3, 7, 9, 48, 4),           # groups of 12
    (1, 1, 7, 9, 33, 1),
    (1, 3, 5, 11, 32, 32),         # instance norm
    (1, 2, 3, 5, 1032, 4),
    (2, 1, 3, 3, 4104, 3),         # more pieces than a workgroup has threads; groups across its tiles
    (1, 1, 2, 5, 1001, 7),
    (2, 16, 32, 32, 32, 8),
    (1, 13, 47, 51, 16, 2),
    (4, 1, 65, 33, 64, 8),         # a 2D batch
    (3000, 1, 1, 2, 8, 2),         # many samples
]


@pytest.fixture(scope='module')
def ops():
    from elektronn3_amd import ops as o
    return o


def make(size, dtype, seed=0, ldc=None, shift=0.5):
    N, D, H, W, C, G = size
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)    # noqa: E731
    wide = r(N, D, H, W, ldc or C) * (0.3 * r(ldc or C)).exp() + shift * r(ldc or C)
    x = wide.to(dtype).cuda()[..., :C]
    dy = (0.1 * r(N, D, H, W, C)).to(dtype).cuda()
    w, b = (1 + 0.3 * r(C)).float().cuda(), (0.3 * r(C)).float().cuda()
    return x, dy, w, b


def grouped(t, G):
    return t.reshape(t.shape[0], -1, G, t.shape[-1] // G)


def spread(m, C):
    return m.repeat_interleave(C // m.shape[1], 1)[:, None, None, None, :]


def ref_stats(x, G, eps):
    g = grouped(x.double(), G)
    return g.mean((1, 3)), 1 / (g.var((1, 3), unbiased=False) + eps).sqrt()


def ref_act(z, act):
    return z * torch.sigmoid(z) if act == 'silu' else torch.where(z > 0, z, SLOPE[act] * z)


def ref_fwd(x, mean, rstd, w, b, act):
    """y and the bound of a kernel's error, without the storage rounding (mean, rstd: 64-bit values, or the fp32 ones it was given)"""
    C = x.shape[-1]
    mu, rs = spread(mean.double(), C), spread(rstd.double(), C)
    a = rs * w.double()
    p = (x.double() - mu) * a
    z = p + b.double()
    y = ref_act(z, act)
    err = U * (8 * p.abs() + 2 * (mu * a).abs() + 2 * z.abs())
    return y, 1.1 * err + (U * (2 * z.abs() + 8) * y.abs() if act == 'silu' else 0)


def ref_bwd(x, mean, rstd, dy, w, b, act):
    C, G = x.shape[-1], mean.shape[1]
    mu, rs = spread(mean.double(), C), spread(rstd.double(), C)
    g = dy.double()
    h = (x.double() - mu) * rs
    z = h * w.double() + b.double()
    if act == 'silu':
        s = torch.sigmoid(z)
        d = s * (1 + z * (1 - s))
        derr = U * (4 * z.abs() + 24)               # of the derivative (at most 1.1 in size), from z's error and the operations
        derr = derr + 2 * U * (8 * (h * w).abs())
    else:
        d, derr = torch.where(z > 0, 1.0, SLOPE[act]).double(), torch.zeros_like(z)
    dz, dzerr = g * d, g.abs() * derr
    u = dz * w.double()
    m1, m2 = grouped(u, G).mean((1, 3)), grouped(u * h, G).mean((1, 3))
    dx = rs * (u - spread(m1, C) - h * spread(m2, C))
    K = 512 + 12
    a1 = spread(grouped(u.abs(), G).mean((1, 3)), C)
    a2 = spread(grouped((u * h).abs(), G).mean((1, 3)), C)
    e1 = spread(grouped((dzerr * w).abs(), G).mean((1, 3)), C)
    e2 = spread(grouped((dzerr * w * h).abs(), G).mean((1, 3)), C)
    dxerr = rs * (U * (8 * u.abs() + K * a1 + h.abs() * (K + 8) * a2) + (dzerr * w).abs() + e1 + h.abs() * e2)
    over = (0, 1, 2, 3)
    dw, db = (dz * h).sum(over), dz.sum(over)
    dwerr = (K * U * (dz * h).abs() + (dzerr * h).abs()).sum(over)
    dberr = (K * U * dz.abs() + dzerr).sum(over)
    return (dx, dw, db), (dxerr, dwerr, dberr)


def within(got, want, err, dtype, what):
    bound = err + HALF[dtype] * (want.abs() + err) + TINY[dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.3g} of the bound'


def check_stats(x, mean, rstd, G, eps):
    m, r = ref_stats(x, G, eps)
    within(mean, m, torch.zeros_like(m), torch.float32, 'mean')
    # fp64 sums of n terms: var is off by n 2^-53 (var + mean^2), at most; one fp32 rounding of the result
    n = x.numel() / mean.numel()
    var = 1 / r ** 2
    within(rstd, r, r * (n * 2.0 ** -53 * (var + m ** 2) / var), torch.float32, 'rstd')


# ------------------------------------------------------------------------------------------------ forward
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', SIZES)
def test_forward(ops, size, dtype):
    for i, act in enumerate(['relu', 'leaky', 'lin', 'silu']):
        x, _, w, b = make(size, dtype, seed=i)
        y, mean, rstd = ops.group_norm_act(x, size[5], w, b, activation=act)
        assert y.dtype == dtype and y.shape == x.shape and mean.shape == rstd.shape == (size[0], size[5])
        check_stats(x, mean, rstd, size[5], 1e-5)
        want, err = ref_fwd(x, *ref_stats(x, size[5], 1e-5), w, b, act)
        within(y, want, err, dtype, act)
        again = ops.group_norm_act_apply(x, mean, rstd, w, b, activation=act)
        assert torch.equal(again, y)


@pytest.mark.parametrize('dtype', DTYPES)
def test_forward_without_parameters_other_eps_and_modules(ops, dtype):
    size = (2, 3, 6, 7, 24, 3)
    x, _, w, b = make(size, dtype)
    one, zero = torch.ones_like(w), torch.zeros_like(w)
    for act, mod in (('relu', torch.nn.ReLU()), ('leaky', torch.nn.LeakyReLU(0.1)), ('silu', torch.nn.SiLU()), ('lin', torch.nn.Identity())):
        y, mean, rstd = ops.group_norm_act(x, 3, eps=0.5, activation=mod)
        want, err = ref_fwd(x, *ref_stats(x, 3, 0.5), one, zero, act)
        within(y, want, err, dtype, act)
        y2, _, _ = ops.group_norm_act(x, 3, one, zero, eps=0.5, activation=act)
        assert torch.equal(y, y2)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('C,G,ldc', [(32, 8, 64), (24, 4, 32), (24, 4, 25), (7, 7, 10), (8, 2, 12)])
def test_views(ops, dtype, C, G, ldc):
    """Halves of a concat buffer, rows that are no multiple of 16 bytes, outputs into a view; what lies between the rows stays."""
    size = (2, 3, 5, 6, C, G)
    x, dy, w, b = make(size, dtype, ldc=ldc)
    buf = torch.full((2, 3, 5, 6, ldc + 8), 7.0, dtype=dtype, device='cuda')
    out = buf[..., 8:8 + C]
    y, mean, rstd = ops.group_norm_act(x, G, w, b, activation='leaky', out=out)
    assert y.data_ptr() == out.data_ptr()
    want, err = ref_fwd(x, *ref_stats(x, G, 1e-5), w, b, 'leaky')
    within(out, want, err, dtype, 'y')
    assert bool((buf[..., :8] == 7).all()) and bool((buf[..., 8 + C:] == 7).all())
    wide = torch.full((2, 3, 5, 6, ldc), 9.0, dtype=dtype, device='cuda')
    wide[..., :C] = dy
    got = ops.group_norm_act_bwd(x, mean, rstd, wide[..., :C], w, b, activation='leaky')
    for g, r in zip(got, ops.group_norm_act_bwd(x.contiguous(), mean, rstd, dy, w, b, activation='leaky')):
        torch.testing.assert_close(g, r, rtol=2e-5 if dtype == torch.float32 else 2 * HALF[dtype] + 2e-5, atol=1e-5)
    # in place
    xin = x.contiguous().clone()
    yin, _, _ = ops.group_norm_act(xin, G, w, b, activation='leaky', out=xin)
    torch.testing.assert_close(yin, y, rtol=2 * HALF[dtype] + 2e-6, atol=1e-5)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', [(2, 5, 9, 13, 32, 4), (1, 3, 4, 5, 16, 2)])
def test_addresses_that_are_no_multiple_of_16(ops, size, dtype):
    """Every tensor one element, every checkpoint three codes behind such an address: the results of aligned copies, up to the order of their sums."""
    C, G = size[4:]
    x, dy, w, b = make(size, dtype, seed=31)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)       # noqa: E731
    x1, dy1, y1 = off(x), off(dy), off(torch.zeros_like(x))
    assert x1.data_ptr() % 16 and x1.is_contiguous()
    y, mean, rstd, ck = ops.group_norm_act(x, G, w, b, checkpoint=True)
    _, mean1, rstd1, ck1 = ops.group_norm_act(x1, G, off(w), off(b), checkpoint=True, out=y1)
    torch.testing.assert_close(mean1, mean, rtol=2 ** -22, atol=1e-7)
    torch.testing.assert_close(rstd1, rstd, rtol=2 ** -22, atol=0)
    torch.testing.assert_close(y1, y, rtol=2 * HALF[dtype] + 2e-6, atol=1e-5)
    assert torch.equal(ck1.scale, ck.scale)
    q3 = torch.cat([ck.q.new_zeros(3), ck.q])[3:]
    ck3 = ops.Checkpoint8(q3, off(ck.scale), x.shape, dtype)
    assert torch.equal(ops.checkpoint8_restore(ck3, out=off(torch.zeros_like(x))), ops.checkpoint8_restore(ck))
    torch.testing.assert_close(ops.group_norm_act_apply(ck3, mean, rstd, w, b), ops.group_norm_act_apply(ck, mean, rstd, w, b), rtol=2 * HALF[dtype] + 2e-6, atol=1e-6)
    for src, at in ((x1, x), (ck3, ck)):
        for g, r in zip(ops.group_norm_act_bwd(src, off(mean), off(rstd), dy1, w, b), ops.group_norm_act_bwd(at, mean, rstd, dy, w, b)):
            torch.testing.assert_close(g, r, rtol=2e-5 if g.dtype == torch.float32 else 2 * HALF[dtype] + 2e-5, atol=1e-5)


def test_large_offset(ops):
    """mean / std = 3000: a variance from fp32 sums of squares would be noise."""
    x, dy, w, b = make((2, 6, 12, 10, 16, 2), torch.float32)
    x = x + 3000
    y, mean, rstd = ops.group_norm_act(x, 2, w, b, activation='silu')
    check_stats(x, mean, rstd, 2, 1e-5)
    want, err = ref_fwd(x, *ref_stats(x, 2, 1e-5), w, b, 'silu')
    within(y, want, err, torch.float32, 'y')


@pytest.mark.parametrize('act', ['relu', 'leaky', 'lin', 'silu'])
def test_extreme_preactivations(ops, act):
    """z far out on both sides: no overflow of the exponential turns into a NaN."""
    x, dy, _, _ = make((1, 2, 4, 4, 8, 1), torch.float32)
    w = torch.tensor([1e4, -1e4, 1e30, -1e30, 0.0, 1.0, 100.0, -100.0], device='cuda')
    b = torch.tensor([0.0, 0, 0, 0, -200.0, 200.0, 0, 0], device='cuda')
    y, mean, rstd = ops.group_norm_act(x, 1, w, b, activation=act)
    assert bool(torch.isfinite(y).all())
    want, err = ref_fwd(x, *ref_stats(x, 1, 1e-5), w, b, act)
    within(y, want, err + 2.0 ** -119, torch.float32, 'y')          # (a sigmoid below the normal range, 2^-126, may be 0: |z| < 128 there)


def test_nan_and_infinity_stay_in_their_sample(ops):
    x, dy, w, b = make((3, 2, 4, 4, 16, 2), torch.float32)
    x[1, 0, 1, 2, 3] = float('nan')
    x[2, 1, 0, 0, 12] = float('inf')
    y, mean, rstd = ops.group_norm_act(x, 2, w, b)
    nan = torch.isnan(y)
    assert not nan[0].any() and nan[1, ..., :8].all() and not nan[1, ..., 8:].any() and not nan[2, ..., :8].any() and nan[2, ..., 8:].all()
    clean = x.clone(); clean[1:] = 0
    assert torch.equal(ops.group_norm_act(clean, 2, w, b)[0][0], y[0])


# ------------------------------------------------------------------------------------------------ backward
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', SIZES)
def test_backward(ops, size, dtype):
    for i, act in enumerate(['relu', 'leaky', 'lin', 'silu']):
        x, dy, w, b = make(size, dtype, seed=10 + i)
        mean, rstd = (t.float() for t in ref_stats(x, size[5], 1e-5))
        got = ops.group_norm_act_bwd(x, mean, rstd, dy, w, b, activation=act)
        want, err = ref_bwd(x, mean, rstd, dy, w, b, act)
        for g, r, e, name in zip(got, want, err, ('dx', 'dweight', 'dbias')):
            assert g.dtype == (dtype if name == 'dx' else torch.float32)
            within(g, r, e, dtype if name == 'dx' else torch.float32, f'{act} {name}')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', [
    (1, 2, 16, 32, 8, 1),          # 8192 elements to a group: the largest that one workgroup takes
    (1, 1, 25, 41, 8, 1),          # 8200
    (2, 1, 16, 32, 8, 1),          # 8192 in two samples
    (2, 1, 19, 27, 8, 1),          # 8208
    (1, 1, 1, 16, 512, 1),         # the widest bundle
    (2, 1, 1, 2, 520, 1),          # wider
    (1, 1, 3, 5, 96, 48),          # groups of 2, 4 channels in pieces of 4 and 8
    (2, 1, 7, 3, 64, 16),
    (2, 3, 4, 5, 24, 24),
    (2, 1, 9, 7, 60, 5),           # groups of 12
    (1, 1, 64, 63, 1, 1),          # single channels
])
def test_backward_of_small_groups(ops, size, dtype):
    N, D, H, W, C, G = size
    for act, ldc in (('relu', C), ('silu', C + 8), ('leaky', C + 3)):
        x, dy, w, b = make(size, dtype, seed=21, ldc=ldc)
        _, mean, rstd, ck = ops.group_norm_act(x, G, w, b, activation=act, checkpoint=True)
        val = (ck.q.cpu().float() * ck.scale.cpu().repeat_interleave(64)[:ck.q.numel()]).view(x.shape).cuda()       # (fp32 product: the checkpoint's values)
        for src, at in ((x, x), (ck, val)):
            got = ops.group_norm_act_bwd(src, mean, rstd, dy, w, b, activation=act)
            want, err = ref_bwd(at, mean, rstd, dy, w, b, act)
            for g, r, e, name in zip(got, want, err, ('dx', 'dweight', 'dbias')):
                within(g, r, e, dtype if name == 'dx' else torch.float32, f'{act} {name}')


def test_backward_against_differences(ops):
    size = (2, 2, 3, 4, 16, 4)
    x, dy, w, b = make(size, torch.float32, seed=3)
    for act in ('silu', 'lin'):
        f = lambda x, w, b: (ref_act(((x - spread(ref_stats(x, 4, 1e-5)[0], 16)) * spread(ref_stats(x, 4, 1e-5)[1], 16)) * w + b, act) * dy.double()).sum()    # noqa: E731
        _, mean, rstd = ops.group_norm_act(x, 4, w, b, activation=act)
        got = ops.group_norm_act_bwd(x, mean, rstd, dy, w, b, activation=act)
        args = [t.double() for t in (x, w, b)]
        g = torch.Generator().manual_seed(1)
        for k in range(3):
            d = torch.randn(args[k].shape, generator=g, dtype=torch.float64).cuda()
            h = 1e-5
            up, dn = list(args), list(args)
            up[k], dn[k] = args[k] + h * d, args[k] - h * d
            num = float((f(*up) - f(*dn)) / (2 * h))
            ana = float((got[k].double() * d).sum())
            # central differences in 64 bits: h^2 and 1e-16 / h relative; the fp32 gradient's own error
            assert abs(num - ana) <= 1e-6 * float((got[k].double() * d).abs().sum()) + 1e-8, (act, k, num, ana)


def test_relu_border_is_decided_as_in_exact_arithmetic(ops):
    """Pre-activations within rounding of 0: the mask is that of the 64-bit formula on the given fp32 statistics."""
    g = torch.Generator().manual_seed(5)
    C, n = 8, 4096
    mean = torch.tensor([[0.3123457]]).cuda()
    rstd = torch.tensor([[1.7320509]]).cuda()
    w = (1 + torch.rand(C, generator=g)).cuda()
    b = torch.randn(C, generator=g).cuda()
    zero_at = mean.double() - b.double() / (rstd.double() * w.double())
    x = zero_at.float() + (torch.randint(-8, 9, (n, C), generator=g).cuda() * zero_at.abs() * 2.0 ** -24).float()
    x = x.reshape(1, 1, 64, 64, C)
    dy = torch.ones_like(x)
    pos = (x.double() - mean.double()) * rstd.double() * w.double() + b.double() > 0
    got = ops.group_norm_act_bwd(x, mean, rstd, dy, w, b, activation='relu')
    assert torch.equal(got[2].double(), pos.double().sum((0, 1, 2, 3)))


def test_backward_sums_over_samples_and_is_repeatable(ops):
    x, dy, w, b = make((5, 4, 9, 11, 64, 8), torch.bfloat16)
    _, mean, rstd = ops.group_norm_act(x, 8, w, b)
    first = ops.group_norm_act_bwd(x, mean, rstd, dy, w, b)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, ops.group_norm_act_bwd(x, mean, rstd, dy, w, b)))
    parts = [ops.group_norm_act_bwd(x[n:n + 1], mean[n:n + 1], rstd[n:n + 1], dy[n:n + 1], w, b) for n in range(5)]
    torch.testing.assert_close(torch.cat([p[0] for p in parts]), first[0], rtol=2 ** -7, atol=1e-5)
    torch.testing.assert_close(sum(p[1] for p in parts), first[1], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(sum(p[2] for p in parts), first[2], rtol=1e-5, atol=1e-5)


# ------------------------------------------------------------------------------------------------ 8-bit checkpoints
def ref_keep(x):
    """Codes, scales and values by the definition, on the CPU: operations in 64 bits rounded to fp32."""
    v = x.detach().cpu().float().reshape(-1).numpy()
    n = v.size
    p = np.zeros(-(-n // 64) * 64, np.float32)
    p[:n] = v
    p = p.reshape(-1, 64)
    with np.errstate(all='ignore'):
        amax = np.abs(p).max(1)
        none, bad = amax < 2.0 ** -110, ~np.isfinite(amax)
        ok = ~none & ~bad
        inv = np.where(ok, (127.0 / np.where(ok, amax, 1).astype(np.float64)).astype(np.float32), np.float32(0))
        q = np.where(ok[:, None], np.rint((p.astype(np.float64) * inv[:, None].astype(np.float64)).astype(np.float32)), 0).astype(np.int8)
        scale = np.where(bad, np.float32(np.nan), np.where(none, np.float32(0), (amax.astype(np.float64) * np.float64(np.float32(1 / 127))).astype(np.float32)))
        val = (q.astype(np.float64) * scale[:, None].astype(np.float64)).astype(np.float32)
    return q.reshape(-1)[:n], scale, val.reshape(-1)[:n]


def ref_side(x, q, scale, mean, rstd, w, b, act):
    """The codes of a norm's input: where an element and its rounded value lie on different sides of a ReLU's border (64 bits), the element's other neighbour."""
    if act in ('silu', 'lin'):
        return q
    C = x.shape[-1]
    v = torch.from_numpy((q.astype(np.float64) * np.repeat(scale.astype(np.float64), 64)[:q.size]).astype(np.float32)).cuda().reshape(x.shape)
    z = lambda t: (t.double() - spread(mean.double(), C)) * spread(rstd.double(), C) * w.double() + b.double()    # noqa: E731
    move = (z(x) > 0) != (z(v) > 0)
    step = torch.where(x.float() > v, 1, -1) * move
    out = q.astype(np.int64) + step.reshape(-1).cpu().numpy()
    return np.where(np.repeat(scale > 0, 64)[:q.size], np.clip(out, -127, 127), q).astype(np.int8)


KEEP = [((1, 1, 1, 1, 1), None), ((1, 1, 1, 7, 9), None), ((2, 3, 5, 7, 24), None), ((2, 3, 5, 7, 24), 40), ((1, 4, 4, 4, 64), None), ((1, 2, 3, 5, 33), 50),
        ((2, 2, 9, 8, 32), 64), ((1, 1, 130, 129, 16), None), ((3, 1, 1, 1, 200), 203)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape,ldc', KEEP)
def test_checkpoint_bits(ops, shape, ldc, dtype):
    x, _, _, _ = make((*shape, 1), dtype, ldc=ldc)
    ck = ops.checkpoint8(x)
    q, scale, val = ref_keep(x)
    assert ck.shape == x.shape and ck.dtype == dtype and ck.nbytes == q.size + 4 * scale.size
    assert np.array_equal(ck.q.cpu().numpy(), q) and np.array_equal(ck.scale.cpu().numpy(), scale)
    back = ops.checkpoint8_restore(ck)
    assert back.dtype == dtype and torch.equal(back.cpu().reshape(-1), torch.from_numpy(val).to(dtype))
    # half a step of the block's largest magnitude, plus the roundings of 127 / amax, the product and the scale (127 steps off by 3 u each), and the storage
    amax = torch.nn.functional.pad(x.detach().double().reshape(-1), (0, -x.numel() % 64)).reshape(-1, 64).abs().amax(1).repeat_interleave(64)[:x.numel()]
    off = (back.double() - x.double()).abs().reshape(-1)
    assert bool((off <= amax * (0.5 / 127 + 6 * U) + HALF[dtype] * amax).all())
    buf = torch.full((*shape[:4], shape[4] + 5), 3.0, dtype=dtype, device='cuda')
    out = ops.checkpoint8_restore(ck, out=buf[..., 2:2 + shape[4]])
    assert torch.equal(out, back) and bool((buf[..., :2] == 3).all()) and bool((buf[..., 2 + shape[4]:] == 3).all())


@pytest.mark.parametrize('dtype', DTYPES)
def test_checkpoint_special_blocks(ops, dtype):
    """Zeros, values that underflow, the type's largest values, infinities and NaNs; a bad block leaves its neighbours alone."""
    x = torch.randn(1, 1, 1, 8, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    x[0, 0, 0, 0] = 0
    x[0, 0, 0, 1] *= 2.0 ** -125 if dtype != torch.float16 else 2.0 ** -24
    x[0, 0, 0, 2, 5] = float('inf')
    x[0, 0, 0, 3, 63] = float('nan')
    x[0, 0, 0, 4, 0] = -float('inf')
    x[0, 0, 0, 5] = torch.finfo(dtype).max
    x[0, 0, 0, 6] = -torch.finfo(dtype).max
    q, scale, val = ref_keep(x)
    ck = ops.checkpoint8(x.cuda())
    assert np.array_equal(ck.q.cpu().numpy(), q) and np.array_equal(ck.scale.cpu().numpy(), scale, equal_nan=True)
    back = ops.checkpoint8_restore(ck).cpu().reshape(8, 64)
    assert torch.equal(torch.isnan(back).all(1), torch.tensor([False, False, True, True, True, False, False, False])) and not torch.isnan(back[[0, 1, 5, 6, 7]]).any()
    assert bool((back[0] == 0).all()) and torch.isfinite(back[[0, 1, 7]]).all()
    torch.testing.assert_close(back.nan_to_num(0, posinf=1e38, neginf=-1e38), torch.from_numpy(val).to(dtype).reshape(8, 64).nan_to_num(0, posinf=1e38, neginf=-1e38), rtol=0, atol=0)


def test_checkpoint_of_nothing(ops):
    ck = ops.checkpoint8(torch.empty(2, 0, 3, 4, 8, device='cuda'))
    assert ck.nbytes == 0 and ops.checkpoint8_restore(ck).shape == (2, 0, 3, 4, 8)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('size', SIZES)
def test_forward_with_checkpoint_and_backward_from_it(ops, size, dtype):
    """The checkpoint that the forward writes along is that of checkpoint8 with its codes on their elements' side of a ReLU's border; the passes from it are those
    from the values it stands for, and take the forward's branch everywhere."""
    for i, act in enumerate(['relu', 'silu', 'leaky', 'lin']):
        x, dy, w, b = make(size, dtype, seed=20 + i)
        y, mean, rstd, ck = ops.group_norm_act(x, size[5], w, b, activation=act, checkpoint=True)
        y2, mean2, rstd2 = ops.group_norm_act(x, size[5], w, b, activation=act)
        assert torch.equal(y, y2) and torch.equal(mean, mean2) and torch.equal(rstd, rstd2)
        q, scale, _ = ref_keep(x)
        q = ref_side(x, q, scale, mean, rstd, w, b, act)
        val = (q.astype(np.float64) * np.repeat(scale.astype(np.float64), 64)[:q.size]).astype(np.float32)
        assert np.array_equal(ck.q.cpu().numpy(), q) and np.array_equal(ck.scale.cpu().numpy(), scale)
        if act == 'relu' and scale.min() > 0:
            ones = torch.ones_like(dy)
            assert torch.equal(ops.group_norm_act_bwd(ck, mean, rstd, ones, w, b)[2], ops.group_norm_act_bwd(x, mean, rstd, ones, w, b)[2])
        xin = x.clone()                                               # in place
        y3, mean3, _, ck3 = ops.group_norm_act(xin, size[5], w, b, activation=act, checkpoint=True, out=xin)
        assert y3 is xin and torch.equal(ck3.q, ck.q) and torch.equal(ck3.scale, ck.scale)
        torch.testing.assert_close(mean3, mean, rtol=2 ** -22, atol=1e-7)
        torch.testing.assert_close(y3, y, rtol=2 * HALF[dtype] + 1e-5, atol=1e-5)
        xt = torch.from_numpy(val).cuda().reshape(x.shape)            # fp32, whatever the type
        again = ops.group_norm_act_apply(ck, mean, rstd, w, b, activation=act)
        want, err = ref_fwd(xt, mean, rstd, w, b, act)
        within(again, want, err, dtype, 'recomputed y')
        got = ops.group_norm_act_bwd(ck, mean, rstd, dy, w, b, activation=act)
        want, err = ref_bwd(xt, mean, rstd, dy, w, b, act)
        for g, r, e, name in zip(got, want, err, ('dx', 'dweight', 'dbias')):
            within(g, r, e, dtype if name == 'dx' else torch.float32, f'{act} {name}')


# ------------------------------------------------------------------------------------------------ streams, graphs, threads
def test_other_stream_and_two_graphs_replayed(ops):
    """A block's whole pass on a side stream and captured twice; the replays, in turn with eager work, give the eager results."""
    cases = []
    for k, size in enumerate([(2, 4, 9, 8, 32, 8), (1, 8, 16, 16, 64, 8)]):
        x, dy, w, b = make(size, torch.bfloat16, seed=k)

        def step(x=x, dy=dy, w=w, b=b, G=size[5]):
            y, mean, rstd, ck = ops.group_norm_act(x, G, w, b, activation='silu', checkpoint=True)
            return (y, ops.group_norm_act_apply(ck, mean, rstd, w, b, activation='silu'), *ops.group_norm_act_bwd(ck, mean, rstd, dy, w, b, activation='silu'),
                    ops.checkpoint8_restore(ck))
        cases.append((x, dy, step, make(size, torch.bfloat16, seed=50 + k)))
    side = torch.cuda.Stream()
    graphs = []
    for x, dy, step, _ in cases:
        want = step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for rep in range(4):
        for (x, dy, step, fresh), (g, outs) in zip(cases, graphs):
            x.copy_(fresh[0] * (1 + rep)); dy.copy_(fresh[1])
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (x, dy, step, fresh), (g, outs) in zip(cases, graphs):
            assert all(torch.equal(p, q) for p, q in zip(outs, step())), rep


def test_two_calls_at_once(ops):
    """Two threads, each on a stream of its own, each with its own workspaces: the results of one after the other."""
    import threading
    data = [make((2, 6, 16, 17, 64, 8), torch.float16, seed=70 + k) for k in range(2)]

    def step(d):
        x, dy, w, b = d
        y, mean, rstd, ck = ops.group_norm_act(x, 8, w, b, checkpoint=True)
        return (y, *ops.group_norm_act_bwd(ck, mean, rstd, dy, w, b), ops.checkpoint8_restore(ck))
    want = [step(d) for d in data]
    torch.cuda.synchronize()
    got = [None, None]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k] = step(data[k])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, r in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, r))


def test_offsets_past_32_bits(ops):
    """A batch of 4.3e9 elements: its last sample, whose offsets do not fit 32 bits, gives what it gives alone."""
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip('needs 100 GB')
    shape = (2, 1, 8200, 8200, 32)
    x = torch.empty(shape, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(1)
    tile = torch.randn(8200, 32, device='cuda', generator=g) + 0.5
    for n in range(2):                       # rows of one tile, scaled: every row of every sample is different
        x[n, 0] = (tile[None] * torch.linspace(0.5 + n, 1.5 + n, 8200, device='cuda')[:, None, None]).to(torch.bfloat16)
    w, b = torch.ones(32, device='cuda'), torch.full((32,), 0.1, device='cuda')
    y, mean, rstd, ck = ops.group_norm_act(x, 8, w, b, checkpoint=True)
    y1, mean1, rstd1, ck1 = ops.group_norm_act(x[1:], 8, w, b, checkpoint=True)
    torch.testing.assert_close(mean[1:], mean1, rtol=2 ** -22, atol=0)
    torch.testing.assert_close(y[1:, :, -3:], y1[:, :, -3:], rtol=2 ** -7, atol=1e-5)
    n = x[0].numel()
    assert torch.equal(ck.scale[n // 64:], ck1.scale) and float((ck.q[n:] != ck1.q).float().mean()) < 1e-6      # (codes at the border go by the statistics' last bit)
    back = ops.checkpoint8_restore(ck)
    assert torch.equal(back[1:, :, -3:], ops.checkpoint8_restore(ops.Checkpoint8(ck.q[n:], ck.scale[n // 64:], x[1:].shape, x.dtype))[:, :, -3:])
    del back, y, y1
    dx, _, _ = ops.group_norm_act_bwd(ck, mean, rstd, x, w, b)
    dx1, _, _ = ops.group_norm_act_bwd(ops.Checkpoint8(ck.q[n:], ck.scale[n // 64:], x[1:].shape, x.dtype), mean[1:], rstd[1:], x[1:], w, b)
    torch.testing.assert_close(dx[1:, :, -3:], dx1[:, :, -3:], rtol=2 ** -6, atol=1e-3)


def test_gradient_written_over_its_source(ops):
    """The C entry's dx may be dy, and a NULL dgamma or dbeta is left out."""
    from elektronn3_amd import _lib
    for shape, dt in (((2, 5, 9, 16, 32, 8), torch.bfloat16), ((1, 3, 7, 5, 24, 3), torch.float32), ((2, 3, 7, 5, 7, 7), torch.float16), ((1, 2, 3, 4, 2048, 256), torch.float32)):
        x, dy, w, b = make(shape, dt, seed=3)
        y, mean, rstd = ops.group_norm_act(x, shape[5], w, b)
        dx, dw, db = ops.group_norm_act_bwd(x, mean, rstd, dy, w, b)
        g, dw2 = dy.clone(), torch.empty_like(dw)
        L = _lib.load()
        ws = torch.empty(L.e3_group_norm_workspace_bytes(*shape, 1), dtype=torch.uint8, device='cuda')
        C = shape[4]
        _lib.check(L.e3_group_norm_act_bwd(_lib.stream_ptr(x.device), ops._DT[dt], x.data_ptr(), C, None, None, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), b.data_ptr(), 0.0,
                                           g.data_ptr(), C, g.data_ptr(), C, dw2.data_ptr(), None, *shape, ws.data_ptr(), ws.numel()))
        assert torch.equal(g, dx) and torch.equal(dw2, dw)


# ------------------------------------------------------------------------------------------------ module
@pytest.mark.parametrize('checkpoint', [False, True])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dims', [1, 2, 3])
def test_module(dims, dtype, checkpoint):
    from elektronn3_amd.norm import GroupNormAct
    g = torch.Generator().manual_seed(dims)
    m = GroupNormAct(4, 24, activation='silu', checkpoint=checkpoint).cuda()
    ref = torch.nn.GroupNorm(4, 24)
    with torch.no_grad():
        m.weight.copy_(1 + 0.2 * torch.randn(24, generator=g)); m.bias.copy_(0.2 * torch.randn(24, generator=g))
    ref.load_state_dict({k: v.cpu() for k, v in m.state_dict().items()})
    ref = ref.double()
    shape = (2, 24, 5, 6, 7)[:2 + dims]
    x0 = torch.randn(shape, generator=g).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    for last in (False, True):
        x = x0.cuda()
        if last and dims > 1:
            x = x.contiguous(memory_format=torch.channels_last if dims == 2 else torch.channels_last_3d)
        x.requires_grad_(True)
        m.zero_grad()
        y = m(x)
        assert y.shape == x.shape and y.dtype == dtype
        y.backward(dy.cuda())
        xr = x0.double().requires_grad_(True)
        yr = torch.nn.functional.silu(ref(xr))
        ref.zero_grad()
        yr.backward(dy.double())
        tol = 4 * HALF[dtype] + 1e-5
        assert float((y.detach().cpu().double() - yr.detach()).abs().max()) <= tol * float(yr.detach().abs().max())
        # with the 8-bit input: half a step of 1 / 127 of a block's largest magnitude (about 4 standard deviations), through a Lipschitz derivative
        lim = tol if not checkpoint else 0.05
        for a, r in ((x.grad, xr.grad), (m.weight.grad, ref.weight.grad), (m.bias.grad, ref.bias.grad)):
            assert float((a.cpu().double() - r).norm()) <= lim * float(r.norm()) + 1e-6


def test_module_captured_with_its_backward():
    """Forward and backward of a small network captured into a graph; replays, with eager work in between, give the eager gradients."""
    from elektronn3_amd.norm import GroupNormAct
    torch.manual_seed(1)
    m = torch.nn.Sequential(GroupNormAct(2, 16, checkpoint=True), GroupNormAct(4, 16, activation='silu')).cuda()
    x = torch.randn(2, 16, 5, 8, 9, device='cuda').contiguous(memory_format=torch.channels_last_3d)
    dy = torch.randn_like(x)
    params = list(m.parameters())

    def step():
        return torch.autograd.grad(m(x), params, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for rep in range(4):
        x.copy_(torch.randn_like(x)); dy.copy_(torch.randn_like(dy))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step())), rep


def test_module_keeps_nothing_without_gradients(monkeypatch):
    from elektronn3_amd import ops as o
    from elektronn3_amd.norm import GroupNormAct
    m, x = GroupNormAct(2, 16, checkpoint=True).cuda(), torch.randn(1, 16, 3, 4, 5, device='cuda')
    y = m(x)
    monkeypatch.setattr(o, '_new_checkpoint', lambda x: pytest.fail('a checkpoint without a backward'))
    with torch.no_grad():
        assert torch.equal(m(x), y)


def test_module_inside_a_network_and_its_state_dict():
    from elektronn3_amd.norm import GroupNormAct
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Conv3d(1, 8, 3, padding=1), GroupNormAct(2, 8, checkpoint=True), torch.nn.Conv3d(8, 2, 1)).cuda()
    assert set(net.state_dict()) == {'0.weight', '0.bias', '1.weight', '1.bias', '2.weight', '2.bias'}
    out = net(torch.randn(2, 1, 6, 7, 8, device='cuda'))
    out.square().mean().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
    y = net[1](torch.randn(2, 8, 6, 7, 8, device='cuda', requires_grad=True))
    kept = y.grad_fn.saved_tensors
    assert sum(t.numel() * t.element_size() for t in kept if t.numel() > 100) < 2 * 8 * 6 * 7 * 8 * 1.1
