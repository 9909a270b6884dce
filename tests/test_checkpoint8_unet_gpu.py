"""UNet.checkpoint8(): training graphs that hold their activations in 8 bits (elektronn3_amd/unet.py, csrc/unet_plan.cpp).

The gradients are checked against a 64-bit network on the CPU in which every convolution's output is REPLACED by what its 8-bit checkpoint stands for while the
statistics stay those of the exact outputs -- what the native backward computes with.  The library's fp32 outputs differ from the 64-bit ones by some 1e-6 of a
block's largest magnitude, i.e. 1e-4 of a step, so about 2e-4 of the codes fall one step further: 1 % of the value in 2e-4 of the elements, 1.4e-4 of a tensor's
norm, and as much again per layer that it passes.  TOL = 2e-3 leaves ten layers; the rounding to 8 bits itself changes the gradients by more (asserted)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

TOL = 2e-3


def kept(x, z, border, pool=None, fn=None):
    """What the 8-bit checkpoint of an NCDHW tensor stands for (blocks of 64 of the NDHWC order); border: rounded to the side of z = 0 that an element is on;
    pool: window of the max-pool behind fn(z), whose first maximum stays where it is."""
    v = x.detach().float().movedim(1, -1).contiguous()
    flat = v.reshape(-1).numpy()
    p = np.zeros(-(-flat.size // 64) * 64, np.float32); p[:flat.size] = flat
    p = p.reshape(-1, 64)
    amax = np.abs(p).max(1, keepdims=True)
    q = np.rint(p * (np.float32(127) / np.maximum(amax, np.float32(1e-30))))
    back = lambda q: torch.from_numpy((q * (amax * np.float32(1 / 127))).reshape(-1)[:flat.size].reshape(v.shape)).double().movedim(-1, 1)    # noqa: E731
    val = back(q)
    if border:
        move = torch.where((z(x) > 0) != (z(val) > 0), torch.where(x > val, 1.0, -1.0), 0.0).movedim(1, -1).reshape(-1).numpy()
        p[:] = 0
        p.reshape(-1)[:flat.size] = move
        q = np.clip(q + p, -127, 127)
        val = back(q)
    if pool:
        step = torch.where(x > val, 1.0, -1.0).movedim(1, -1).reshape(-1).numpy()
        p[:] = 0
        p.reshape(-1)[:flat.size] = step
        val = windows(x, val, back(np.clip(q + p, -127, 127)), z, fn, border, pool)
    return val


def windows(x, v0, v1, z, fn, border, pool):
    """v0, v1: the two neighbours of x on the grid of its block, v0 the one in use.  Per window: the maximum of fn(z(x)) takes the larger of its two where the rounded
    values have another maximum, then what still reaches it the smaller of its two."""
    def cut(t, fill):
        t = torch.nn.functional.pad(t, [n for s, k in zip(t.shape[:1:-1], pool[::-1]) for n in (0, -s % k)], value=fill)
        return torch.stack([t[:, :, d::pool[0], h::2, w::2] for d in range(pool[0]) for h in range(2) for w in range(2)])
    ok = cut(torch.ones_like(x), 0) > 0
    inf = torch.tensor(float('-inf'), dtype=torch.float64)
    o, o0, o1 = (torch.where(ok, cut(fn(z(t)), 0), inf) for t in (x, v0, v1))
    allowed = ok & (cut(((z(v0) > 0) == (z(v1) > 0)).double(), 0) > 0) if border else ok
    first = lambda t: (t == t.max(0, keepdim=True).values).double().argmax(0, keepdim=True)      # noqa: E731
    m, wrong = first(o), first(o) != first(o0)
    k = torch.arange(o.shape[0]).view(-1, 1, 1, 1, 1, 1)
    take = wrong & (k == m) & allowed & (o1 > o0)
    now = torch.where(take, o1, o0)
    top = now.gather(0, m)
    reach = torch.where(k < m, now >= top, now > top) & (k != m)
    take = take | (wrong & reach & allowed & (o1 < o0))
    out = torch.where(take, cut(v1, 0), cut(v0, 0))
    full = torch.zeros(*x.shape[:2], *(n * s for n, s in zip(out.shape[3:], pool)), dtype=torch.float64)
    for i, t in enumerate(out):
        full[:, :, i // 4::pool[0], i // 2 % 2::2, i % 2::2] = t
    return full[:, :, :x.shape[2], :x.shape[3], :x.shape[4]]


class Norm(torch.autograd.Function):
    """Batch / group norm with given statistics (1, G) or (C,): the train-mode backward at the given x."""
    @staticmethod
    def forward(ctx, x, gamma, beta, mean, invstd, dims):
        h = (x - mean) * invstd
        ctx.save_for_backward(h, gamma, invstd); ctx.dims = dims
        return h * gamma.view(1, -1, 1, 1, 1) + beta.view(1, -1, 1, 1, 1)

    @staticmethod
    def backward(ctx, dz):
        h, gamma, invstd = ctx.saved_tensors
        u = dz * gamma.view(1, -1, 1, 1, 1)
        g = u if ctx.dims is None else u.view(u.shape[0], ctx.dims, -1)
        hg = h if ctx.dims is None else h.view(h.shape[0], ctx.dims, -1)
        over = (0, 2, 3, 4) if ctx.dims is None else (2,)
        m1, m2 = g.mean(over, keepdim=True), (g * hg).mean(over, keepdim=True)
        dx = (g - m1 - hg * m2).view_as(u) * invstd
        return dx, (dz * h).sum((0, 2, 3, 4)), dz.sum((0, 2, 3, 4)), None, None, None


def emulate(m, x, dy, act, groups=None, add=False, replace=True, frozen=False):
    """Gradients of sum(dy * net(x)) in 64 bits, the raw tensors replaced by their checkpoints' values.  groups: None = batch norm, 0 = instance norm;
    frozen: batch norm with the running statistics as constants."""
    sd = {k: p.detach().cpu().double().requires_grad_(True) for k, p in m.named_parameters()}
    bufs = {k: b.detach().cpu().double() for k, b in m.named_buffers()}
    flat = m.dim == 2
    if flat:
        x, dy = x.unsqueeze(2), dy.unsqueeze(2)

    def unit(conv, a, a_exact, prefix, norm, up=False, slope=None, pool=None):
        w, b = sd[f'{prefix}.weight'], sd[f'{prefix}.bias']
        w = w.unsqueeze(2) if flat else w
        k = tuple(w.shape[2:])
        f = (lambda t: F.conv_transpose3d(t, w, b, stride=k)) if up else (lambda t: F.conv3d(t, w, b, padding=tuple(n // 2 for n in k)))
        raw = f(a_exact).detach()
        y = f(a)
        G = raw.shape[1] if groups == 0 else groups
        if frozen:
            mean, var = (bufs[f'{norm}.running_{s}'].view(1, -1, 1, 1, 1) for s in ('mean', 'var'))
        elif groups is None:
            mean, var = raw.mean((0, 2, 3, 4), keepdim=True), raw.var((0, 2, 3, 4), unbiased=False, keepdim=True)
        else:
            r = raw.view(raw.shape[0], G, -1)
            mean, var = (t.repeat_interleave(raw.shape[1] // G, 1).view(raw.shape[0], -1, 1, 1, 1) for t in (r.mean(2), r.var(2, unbiased=False)))
        inv = 1 / (var + 1e-5).sqrt()
        ga, be = (sd[f'{norm}.weight'], sd[f'{norm}.bias']) if groups != 0 else (torch.ones(raw.shape[1], dtype=torch.float64), torch.zeros(raw.shape[1], dtype=torch.float64))
        aff = lambda t: ((t - mean) * inv * ga.view(1, -1, 1, 1, 1) + be.view(1, -1, 1, 1, 1)).detach()    # noqa: E731
        fn = {'relu': F.relu, 'leaky': lambda t: F.leaky_relu(t, 0.1), 'leaky2': lambda t: F.leaky_relu(t, 0.2), 'silu': F.silu, 'prelu': lambda t: F.prelu(t, sd[slope])}[act]
        y = y + ((kept(raw, aff, act not in ('silu', 'lin'), pool, lambda t: fn(t).detach()) if replace else raw) - y).detach()
        if frozen:
            z = (y - mean) * inv * ga.view(1, -1, 1, 1, 1) + be.view(1, -1, 1, 1, 1)
        else:
            z = Norm.apply(y, ga, be, mean, inv, G)
        ze = aff(raw)
        return fn(z), fn(ze).detach()

    a = ae = x.cpu().double()
    skips = []
    nb = len(m.down_convs)
    for i in range(nb):
        for c in (1, 2):
            a, ae = unit(None, a, ae, f'down_convs.{i}.conv{c}', f'down_convs.{i}.norm{c - 1}', slope=f'down_convs.{i}.act{c}.weight',
                         pool=(1 if flat or i in m.planar_blocks else 2, 2, 2) if c == 2 and i < nb - 1 else None)
        if i < nb - 1:
            skips.append((a, ae))
            a, ae = (F.max_pool3d(t, (1, 2, 2) if flat or i in m.planar_blocks else 2, ceil_mode=True) for t in (a, ae))
    for i in range(nb - 1):
        a, ae = unit(None, a, ae, f'up_convs.{i}.upconv', f'up_convs.{i}.norm0', up=True, slope=f'up_convs.{i}.act0.weight')
        s, se = skips.pop()
        a, ae = ((t + u) if add else torch.cat((t, u), 1) for t, u in ((a, s), (ae, se)))
        for c in (1, 2):
            a, ae = unit(None, a, ae, f'up_convs.{i}.conv{c}', f'up_convs.{i}.norm{c}', slope=f'up_convs.{i}.act{c}.weight')
    w = sd['conv_final.weight']
    out = F.conv3d(a, w.unsqueeze(2) if flat else w, sd['conv_final.bias'])
    out.backward(dy.cpu().double())
    return {k: p.grad for k, p in sd.items()}


def build(seed=0, **kw):
    from elektronn3_amd.unet import UNet
    torch.manual_seed(seed)
    m = UNet(kw.pop('in_channels', 1), 2, start_filts=8, **kw).cuda().train()
    with torch.no_grad():
        for k, p in m.named_parameters():
            if 'norm' in k:
                p.add_(0.2 * torch.randn_like(p))
    return m


CASES = [
    (dict(n_blocks=2), (2, 1, 8, 12, 10), 'relu'),
    (dict(n_blocks=3, activation='silu'), (1, 1, 8, 16, 12), 'silu'),
    (dict(n_blocks=2, activation='leaky', merge_mode='add', in_channels=3), (2, 3, 4, 10, 8), 'leaky'),
    (dict(n_blocks=2, activation='prelu'), (1, 1, 6, 8, 10), 'prelu'),
    (dict(n_blocks=2, normalization='group4'), (2, 1, 8, 8, 12), 'relu'),
    (dict(n_blocks=2, normalization='instance'), (2, 1, 8, 8, 12), 'relu'),
    (dict(n_blocks=2, dim=2), (2, 1, 16, 20), 'relu'),
    (dict(n_blocks=3, planar_blocks=(0,)), (1, 1, 4, 16, 12), 'relu'),
    (dict(n_blocks=2, activation=torch.nn.RReLU(0.2, 0.2)), (1, 1, 8, 8, 10), 'leaky2'),      # (its slopes are drawn from [0.2, 0.2])
]


@pytest.mark.parametrize('kw,shape,act', CASES)
def test_gradients_are_those_of_the_rounded_tensors(kw, shape, act):
    m = build(**dict(kw))
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(shape, generator=g).cuda(), torch.randn(shape[0], 2, *shape[2:], generator=g).cuda()
    groups = {'group4': 4, 'instance': 0}.get(kw.get('normalization'))
    add = kw.get('merge_mode') == 'add'
    m.checkpoint8()
    out8 = check(m, x, dy, emulate(m, x, dy, act, groups, add))
    want, plain = emulate(m, x, dy, act, groups, add), emulate(m, x, dy, act, groups, add, replace=False)
    change = [float((plain[k] - w).norm()) / float(w.norm()) for k, w in want.items() if counts(k)]
    print('change of the gradients: median %.2g, largest %.2g' % (sorted(change)[len(change) // 2], max(change)))
    assert sum(c > TOL for c in change) > len(change) // 3, 'the checkpoints make no difference: nothing is tested'
    # the outputs do not change, and switched off the gradients are the full ones again
    m.checkpoint8(False)
    assert torch.equal(check(m, x, dy, plain), out8)


def counts(k):
    return not (k.endswith('.bias') and 'norm' not in k and not k.startswith('conv_final'))      # (a bias that feeds a norm: zero up to rounding)


def check(m, x, dy, want):
    m.zero_grad()
    out = m(x)
    out.backward(dy)
    for k, p in m.named_parameters():
        if counts(k):
            off = float((p.grad.cpu().double() - want[k]).norm())
            assert off <= TOL * float(want[k].norm()), (k, off / float(want[k].norm()))
    return out.detach()


def test_frozen_statistics():
    m = build(n_blocks=2)
    x, dy = torch.randn(2, 1, 8, 12, 10, device='cuda'), torch.randn(2, 2, 8, 12, 10, device='cuda')
    with torch.no_grad():
        for _ in range(3):
            m(x)
    m.eval().checkpoint8()
    want = {k: g for k, g in emulate(m, x, dy, 'relu', frozen=True).items()}
    check(m, x, dy, want)


def test_memory_of_pending_graphs_and_order_of_their_backwards():
    """Three graphs alive at once: each holds about 1/7 of the full arena; their backwards in another order give the gradients of each alone."""
    m = build(n_blocks=3)
    xs = [torch.randn(1, 1, 32, 64, 64, device='cuda') for _ in range(3)]
    dy = torch.randn(1, 2, 32, 64, 64, device='cuda')

    def alone(x):
        m.zero_grad(); m(x).backward(dy)
        return [p.grad.clone() for p in m.parameters()]

    def held():
        torch.cuda.synchronize(); before = torch.cuda.memory_allocated()
        outs = [m(x) for x in xs]
        return outs, torch.cuda.memory_allocated() - before - sum(o.numel() * 4 for o in outs)
    outs, full = held(); del outs
    m.checkpoint8()
    want = [alone(x) for x in xs]
    outs, small = held()
    assert small < full / 6, (small, full)
    for i in (1, 2, 0):
        m.zero_grad()
        outs[i].backward(dy)
        assert all(torch.equal(p.grad, w) for p, w in zip(m.parameters(), want[i]))


def test_other_ways_through_the_module():
    """The criterion inside the head, no graph at all."""
    from elektronn3_amd.loss import CombinedCEDiceLoss
    m = build(n_blocks=2).checkpoint8()
    x, t = torch.randn(2, 1, 8, 16, 16, device='cuda'), torch.randint(0, 2, (2, 8, 16, 16), device='cuda')
    crit = CombinedCEDiceLoss(weight=[0.3, 0.7]).cuda()
    out, loss = m.forward_with_loss(x, t, crit)
    m.zero_grad(); loss.backward()
    fused = [p.grad.clone() for p in m.parameters()]
    m.zero_grad(); crit(m(x), t).backward()
    for a, p in zip(fused, m.parameters()):
        torch.testing.assert_close(a, p.grad, rtol=1e-3, atol=1e-6)
    with torch.no_grad():
        assert bool(torch.isfinite(m(x)).all())


def test_what_is_not_covered_is_refused():
    from elektronn3_amd import resunet
    from elektronn3_amd.unet import UNet
    for kw in (dict(normalization='none'), dict(full_norm=False), dict(attention=True), dict(up_mode='resizeconv_nearest'), dict(conv_mode='valid')):
        m = UNet(1, 2, n_blocks=2, start_filts=8, **kw)
        with pytest.raises(NotImplementedError):
            m.checkpoint8()
        m.checkpoint8(False)
    with pytest.raises(NotImplementedError):
        resunet.UNet(1, 2, n_blocks=2, start_filts=8).checkpoint8()
    m = UNet(1, 2, n_blocks=2, start_filts=32).cuda().train().checkpoint8()
    x = torch.randn(1, 1, 8, 16, 16, device='cuda')
    before = {k: v.clone() for k, v in m.state_dict().items()}
    with pytest.raises(NotImplementedError), torch.autocast('cuda', dtype=torch.bfloat16):
        m(x)
    assert all(torch.equal(v, before[k]) for k, v in m.state_dict().items())
