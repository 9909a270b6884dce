"""What UNet.checkpoint8() hands its backward, tensor by tensor: the buffer of saved activations after the way through the 8 bits against the one that the same forward left, at the channel
counts of the headline network.

The codes are checked bit by bit against the format's definition (x * (127 / amax) and amax * (1 / 127), each operation rounded to fp32, round to even) and its side rule; the codes that the
pooling windows' rule may change, by what it promises: an element stays at one of its two neighbours on the grid, a window whose rounded values had the right maximum is left alone, and a
window's first maximum moves only where a neighbouring code does not allow to keep it there.  Recomputed activations: fmaf is one rounding, a slope another, both evaluated in 64 bits here
(one more, u = 2^-24 each): 4 u |y|; SiLU as in test_group_norm_gpu.py; pooled tensors are the exact maxima of the recomputed activations."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Arena:
    """Views of the tensors in a buffer of saved activations (batch norm, 'same' convolutions, transposed convolutions): channels last, every tensor at a multiple of 256 bytes."""

    def __init__(self, m, shape, buf):
        self.buf, self.off = buf, 0
        N, cin, nb = shape[0], shape[1], len(m.down_convs)
        ch = [m.down_convs[i].conv2.weight.shape[0] for i in range(nb)]
        planar = [i in m.planar_blocks for i in range(nb)]
        dims = [tuple(shape[2:])]
        for i in range(nb - 1):
            d, h, w = dims[-1]
            dims.append((d if planar[i] else -(-d // 2), -(-h // 2), -(-w // 2)))
        add = m.merge_mode == 'add'
        self.xin = self.take(N, *dims[0], cin) if cin > 1 else None
        self.cat, self.pooled, self.sum = [], [], []
        for j in range(nb - 1):
            self.cat.append(self.take(N, *dims[j], 2 * ch[j]))
            self.pooled.append(self.take(N, *dims[j + 1], ch[j]))
            self.sum.append(self.take(N, *dims[j], ch[j]) if add else None)
        plan = [(i, c, False) for i in range(nb) for c in (1, 2)] + [(j, c, c == 0) for j in range(nb - 2, -1, -1) for c in (0, 1, 2)]
        self.units = []
        for k, (lv, c, up) in enumerate(plan):
            u = {'level': lv, 'planar': planar[lv], 'C': ch[lv], 'last': k + 1 == len(plan), 'raw': self.take(N, *dims[lv], ch[lv])}
            u['skip'] = k < 2 * nb and c == 2 and lv < nb - 1
            u['act'] = self.cat[lv][..., ch[lv]:] if u['skip'] else self.cat[lv][..., :ch[lv]] if up else self.take(N, *dims[lv], ch[lv])
            u['vec'] = [self.take(ch[lv]) for _ in range(4)]           # mean, 1 / std, scale, shift
            self.units.append(u)

    def take(self, *shape):
        n = 4 * torch.Size(shape).numel()
        t = self.buf[self.off:self.off + n].view(torch.float32).view(shape)
        self.off += -(-n // 256) * 256
        return t


def codes(x):
    """(codes as fp32, scale per element) of a channels-last tensor, to the nearest"""
    flat = x.reshape(-1)
    p = F.pad(flat, (0, -flat.numel() % 64)).view(-1, 64)
    amax = p.abs().amax(1, keepdim=True)
    none = amax < 2.0 ** -110
    q = torch.round(p * (torch.full_like(amax, 127.0) / amax.masked_fill(none, 1.0))).masked_fill(none, 0.0)
    s = (amax * torch.tensor(1 / 127, dtype=torch.float32, device=x.device)).masked_fill(none, 0.0).expand_as(p)
    return q.reshape(-1)[:flat.numel()].view(x.shape), s.reshape(-1)[:flat.numel()].view(x.shape)


def positive(x, a, b):
    return x.double() * a.double() + b.double() > 0          # (the product of two fp32 is exact in 64 bits: the sign of fmaf)


def windows(t, planar, fill):
    """[position in the window, in the pool's order][N, D', H', W', C]"""
    kd = 1 if planar else 2
    t = F.pad(t, (0, 0, 0, -t.shape[3] % 2, 0, -t.shape[2] % 2, 0, -t.shape[1] % kd), value=fill)
    return torch.stack([t[:, d::kd, h::2, w::2] for d in range(kd) for h in range(2) for w in range(2)])


def first(w):
    top = w.max(0, keepdim=True).values
    return (w == top).float().argmax(0)


def forward(m, x, seed):
    torch.manual_seed(seed)
    out = m(x)
    return out, out.grad_fn


CASES = [
    # the headline network (32 ... 256 channels) at its full size, and at sizes that no window or block divides
    (dict(n_blocks=4, start_filts=32), (2, 1, 64, 128, 128), 'relu'),
    (dict(n_blocks=4, start_filts=32), (1, 1, 13, 37, 51), 'relu'),
    (dict(n_blocks=4, start_filts=32, planar_blocks=(0,), activation='leaky'), (1, 1, 9, 41, 70), 'leaky'),
    (dict(n_blocks=3, start_filts=32, activation='silu', merge_mode='add', in_channels=3), (2, 3, 11, 22, 35), 'silu'),
    (dict(n_blocks=3, start_filts=16, activation=torch.nn.RReLU(1 / 8, 1 / 3)), (2, 1, 15, 26, 33), 'rrelu'),
    (dict(n_blocks=4, start_filts=32, activation='rrelu'), (1, 1, 16, 33, 64), 'rrelu'),
]


@pytest.mark.parametrize('kw,shape,act', CASES)
def test_saved_activations(kw, shape, act):
    from elektronn3_amd.unet import UNet
    torch.manual_seed(5)
    kw = dict(kw)
    m = UNet(kw.pop('in_channels', 1), 2, **kw).cuda().train()
    with torch.no_grad():
        for k, p in m.named_parameters():
            if 'norm' in k:
                p.add_(0.2 * torch.randn_like(p))
    x = torch.randn(shape, generator=torch.Generator().manual_seed(7)).cuda()
    out, node = forward(m, x, 11)
    exact = Arena(m, shape, node.saved_buf)
    assert exact.off == node.saved_buf.numel()
    m.checkpoint8()
    out8, node8 = forward(m, x, 11)
    assert torch.equal(out8, out)
    from elektronn3_amd import _lib
    if node8.rrelu is not None:
        assert node8.rrelu == node.rrelu
        other, node_other = forward(m, x, 12)                  # (another graph, with slopes of its own, in between)
        assert node_other.rrelu != node8.rrelu
        _lib.check(_lib.load().e3_unet_set_rrelu(m._plan().handle, *node8.rrelu))
    got = Arena(m, shape, node8.saved_buf.restore(node8.tens.tens))
    assert got.off == got.buf.numel()
    if exact.xin is not None:
        assert torch.equal(got.xin, exact.xin)
    moved = count = 0
    for k, (e, g) in enumerate(zip(exact.units, got.units)):
        assert all(torch.equal(p, q) for p, q in zip(e['vec'], g['vec'])), k
        a, b = e['vec'][2], e['vec'][3]
        q, s = codes(e['raw'])
        if act != 'silu':
            step = torch.where(e['raw'] > q * s, 1.0, -1.0)
            q = torch.where(positive(e['raw'], a, b) != positive(q * s, a, b), (q + step).clamp_(-127, 127), q)
        v0 = q * s
        if not e['skip']:
            assert torch.equal(g['raw'], v0), k
        else:
            v1 = torch.where(e['raw'] > v0, q + 1, q - 1).clamp_(-127, 127) * s
            assert bool(((g['raw'] == v0) | (g['raw'] == v1)).all()), k
            if act != 'silu':
                assert torch.equal(positive(g['raw'], a, b), positive(v0, a, b)), k
        if g['last']:
            break                                              # (the head reads the raw tensor)
        z = g['raw'].double() * a.double() + b.double()
        if act == 'rrelu':
            # the slope of every element, from the activation that the forward left and from the recomputed one
            ze = e['raw'].double() * a.double() + b.double()
            neg = (ze < -1e-3) & (z < -1e-3)
            want, have = e['act'].double()[neg] / ze[neg], g['act'].double()[neg] / z[neg]
            assert bool(((have - want).abs() <= 8 * U * want.abs()).all()), k
            assert bool((want > 1 / 8 - 1e-6).all()) and bool((want < 1 / 3 + 1e-6).all()) and float(want.std()) > 0.04, k
            assert torch.equal(g['act'][z > 0], z[z > 0].float()) or bool(((g['act'].double() - z).abs()[z > 0] <= 2 * U * z[z > 0]).all()), k
        else:
            y = {'relu': F.relu, 'leaky': lambda t: F.leaky_relu(t, 0.1), 'silu': F.silu}[act](z)
            err = U * (2 * z.abs() + 8) * y.abs() + 1.1 * 2 * U * z.abs() if act == 'silu' else 4 * U * y.abs()
            assert bool(((g['act'].double() - y).abs() <= err).all()), k
        if e['skip']:
            w = windows(g['act'], e['planar'], float('-inf'))
            assert torch.equal(got.pooled[e['level']], w.max(0).values), k
            if act == 'rrelu':
                continue
            fn = {'relu': F.relu, 'leaky': lambda t: F.leaky_relu(t, 0.1), 'silu': F.silu}[act]
            ze, z0 = (t.double() * a.double() + b.double() for t in (e['raw'], v0))
            inf = float('-inf')
            order = lambda zz: first(windows(fn(zz.float()) if act != 'silu' else fn(zz), e['planar'], inf))     # noqa: E731
            right, rounded, now = order(ze), order(z0), first(w)
            same = windows((g['raw'] == v0).float(), e['planar'], 1.0).amin(0) > 0
            if act != 'silu':                                  # (SiLU's order by its approximation is the kernel's own)
                assert bool(same[right == rounded].all()), k
            off = now != right
            count += off.numel()
            moved += int(off.sum())
            # what forbids to keep a maximum: an element of the window within a step of the border (ReLU, LeakyReLU), or where SiLU is not monotone (z < 0)
            close = (ze.abs() <= (s * a.abs()).double() * (1 + 1e-6)) if act != 'silu' else ze < 0
            assert bool((windows(close.float(), e['planar'], 0.0).amax(0) > 0)[off].all()), k
    print(f'first maxima that moved: {moved} of {count} windows')
    if act != 'rrelu':
        assert moved <= count // 1000
    for j, t in enumerate(got.sum):
        if t is not None:
            C = t.shape[-1]
            assert torch.equal(t, got.cat[j][..., :C] + got.cat[j][..., C:])


@pytest.mark.parametrize('kw,shape,act', CASES[1:])
def test_backward_reads_only_what_is_restored(monkeypatch, kw, shape, act):
    """The gradients from buffers whose bytes were all NaN before the forward or the restoring filled them; and those of a full graph that is given the restored tensors."""
    from elektronn3_amd import _lib, unet
    torch.manual_seed(5)
    kw = dict(kw)
    m = unet.UNet(kw.pop('in_channels', 1), 2, **kw).cuda().train()
    g = torch.Generator().manual_seed(9)
    x, dy = torch.randn(shape, generator=g).cuda(), torch.randn(shape[0], 2, *shape[2:], generator=g).cuda()

    def gradients(out):
        m.zero_grad()
        out.backward(dy)
        return [p.grad.clone() for p in m.parameters()]
    m.checkpoint8()
    want = gradients(forward(m, x, 11)[0])
    monkeypatch.setattr(unet, '_alloc_saved', lambda device, n: torch.full((int(n),), 255, dtype=torch.uint8, device=device))
    got = gradients(forward(m, x, 11)[0])
    assert all(bool(torch.isfinite(p).all()) and torch.equal(p, q) for p, q in zip(got, want))
    out8, node8 = forward(m, x, 11)
    m.checkpoint8(False)
    out, node = forward(m, x, 11)
    if node8.rrelu is not None:
        _lib.check(_lib.load().e3_unet_set_rrelu(m._plan().handle, *node8.rrelu))
    node.saved_buf = node8.saved_buf.restore(node8.tens.tens)
    assert all(torch.equal(p, q) for p, q in zip(gradients(out), want))
