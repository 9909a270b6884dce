"""Timing cases of the normalisation operators of a U-Net block and of their 8-bit activation checkpoints.

Every case is ONE pass that a training program makes over a channels-last tensor (N, D, H, W, C):

  fwd    group norm with an activation                                       y, mean, rstd
  bwd    its gradients from the kept input                                   dx, dweight, dbias
  bwd8   its gradients from an 8-bit checkpoint of the input                 dx, dweight, dbias
  keep   an activation put into an 8-bit checkpoint and taken out again      the restored tensor, the scales
  step   a block's whole pass with the checkpoint in place of its input: forward, the activation recomputed for the weight
         gradient of the next convolution, and the gradients                 y, mean, rstd, the recomputed y, dx, dweight, dbias

``run`` computes them with elementary torch operations; with ``own`` set it calls ``elektronn3_amd.ops``.  ``exact`` evaluates the
definitions in 64 bits.

The operators.  With groups of C / G consecutive channels, mean and variance over a group's channels and voxels of one sample:
    z = (x - mean) * rstd * weight + bias,   y = act(z),   rstd = 1 / sqrt(var + eps)
    dz = dy * act'(z),   h = (x - mean) * rstd,   dweight = sum(dz * h),   dbias = sum(dz)     (sums over samples and voxels)
    dx = rstd * (weight * dz - mean_g(weight * dz) - h * mean_g(weight * dz * h))
act'(z) at z = 0 is that of z < 0.  An 8-bit checkpoint cuts the packed [N][D][H][W][C] elements into blocks of 64; a block keeps
q = round_to_even(x * (127 / amax)) and the scale amax * (1 / 127), with every operation rounded to 32 bits, and stands for q * scale.
"""
import math

import torch

own = False

EPS = 1e-5
BLOCK = 64                              # elements that share one scale of an 8-bit checkpoint
TINY = 2.0 ** -110                      # a block whose largest magnitude is below this is kept as zeros
SLOPE = {'relu': 0.0, 'leaky': 0.1, 'lin': 1.0}
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
KINDS = ('fwd', 'bwd', 'bwd8', 'keep', 'step')
MOST = 2 * 64 * 128 * 128 * 32          # elements of the largest case: level 0 of the benchmarked training step


def _case(name, kind, dtype, N, D, H, W, C, G, act, ldc=0):
    return {'name': name, 'kind': kind, 'dtype': dtype, 'N': N, 'D': D, 'H': H, 'W': W, 'C': C, 'G': G, 'act': act, 'ldc': ldc or C}


def listed():
    return [
        # level 0 of the benchmarked network (batch 2 of 64 x 128 x 128 voxels, 32 channels): the largest tensors of a training step
        _case('fwd_f32_level0', 'fwd', 'float32', 2, 64, 128, 128, 32, 8, 'relu'),
        # level 1 of the same network in its 16-bit form
        _case('fwd_bf16_level1', 'fwd', 'bfloat16', 2, 32, 64, 64, 64, 8, 'silu'),
        # the bottom of a small-tile network: a call whose time is its latency
        _case('fwd_f16_bottom', 'fwd', 'float16', 1, 4, 8, 8, 128, 8, 'relu'),
        # a ragged tile with a channel count that is no multiple of 8
        _case('fwd_f32_ragged', 'fwd', 'float32', 3, 17, 45, 51, 20, 5, 'leaky'),
        # the backward of level 0 with 16-bit storage
        _case('bwd_bf16_level0', 'bwd', 'bfloat16', 2, 64, 128, 128, 32, 8, 'relu'),
        # fp32 backward of level 2 on odd sizes
        _case('bwd_f32_odd', 'bwd', 'float32', 2, 17, 33, 31, 128, 16, 'silu'),
        # the same passes with the input kept in 8 bits: level 0 in fp32 (the reads shrink most there) and a deep level in float16
        _case('bwd8_f32_level0', 'bwd8', 'float32', 2, 64, 128, 128, 32, 8, 'relu'),
        _case('bwd8_f16_level3', 'bwd8', 'float16', 2, 8, 16, 16, 256, 32, 'leaky'),
        # one half of a decoder's concat buffer (rows of 64 channels, 32 of them kept), and a 2D network's activation of odd size
        _case('keep_f32_concat', 'keep', 'float32', 2, 64, 128, 128, 32, 1, 'lin', 64),
        _case('keep_bf16_2d_odd', 'keep', 'bfloat16', 4, 1, 333, 517, 24, 1, 'lin'),
        # a block with its input kept in 8 bits: 16-bit training at level 1, and a 2D batch in fp32
        _case('step_bf16_level1', 'step', 'bfloat16', 4, 32, 64, 64, 64, 8, 'silu'),
        _case('step_f32_2d', 'step', 'float32', 8, 1, 188, 188, 32, 4, 'silu'),
    ]


def draw(rng):
    kind, dtype = rng.choice(KINDS), rng.choice(sorted(DTYPES))
    # channel counts of the networks (multiples of 8) three times out of four, any count otherwise
    C = 8 * round(2 ** rng.uniform(0, 6)) if rng.random() < 0.75 else rng.randrange(2, 200)
    G = rng.choice([g for g in range(1, C + 1) if C % g == 0 and g <= 64])
    most = MOST // 2                    # (half: a step makes two passes more than a forward)
    if C % 8:
        most //= 8
    total = 2 ** rng.uniform(12, math.log2(most))      # elements of the whole batch
    N = rng.choice([1, 1, 2, 3, 4])
    vox = max(32, total / N / C)
    D = 1 if rng.random() < 0.25 else max(1, round(vox ** rng.uniform(0.15, 0.33)))
    H = max(1, round((vox / D) ** rng.uniform(0.4, 0.6)))
    W = max(1, int(vox / (D * H)))
    act = 'silu' if kind == 'step' else rng.choice(['relu', 'leaky', 'lin', 'silu'])
    ldc = C * rng.choice([1, 1, 2]) if kind in ('fwd', 'keep') else C
    return {'kind': kind, 'dtype': dtype, 'N': N, 'D': D, 'H': H, 'W': W, 'C': C, 'G': G, 'act': act, 'ldc': ldc}


def prepare(case, seed):
    """A block's tensors as a training program holds them: the raw output of a convolution (its channels have offsets and widths of their
    own), the norm's parameters, the incoming gradient, and what an earlier forward kept."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    N, C, G = case['N'], case['C'], case['G']
    shape = (N, case['D'], case['H'], case['W'])
    rand = lambda *s: torch.randn(*s, device='cuda', generator=gen)   # noqa: E731
    wide = rand(*shape, case['ldc']) * (0.3 * rand(case['ldc'])).exp() + 0.5 * rand(case['ldc'])
    x = wide.to(dtype)[..., :C]
    s = {'case': dict(case), 'x': x, 'weight': 1 + 0.2 * rand(C), 'bias': 0.2 * rand(C)}
    if case['kind'] in ('bwd', 'bwd8', 'step'):
        s['dy'] = (0.05 * rand(*shape, C)).to(dtype)
    if case['kind'] in ('bwd', 'bwd8'):
        s['mean'], s['rstd'] = _statistics(x, G)
    if case['kind'] == 'bwd8':
        s['q'], s['scale'] = _keep8(x)
        del s['x']
    return s


# ------------------------------------------------------------------------------------------------ the plain form
def _statistics(x, G):
    N, C = x.shape[0], x.shape[-1]
    g = x.float().reshape(N, -1, G, C // G)
    mean = g.mean((1, 3), keepdim=True, dtype=torch.float64)        # (long sums)
    var = (g - mean).square().mean((1, 3))
    return mean.reshape(N, G).float(), (var + EPS).rsqrt().float()


def _per_channel(v, C):
    """(N, G) -> (N, 1, 1, 1, C)"""
    return v.repeat_interleave(C // v.shape[1], 1)[:, None, None, None, :]


def _normalised(x, mean, rstd):
    C = x.shape[-1]
    return (x - _per_channel(mean, C)) * _per_channel(rstd, C)


def _activated(z, act):
    if act == 'silu':
        return z / (1 + torch.exp(-z))
    return torch.where(z > 0, z, SLOPE[act] * z)


def _plain_apply(x, mean, rstd, weight, bias, act, dtype):
    return _activated(_normalised(x.float(), mean, rstd) * weight + bias, act).to(dtype)


def _plain_backward(x, mean, rstd, dy, weight, bias, act):
    N, C, G = x.shape[0], x.shape[-1], mean.shape[1]
    x, g = x.float(), dy.float()
    h = _normalised(x, mean, rstd)
    if act == 'silu':
        z = h * weight + bias
        sig = 1 / (1 + torch.exp(-z))
        dz = g * (sig * (1 + z * (1 - sig)))
    else:       # the side of the border that a value falls on: in 64 bits
        z = _normalised(x.double(), mean, rstd) * weight + bias
        dz = torch.where(z > 0, g, SLOPE[act] * g)
    over = (0, 1, 2, 3)
    dweight = (dz * h).sum(over, dtype=torch.float64).float()
    dbias = dz.sum(over, dtype=torch.float64).float()
    wdz = dz * weight
    m1 = wdz.reshape(N, -1, G, C // G).mean((1, 3), dtype=torch.float64).float()
    m2 = (wdz * h).reshape(N, -1, G, C // G).mean((1, 3), dtype=torch.float64).float()
    dx = _per_channel(rstd, C) * (wdz - _per_channel(m1, C) - h * _per_channel(m2, C))
    return dx.to(dy.dtype), dweight, dbias


def _keep8(x):
    flat = x.reshape(-1).float()
    n = flat.numel()
    blocks = torch.nn.functional.pad(flat, (0, -n % BLOCK)).reshape(-1, BLOCK)
    amax = blocks.abs().amax(1)
    small = amax < TINY
    inv = torch.full_like(amax, 127.0) / torch.where(small, torch.ones_like(amax), amax)
    q = torch.where(small[:, None], torch.zeros_like(blocks), torch.round(blocks * inv[:, None]))
    scale = torch.where(small, torch.zeros_like(amax), amax * (1 / 127))
    bad = ~torch.isfinite(amax)
    q = torch.where(bad[:, None], torch.zeros_like(q), q)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    return q.reshape(-1)[:n].to(torch.int8), scale


def _stands_for(q, scale, shape):
    wide = torch.nn.functional.pad(q.float(), (0, -q.numel() % BLOCK)).reshape(-1, BLOCK) * scale[:, None]
    return wide.reshape(-1)[:q.numel()].reshape(shape)


def _shape(case):
    return case['N'], case['D'], case['H'], case['W'], case['C']


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    c = s['case']
    kind, act, dtype = c['kind'], c['act'], DTYPES[c['dtype']]
    if kind == 'keep':
        q, scale = _keep8(s['x'])
        return {'restored': _stands_for(q, scale, _shape(c)).to(dtype), 'scale': scale}
    if kind == 'bwd8':
        x = _stands_for(s['q'], s['scale'], _shape(c))
    else:
        x = s['x']
    out = {}
    if kind in ('fwd', 'step'):
        mean, rstd = _statistics(x, c['G'])
        out = {'y': _plain_apply(x, mean, rstd, s['weight'], s['bias'], act, dtype), 'mean': mean, 'rstd': rstd}
        if kind == 'fwd':
            return out
        x = _stands_for(*_keep8(x), _shape(c))
        out['again'] = _plain_apply(x, mean, rstd, s['weight'], s['bias'], act, dtype)
    else:
        mean, rstd = s['mean'], s['rstd']
    dx, dweight, dbias = _plain_backward(x, mean, rstd, s['dy'], s['weight'], s['bias'], act)
    return {**out, 'dx': dx, 'dweight': dweight, 'dbias': dbias}


# ------------------------------------------------------------------------------------------------ the framework's operators
def _run_own(s):
    from elektronn3_amd import ops
    c = s['case']
    kind, act, dtype = c['kind'], c['act'], DTYPES[c['dtype']]
    if kind == 'keep':
        kept = ops.checkpoint8(s['x'])
        return {'restored': ops.checkpoint8_restore(kept), 'scale': kept.scale}
    if kind == 'fwd':
        y, mean, rstd = ops.group_norm_act(s['x'], c['G'], s['weight'], s['bias'], eps=EPS, activation=act)
        return {'y': y, 'mean': mean, 'rstd': rstd}
    out = {}
    if kind == 'step':
        y, mean, rstd, kept = ops.group_norm_act(s['x'], c['G'], s['weight'], s['bias'], eps=EPS, activation=act, checkpoint=True)
        out = {'y': y, 'mean': mean, 'rstd': rstd,
               'again': ops.group_norm_act_apply(kept, mean, rstd, s['weight'], s['bias'], activation=act)}
    else:
        mean, rstd = s['mean'], s['rstd']
        kept = s['x'] if kind == 'bwd' else ops.Checkpoint8(s['q'], s['scale'], _shape(c), dtype)
    dx, dweight, dbias = ops.group_norm_act_bwd(kept, mean, rstd, s['dy'], s['weight'], s['bias'], activation=act)
    return {**out, 'dx': dx, 'dweight': dweight, 'dbias': dbias}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n = math.prod(_shape(case))
    item = 4 if case['dtype'] == 'float32' else 2
    t, kept = n * item, n + 4 * -(-n // BLOCK)         # bytes of one tensor, of one checkpoint
    small = 8 * case['N'] * case['G'] + 16 * case['C']
    return {
        'fwd': {'bytes': 2 * t + small, 'flops': 10 * n},
        'bwd': {'bytes': 3 * t + small, 'flops': 20 * n},
        'bwd8': {'bytes': 2 * t + kept + small, 'flops': 21 * n},
        'keep': {'bytes': 2 * t + 2 * kept, 'flops': 5 * n},
        'step': {'bytes': 5 * t + 2 * kept + small, 'flops': 42 * n},
    }[case['kind']]


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_codes(x):
    """(values that the checkpoint stands for, scales): the operations that the definition rounds to 32 bits are evaluated in 64 and rounded."""
    n = x.numel()
    v = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    v[:n] = x.reshape(-1).double()
    v = v.view(-1, BLOCK)
    top = v.abs().max(1, keepdim=True).values
    zero = top < TINY
    inv = (127.0 / top.masked_fill(zero, 1.0)).float().double()
    code = (v * inv).float().double().round().masked_fill(zero, 0.0)
    unit = torch.tensor(1 / 127, dtype=torch.float32).double().item()
    scale = (top * unit).float().double().masked_fill(zero, 0.0)
    return (code * scale).view(-1)[:n].view(x.shape), scale.view(-1)


def exact(case, seed):
    s = prepare(case, seed)
    c, act = s['case'], case['act']
    shape, G = _shape(c), c['G']
    N, C = shape[0], shape[-1]
    if c['kind'] == 'keep':
        values, scale = _exact_codes(s['x'])
        return {'restored': values, 'scale': scale}
    if c['kind'] == 'bwd8':
        x = s['q'].double()
        x = (x * s['scale'].double().repeat_interleave(BLOCK)[:x.numel()]).float().double().view(shape)
    else:
        x = s['x'].double()
    w, b = s['weight'].double(), s['bias'].double()
    grouped = lambda t: t.reshape(N, -1, G, C // G)                     # noqa: E731
    spread = lambda m: m[:, None, :, None].expand(N, 1, G, C // G).reshape(N, 1, 1, 1, C)   # noqa: E731

    def act_of(z):
        return z * torch.sigmoid(z) if act == 'silu' else torch.where(z > 0, z, z * SLOPE[act])

    out = {}
    if 'mean' in s:
        mean, rstd = s['mean'].double(), s['rstd'].double()
    else:
        mean = grouped(x).mean((1, 3))
        rstd = 1 / (grouped(x).var((1, 3), unbiased=False) + EPS).sqrt()
        out = {'y': act_of((x - spread(mean)) * spread(rstd) * w + b), 'mean': mean, 'rstd': rstd}
        if c['kind'] == 'fwd':
            return out
        x = _exact_codes(s['x'])[0].float().double()
        out['again'] = act_of((x - spread(mean)) * spread(rstd) * w + b)
    h = (x - spread(mean)) * spread(rstd)
    z = h * w + b
    if act == 'silu':
        p = torch.sigmoid(z)
        slope = p * (1 + z * (1 - p))
    else:
        slope = torch.where(z > 0, 1.0, SLOPE[act]).double()
    dz = s['dy'].double() * slope
    u = dz * w
    dx = spread(rstd) * (u - spread(grouped(u).mean((1, 3))) - h * spread(grouped(u * h).mean((1, 3))))
    return {**out, 'dx': dx, 'dweight': (dz * h).sum((0, 1, 2, 3)), 'dbias': dz.sum((0, 1, 2, 3))}
