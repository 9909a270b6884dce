"""Thin torch-tensor wrappers over the per-op C ABI (include/e3unet.h).

Tensors here are fp32 NDHWC ("channels-last-3d") CUDA tensors of shape (N, D, H, W, C); a trailing-dim slice of a
wider buffer is a valid "view" (ldc = stride of the W axis).  These wrappers exist for unit parity tests and for
callers that want single ops; UNet.forward uses the whole-network entry points instead (one native call per pass).
"""
import torch

from . import _lib
from ._lib import c_size_t, check, ptr, stream_ptr


def _ldc(t):
    """Floats between consecutive voxels of an (N,D,H,W,C) NDHWC view (strides of size-1 dims are ignored)."""
    N, D, H, W, C = t.shape
    sN, sD, sH, sW, sC = t.stride()
    if C > 1 and sC != 1:
        raise ValueError('not an NDHWC view: channel stride must be 1')
    if W > 1:
        ldc = sW
    elif H > 1:
        ldc = sH
    elif D > 1:
        ldc = sD
    elif N > 1:
        ldc = sN
    else:
        ldc = C
    ok = ldc >= C and (H == 1 or W == 1 or sH == W * ldc) and (D == 1 or sD == H * W * ldc or (H == 1 and W == 1)) \
        and (N == 1 or sN == D * H * W * ldc or (D == 1 and H == 1 and W == 1))
    if not ok:
        raise ValueError(f'not an NDHWC view: shape {tuple(t.shape)} strides {t.stride()}')
    return _rows(ldc)


def _rows(ldc):
    """A row length that fits the C ABI's int (ctypes cuts a longer one to 32 bits without an error)."""
    if ldc >= 1 << 31:
        raise ValueError(f'rows of {ldc} elements: longer than the kernels address')
    return ldc


def _chk(t, name):
    if not (t.is_cuda and t.dtype == torch.float32):
        raise ValueError(f'{name}: expected a float32 CUDA tensor (the HIP path has no CPU fallback)')
    if t.dim() == 5:
        _ldc(t)
    return t


def _ws(nbytes, device):
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def conv3d(x, w, bias=None, planar=False, pro=None, epi=None, want_stats=False, out=None):
    """3x3x3 (or 1x3x3) 'same' convolution. x: (N,D,H,W,Cin); w: torch layout (Cout,Cin,kd,3,3)."""
    L = _lib.load()
    _chk(x, 'x')
    N, D, H, W, Cin = x.shape
    Cout = w.shape[0]
    y = out if out is not None else torch.empty((N, D, H, W, Cout), device=x.device, dtype=torch.float32)
    ws = _ws(L.e3_conv3d_workspace_bytes(Cin, Cout, int(planar)), x.device)
    stats = None
    if want_stats:
        parts = L.e3_conv3d_stats_parts(Cin, Cout, N, D, H, W, int(planar))
        stats = torch.zeros((parts, Cout, 3), device=x.device, dtype=torch.float32)
    w = w.contiguous()
    check(L.e3_conv3d_fwd(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(w), ptr(bias), ptr(y), _ldc(y), Cout, N, D, H, W,
                          int(planar), ptr(pro[0]) if pro else None, ptr(pro[1]) if pro else None,
                          ptr(epi[0]) if epi else None, ptr(epi[1]) if epi else None, ptr(stats), ptr(ws), c_size_t(ws.numel())))
    return (y, stats) if want_stats else y


def conv3d_dgrad(dy, w, planar=False):
    L = _lib.load()
    _chk(dy, 'dy')
    N, D, H, W, Cout = dy.shape
    Cin = w.shape[1]
    dx = torch.empty((N, D, H, W, Cin), device=dy.device, dtype=torch.float32)
    ws = _ws(L.e3_conv3d_workspace_bytes(Cin, Cout, int(planar)), dy.device)
    w = w.contiguous()
    check(L.e3_conv3d_dgrad(stream_ptr(dy.device), ptr(dy), _ldc(dy), Cout, ptr(w), ptr(dx), Cin, Cin, N, D, H, W, int(planar),
                            ptr(ws), c_size_t(ws.numel())))
    return dx


def conv3d_wgrad(x, dy, planar=False):
    L = _lib.load()
    _chk(x, 'x'); _chk(dy, 'dy')
    N, D, H, W, Cin = x.shape
    Cout = dy.shape[-1]
    kd = 1 if planar else 3
    dw = torch.empty((Cout, Cin, kd, 3, 3), device=x.device, dtype=torch.float32)
    ws = _ws(L.e3_conv3d_wgrad_workspace_bytes(Cin, Cout, N, D, H, W, int(planar)), x.device)
    check(L.e3_conv3d_wgrad(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(dy), _ldc(dy), Cout, ptr(dw), N, D, H, W, int(planar),
                            ptr(ws), c_size_t(ws.numel())))
    return dw


def convT(x, w, bias=None, out_dims=None, want_stats=False, out=None):
    """ConvTranspose3d(kernel=stride=(sd,2,2)). x: (N,D,H,W,Cin); w: (Cin,Cout,sd,2,2)."""
    L = _lib.load()
    _chk(x, 'x')
    N, D, H, W, Cin = x.shape
    Cout, sd = w.shape[1], w.shape[2]
    Do, Ho, Wo = out_dims if out_dims is not None else (sd * D, 2 * H, 2 * W)
    y = out if out is not None else torch.empty((N, Do, Ho, Wo, Cout), device=x.device, dtype=torch.float32)
    ws = _ws(L.e3_convT_workspace_bytes(Cin, Cout, sd), x.device)
    stats = None
    if want_stats:
        stats = torch.zeros((L.e3_convT_stats_parts(Cin, Cout, N, D, H, W, sd), Cout, 3), device=x.device, dtype=torch.float32)
    w = w.contiguous()
    check(L.e3_convT_fwd(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(w), ptr(bias), ptr(y), _ldc(y), Cout, N, D, H, W, sd,
                         Do, Ho, Wo, ptr(stats), ptr(ws), c_size_t(ws.numel())))
    return (y, stats) if want_stats else y


def convT_dgrad(dy, w, in_dims):
    L = _lib.load()
    _chk(dy, 'dy')
    N, Do, Ho, Wo, Cout = dy.shape
    Cin, sd = w.shape[0], w.shape[2]
    D, H, W = in_dims
    dx = torch.empty((N, D, H, W, Cin), device=dy.device, dtype=torch.float32)
    ws = _ws(L.e3_convT_workspace_bytes(Cin, Cout, sd), dy.device)
    w = w.contiguous()
    check(L.e3_convT_dgrad(stream_ptr(dy.device), ptr(dy), _ldc(dy), Cout, ptr(w), ptr(dx), Cin, Cin, N, D, H, W, sd, Do, Ho, Wo,
                           ptr(ws), c_size_t(ws.numel())))
    return dx


def convT_wgrad(x, dy, sd):
    L = _lib.load()
    _chk(x, 'x'); _chk(dy, 'dy')
    N, D, H, W, Cin = x.shape
    _, Do, Ho, Wo, Cout = dy.shape
    dw = torch.empty((Cin, Cout, sd, 2, 2), device=x.device, dtype=torch.float32)
    ws = _ws(L.e3_convT_wgrad_workspace_bytes(Cin, Cout, N, D, H, W, sd), x.device)
    check(L.e3_convT_wgrad(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(dy), _ldc(dy), Cout, ptr(dw), N, D, H, W, sd, Do, Ho, Wo,
                           ptr(ws), c_size_t(ws.numel())))
    return dw


def bn_finalize(stats, gamma, beta, running_mean=None, running_var=None, momentum=0.1, eps=1e-5):
    L = _lib.load()
    parts, C, _ = stats.shape
    mean, invstd, scale, shift = (torch.empty(C, device=stats.device, dtype=torch.float32) for _ in range(4))
    check(L.e3_bn_finalize(stream_ptr(stats.device), ptr(stats), parts, C, ptr(gamma), ptr(beta), ptr(running_mean), ptr(running_var),
                           float(momentum), float(eps), ptr(mean), ptr(invstd), ptr(scale), ptr(shift)))
    return mean, invstd, scale, shift


def bn_relu_apply(x, scale, shift, pool_kd=0, out=None):
    """a = relu(x*scale+shift); with pool_kd in (1,2) also returns MaxPool3d((kd,2,2), ceil_mode=True)(a)."""
    L = _lib.load()
    _chk(x, 'x')
    N, D, H, W, C = x.shape
    a = out if out is not None else torch.empty((N, D, H, W, C), device=x.device, dtype=torch.float32)
    pooled = None
    if pool_kd:
        pooled = torch.empty((N, -(-D // pool_kd), -(-H // 2), -(-W // 2), C), device=x.device, dtype=torch.float32)
    check(L.e3_bn_relu_apply(stream_ptr(x.device), ptr(x), _ldc(x), ptr(scale), ptr(shift), ptr(a), _ldc(a), ptr(pooled), pool_kd or 2,
                             N, D, H, W, C))
    return (a, pooled) if pool_kd else a


def maxpool(a, kd):
    L = _lib.load()
    _chk(a, 'a')
    N, D, H, W, C = a.shape
    pooled = torch.empty((N, -(-D // kd), -(-H // 2), -(-W // 2), C), device=a.device, dtype=torch.float32)
    check(L.e3_maxpool(stream_ptr(a.device), ptr(a), _ldc(a), ptr(pooled), kd, N, D, H, W, C))
    return pooled


def bn_relu_bwd(x, mean, invstd, gamma, scale, shift, g1=None, gpool=None, a=None, pooled=None, kd=2):
    """Returns dx, dgamma, dbeta, dxsum."""
    L = _lib.load()
    _chk(x, 'x')
    N, D, H, W, C = x.shape
    dx = torch.empty((N, D, H, W, C), device=x.device, dtype=torch.float32)
    dg, db, dxs = (torch.empty(C, device=x.device, dtype=torch.float32) for _ in range(3))
    ws = _ws(L.e3_bn_bwd_workspace_bytes(N, D, H, W, C), x.device)
    check(L.e3_bn_relu_bwd(stream_ptr(x.device), ptr(x), _ldc(x), ptr(mean), ptr(invstd), ptr(gamma), ptr(scale), ptr(shift),
                           ptr(g1), _ldc(g1) if g1 is not None else 0, ptr(gpool), ptr(a), _ldc(a) if a is not None else 0, ptr(pooled), kd,
                           N, D, H, W, C, ptr(dx), C, ptr(dg), ptr(db), ptr(dxs), ptr(ws), c_size_t(ws.numel())))
    return dx, dg, db, dxs


def conv1(a, w, bias, softmax=False):
    """Final 1x1x1 conv; returns NCDHW logits (or probabilities)."""
    L = _lib.load()
    _chk(a, 'a')
    N, D, H, W, C = a.shape
    Cout = w.shape[0]
    y = torch.empty((N, Cout, D, H, W), device=a.device, dtype=torch.float32)
    w = w.contiguous()
    check(L.e3_conv1_fwd(stream_ptr(a.device), ptr(a), _ldc(a), C, ptr(w), ptr(bias), ptr(y), Cout, N, D, H, W, int(softmax)))
    return y


def conv1_bwd(a, w, dy):
    L = _lib.load()
    _chk(a, 'a')
    N, D, H, W, C = a.shape
    Cout = w.shape[0]
    da = torch.empty((N, D, H, W, C), device=a.device, dtype=torch.float32)
    dw = torch.empty((Cout, C, 1, 1, 1), device=a.device, dtype=torch.float32)
    db = torch.empty(Cout, device=a.device, dtype=torch.float32)
    ws = _ws(L.e3_conv1_bwd_workspace_bytes(C, Cout, N, D, H, W), a.device)
    w = w.contiguous(); dy = dy.contiguous()
    check(L.e3_conv1_bwd(stream_ptr(a.device), ptr(a), _ldc(a), C, ptr(w), ptr(dy), ptr(da), C, ptr(dw), ptr(db), Cout, N, D, H, W,
                         ptr(ws), c_size_t(ws.numel())))
    return da, dw, db


def to_ndhwc(x_ncdhw):
    """(N,C,D,H,W) contiguous -> (N,D,H,W,C) contiguous, on device."""
    L = _lib.load()
    N, C, D, H, W = x_ncdhw.shape
    x_ncdhw = x_ncdhw.contiguous()
    out = torch.empty((N, D, H, W, C), device=x_ncdhw.device, dtype=torch.float32)
    check(L.e3_ncdhw_to_ndhwc(stream_ptr(x_ncdhw.device), ptr(x_ncdhw), ptr(out), N, C, D, H, W))
    return out


def to_ncdhw(x_ndhwc):
    L = _lib.load()
    _chk(x_ndhwc, 'x')
    N, D, H, W, C = x_ndhwc.shape
    out = torch.empty((N, C, D, H, W), device=x_ndhwc.device, dtype=torch.float32)
    check(L.e3_ndhwc_to_ncdhw(stream_ptr(x_ndhwc.device), ptr(x_ndhwc), _ldc(x_ndhwc), ptr(out), N, C, D, H, W))
    return out


# ---------------------------------------------------------------------------------------------- native bf16 ops
class _L16:
    """The per-op entry points of the 16-bit path for a tensor's element type: `.e3_conv3d_fwd_bf16` resolves to the `_f16` twin for float16."""

    def __init__(self, t):
        self._lib, self._f16 = _lib.load(), t.dtype == torch.float16

    def __getattr__(self, name):
        return getattr(self._lib, name.replace('_bf16', '_f16') if self._f16 else name)


def _chk16(t, name):
    if not (t.is_cuda and t.dtype in (torch.bfloat16, torch.float16)):
        raise ValueError(f'{name}: expected a bfloat16 / float16 CUDA tensor')
    if t.dim() == 5:
        _ldc(t)
    return t


def conv3d_bf16(x, w, bias=None, planar=False, epi=None, want_stats=False, out=None):
    """bf16 3x3x3 / 1x3x3 'same' conv on the bf16 matrix cores. x: (N,D,H,W,Cin) bf16; w: fp32 torch layout (rounded to bf16 when packed)."""
    L = _L16(x)
    _chk16(x, 'x')
    N, D, H, W, Cin = x.shape
    Cout = w.shape[0]
    y = out if out is not None else torch.empty((N, D, H, W, Cout), device=x.device, dtype=x.dtype)
    ws = _ws(L.e3_conv3d_workspace_bytes_bf16(Cin, Cout, N, D, H, W, int(planar)), x.device)
    stats = None
    if want_stats:
        stats = torch.zeros((L.e3_conv3d_stats_parts_bf16(Cin, Cout, N, D, H, W, int(planar)), Cout, 3), device=x.device, dtype=torch.float32)
    w = w.float().contiguous()
    check(L.e3_conv3d_fwd_bf16(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(w), ptr(bias), ptr(y), _ldc(y), Cout, N, D, H, W, int(planar),
                               ptr(epi[0]) if epi else None, ptr(epi[1]) if epi else None, ptr(stats), ptr(ws), c_size_t(ws.numel())))
    return (y, stats) if want_stats else y


def conv3d_dgrad_bf16(dy, w, planar=False):
    L = _L16(dy)
    _chk16(dy, 'dy')
    N, D, H, W, Cout = dy.shape
    Cin = w.shape[1]
    dx = torch.empty((N, D, H, W, Cin), device=dy.device, dtype=dy.dtype)
    ws = _ws(L.e3_conv3d_workspace_bytes_bf16(Cin, Cout, N, D, H, W, int(planar)), dy.device)
    w = w.float().contiguous()
    check(L.e3_conv3d_dgrad_bf16(stream_ptr(dy.device), ptr(dy), _ldc(dy), Cout, ptr(w), ptr(dx), Cin, Cin, N, D, H, W, int(planar),
                                 ptr(ws), c_size_t(ws.numel())))
    return dx


def conv3d_wgrad_bf16(x, dy, planar=False):
    L = _L16(x)
    _chk16(x, 'x'); _chk16(dy, 'dy')
    N, D, H, W, Cin = x.shape
    Cout = dy.shape[-1]
    dw = torch.empty((Cout, Cin, 1 if planar else 3, 3, 3), device=x.device, dtype=torch.float32)
    ws = _ws(L.e3_conv3d_workspace_bytes_bf16(Cin, Cout, N, D, H, W, int(planar)), x.device)
    check(L.e3_conv3d_wgrad_bf16(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(dy), _ldc(dy), Cout, ptr(dw), N, D, H, W, int(planar),
                                 ptr(ws), c_size_t(ws.numel())))
    return dw


def convT_bf16(x, w, bias=None, out_dims=None, want_stats=False, out=None):
    """bf16 ConvTranspose3d(kernel = stride = 2). x: (N,D,H,W,Cin) bf16; w: (Cin,Cout,2,2,2) fp32."""
    L = _L16(x)
    _chk16(x, 'x')
    N, D, H, W, Cin = x.shape
    Cout = w.shape[1]
    Do, Ho, Wo = out_dims if out_dims is not None else (2 * D, 2 * H, 2 * W)
    y = out if out is not None else torch.empty((N, Do, Ho, Wo, Cout), device=x.device, dtype=x.dtype)
    ws = _ws(L.e3_convT_workspace_bytes_bf16(Cin, Cout, N, D, H, W), x.device)
    stats = torch.zeros((L.e3_convT_stats_parts_bf16(Cin, N, D, H, W), Cout, 3), device=x.device, dtype=torch.float32) if want_stats else None
    w = w.float().contiguous()
    check(L.e3_convT_fwd_bf16(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(w), ptr(bias), ptr(y), _ldc(y), Cout, N, D, H, W, Do, Ho, Wo,
                              ptr(stats), ptr(ws), c_size_t(ws.numel())))
    return (y, stats) if want_stats else y


def convT_dgrad_bf16(dy, w, in_dims):
    L = _L16(dy)
    _chk16(dy, 'dy')
    N, Do, Ho, Wo, Cout = dy.shape
    Cin = w.shape[0]
    D, H, W = in_dims
    dx = torch.empty((N, D, H, W, Cin), device=dy.device, dtype=dy.dtype)
    ws = _ws(L.e3_convT_workspace_bytes_bf16(Cin, Cout, N, D, H, W), dy.device)
    w = w.float().contiguous()
    check(L.e3_convT_dgrad_bf16(stream_ptr(dy.device), ptr(dy), _ldc(dy), Cout, ptr(w), ptr(dx), Cin, Cin, N, D, H, W, Do, Ho, Wo,
                                ptr(ws), c_size_t(ws.numel())))
    return dx


def convT_wgrad_bf16(x, dy):
    L = _L16(x)
    _chk16(x, 'x'); _chk16(dy, 'dy')
    N, D, H, W, Cin = x.shape
    _, Do, Ho, Wo, Cout = dy.shape
    dw = torch.empty((Cin, Cout, 2, 2, 2), device=x.device, dtype=torch.float32)
    ws = _ws(L.e3_convT_workspace_bytes_bf16(Cin, Cout, N, D, H, W), x.device)
    check(L.e3_convT_wgrad_bf16(stream_ptr(x.device), ptr(x), _ldc(x), Cin, ptr(dy), _ldc(dy), Cout, ptr(dw), N, D, H, W, Do, Ho, Wo,
                                ptr(ws), c_size_t(ws.numel())))
    return dw


# ------------------------------------------------------------------ group norm with an activation, 8-bit activation checkpoints
# (small calls are bound by this file: a forward is two launches of 4 us, so the checks below look at every property once and tensors are allocated once)
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}       # E3_DT_*
_SLOPES = {'relu': 0.0, 'leaky': 0.1, 'lin': 1.0, 'silu': 2.0}
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device, fn, *args):
    """One native call on the tensors' device and its current stream."""
    if _current_device() == device.index:
        rc = fn(_raw_stream(device.index), *args)
    else:
        with torch.cuda.device(device):
            rc = fn(_raw_stream(device.index), *args)
    if rc:
        check(rc)


def _chk_any(t, name, shape=None, dtype=None, device=None):
    """Row length of an fp32 / bf16 / fp16 NDHWC view on a ROCm device (with the given shape, type and device)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DT:
        raise ValueError(f'{name}: expected a float32, bfloat16 or float16 tensor')
    if not t.is_cuda:
        raise ValueError(f'{name}: expected a CUDA tensor (the HIP path has no CPU fallback)')
    if shape is not None and (t.shape != shape or t.dtype != dtype or t.device != device):
        raise ValueError(f'{name}: expected shape {tuple(shape)}, {dtype} on {device}, got {tuple(t.shape)}, {t.dtype} on {t.device}')
    if t.dim() != 5:
        raise ValueError(f'{name}: expected a 5D (N, D, H, W, C) tensor, got {t.dim()}D')
    if not t.is_contiguous():
        return _ldc(t)
    C = t.shape[4]
    return C or 1 if C < 1 << 31 else _rows(C)


def _span(t):
    lo = t.data_ptr()
    return lo, lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _chk_out(out, t, name='out'):
    """`out` may be the input itself (the same view); a view that overlaps it otherwise would be read after it was written."""
    if out.numel() == 0 or (t.data_ptr() == out.data_ptr() and (t.stride() == out.stride() or _ldc(t) == _ldc(out))):      # (axes of one element may have any stride)
        return
    (a, b), (c, d) = _span(t), _span(out)
    if a < d and c < b:
        # (halves of one concat buffer interleave in memory without sharing an element: rows of the same length, other channels)
        ldc, size = _ldc(out), out.element_size()
        off = (a - c) // size % ldc
        if _ldc(t) != ldc or (a - c) % size or off < out.shape[4] or off + t.shape[4] > ldc:
            raise ValueError(f'{name} overlaps the input without being the same view')


def _chk_vec(t, n, name, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.numel() != n or t.device != device:
        raise ValueError(f'{name}: expected {n} float32 values on {device}')
    return t if t.is_contiguous() else t.contiguous()


def _act_slope(activation):
    """Slope code of the C ABI from an activation's name or module (those of UNet(activation=...)); nn.PReLU and nn.RReLU are not covered."""
    if isinstance(activation, str):
        slope = _SLOPES.get(activation)
    else:
        from .unet import _activation_slope
        slope = _activation_slope(activation)
    if slope is None or slope == 3.0 or isinstance(activation, torch.nn.RReLU):
        raise NotImplementedError(f"activation {activation!r}: 'relu', 'leaky', 'lin', 'silu' or their modules")
    return slope


class Checkpoint8:
    """An (N, D, H, W, C) activation kept in 8 bits: ``q`` (int8, one code per element in packed NDHWC order) and ``scale`` (float32, one per 64
    elements).  It stands for ``q * scale`` (3.76 times smaller than float32, 1.88 times than a 16-bit type); an element is off by at most half
    a step, ``amax / 254`` of its block's largest magnitude -- by up to a whole step in the checkpoint that :func:`group_norm_act` writes for ReLU or LeakyReLU,
    where an element whose rounded value lies on the other side of the activation's border takes its other neighbour.  A block with a NaN or an infinity stands for NaNs.  Made by :func:`checkpoint8` or
    :func:`group_norm_act`; read by :func:`checkpoint8_restore`, :func:`group_norm_act_apply` and :func:`group_norm_act_bwd`."""
    __slots__ = ('q', 'scale', 'shape', 'dtype', 'device')

    def __init__(self, q, scale, shape, dtype):
        shape = torch.Size(shape)
        n = shape.numel()
        if len(shape) != 5 or dtype not in _DT:
            raise ValueError('Checkpoint8: expected the (N, D, H, W, C) shape and the float32, bfloat16 or float16 type of the tensor it stands for')
        if q.dtype != torch.int8 or q.numel() != n or not q.is_contiguous():
            raise ValueError(f'Checkpoint8: q: expected {n} contiguous int8 codes')
        if scale.dtype != torch.float32 or scale.numel() != -(-n // 64) or not scale.is_contiguous() or scale.device != q.device:
            raise ValueError(f'Checkpoint8: scale: expected {-(-n // 64)} contiguous float32 values on {q.device}')
        _rows(shape[4])
        if not q.is_cuda:
            raise ValueError('Checkpoint8: expected CUDA tensors (the HIP path has no CPU fallback)')
        self.q, self.scale, self.shape, self.dtype, self.device = q, scale, shape, dtype, q.device

    @property
    def nbytes(self):
        return self.q.numel() + 4 * self.scale.numel()

    def numel(self):
        return self.q.numel()

    def __repr__(self):
        return f'Checkpoint8(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})'


def _like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _new_checkpoint(x):
    n = x.numel()
    ck = Checkpoint8.__new__(Checkpoint8)
    ck.q, ck.scale = torch.empty(n, dtype=torch.int8, device=x.device), torch.empty(-(-n // 64), dtype=torch.float32, device=x.device)
    ck.shape, ck.dtype, ck.device = x.shape, x.dtype, x.device
    return ck


def checkpoint8(x):
    """Keeps an activation (float32 / bfloat16 / float16 NDHWC view) in 8 bits; see :class:`Checkpoint8`."""
    ldc = _chk_any(x, 'x')
    ck = _new_checkpoint(x)
    C = x.shape[4] or 1
    _call(ck.device, _lib.load().e3_checkpoint8_pack, _DT[x.dtype], x.data_ptr(), ldc, x.numel() // C, C, ck.q.data_ptr(), ck.scale.data_ptr())
    return ck


def checkpoint8_restore(ck, out=None):
    """The tensor that a :class:`Checkpoint8` stands for, rounded to its type (into ``out``, an NDHWC view, if given)."""
    if not isinstance(ck, Checkpoint8):
        raise ValueError('expected a Checkpoint8')
    C = ck.shape[4] or 1
    if out is None:
        out, ldc = torch.empty(*ck.shape, dtype=ck.dtype, device=ck.device), C
    else:
        ldc = _chk_any(out, 'out', ck.shape, ck.dtype, ck.device)
    _call(ck.device, _lib.load().e3_checkpoint8_unpack, _DT[ck.dtype], ck.q.data_ptr(), ck.scale.data_ptr(), ck.q.numel() // C, C, out.data_ptr(), ldc)
    return out


def _source(x):
    """(x pointer, ldc, q pointer, scale pointer) of a tensor or a checkpoint of it."""
    if isinstance(x, Checkpoint8):
        return None, 0, x.q.data_ptr(), x.scale.data_ptr()
    ldc = _chk_any(x, 'x')
    return x.data_ptr(), ldc, None, None


def _gn_dims(shape, num_groups):
    N, D, H, W, C = shape
    if N < 1 or D < 1 or H < 1 or W < 1 or C < 1:
        raise ValueError(f'x: expected at least one element, got shape {tuple(shape)}')
    if (N | D | H | W | C) >> 31:                # (ctypes cuts longer ones to 32 bits without an error)
        raise ValueError(f'x: expected axes below 2^31, got shape {tuple(shape)}')
    if num_groups < 1 or C % num_groups != 0:
        raise ValueError('num_channels must be divisible by num_groups')
    return N, D, H, W, C, num_groups


def _affine(weight, bias, C, device):
    """(tensors to keep alive, pointers) of the norm's parameters"""
    if weight is not None:
        weight = _chk_vec(weight, C, 'weight', device)
    if bias is not None:
        bias = _chk_vec(bias, C, 'bias', device)
    return weight, bias, weight.data_ptr() if weight is not None else None, bias.data_ptr() if bias is not None else None


def _stats(mean, rstd, N, device):
    if not isinstance(mean, torch.Tensor) or mean.dim() != 2 or mean.shape[0] != N:
        raise ValueError(f'mean: expected shape ({N}, num_groups)')
    n = mean.numel()
    return _chk_vec(mean, n, 'mean', device), _chk_vec(rstd, n, 'rstd', device), mean.shape[1]


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation='relu', checkpoint=False, out=None):
    """``act(group_norm(x, num_groups, weight, bias, eps))`` over a float32 / bfloat16 / float16 NDHWC view (weight, bias: float32 (C,)), with the statistics
    that the backward needs: ``(y, mean, rstd)``, mean and rstd (N, num_groups) float32.  ``checkpoint=True`` also keeps ``x`` in 8 bits on the way:
    ``(y, mean, rstd, Checkpoint8)``.  ``out`` may be ``x`` itself."""
    slope = _act_slope(activation)
    ldc = _chk_any(x, 'x')
    shape, dtype, device = x.shape, x.dtype, x.device
    dims = _gn_dims(shape, num_groups)
    C = dims[4]
    weight, bias, wp, bp = _affine(weight, bias, C, device)
    if not eps >= 0:
        raise ValueError('eps must not be negative')
    if out is None:
        y, y_ldc = _like(x), C
    else:
        y, y_ldc = out, _chk_any(out, 'out', shape, dtype, device)
        _chk_out(out, x)
    L = _lib.load()
    mean = torch.empty(dims[0], num_groups, dtype=torch.float32, device=device)
    rstd = torch.empty_like(mean)
    ck = _new_checkpoint(x) if checkpoint else None
    nbytes = L.e3_group_norm_workspace_bytes(*dims, 0)           # (0 for small groups)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _call(device, L.e3_group_norm_act_fwd, _DT[dtype], x.data_ptr(), ldc, wp, bp, eps, slope, y.data_ptr(), y_ldc, mean.data_ptr(), rstd.data_ptr(),
          ck.q.data_ptr() if ck else None, ck.scale.data_ptr() if ck else None, *dims, ws.data_ptr() if nbytes else None, nbytes)
    return (y, mean, rstd, ck) if checkpoint else (y, mean, rstd)


def group_norm_act_apply(x, mean, rstd, weight=None, bias=None, activation='relu', out=None):
    """``y`` of :func:`group_norm_act` from its statistics and its input or the input's :class:`Checkpoint8` (the activation recomputed in a backward
    pass; a checkpoint's values enter in float32).  ``out`` may be ``x`` itself."""
    slope = _act_slope(activation)
    src = _source(x)
    shape, dtype, device = x.shape, x.dtype, x.device
    mean, rstd, G = _stats(mean, rstd, shape[0], device)
    dims = _gn_dims(shape, G)
    C = dims[4]
    weight, bias, wp, bp = _affine(weight, bias, C, device)
    if out is None:
        y, y_ldc = torch.empty(*shape, dtype=dtype, device=device) if src[0] is None else _like(x), C
    else:
        y, y_ldc = out, _chk_any(out, 'out', shape, dtype, device)
        if src[0] is not None:
            _chk_out(out, x)
    _call(device, _lib.load().e3_group_norm_act_apply, _DT[dtype], *src, mean.data_ptr(), rstd.data_ptr(), wp, bp, slope, y.data_ptr(), y_ldc, *dims)
    return y


def group_norm_act_bwd(x, mean, rstd, dy, weight=None, bias=None, activation='relu'):
    """Gradients ``(dx, dweight, dbias)`` of :func:`group_norm_act` from its statistics and its input or the input's :class:`Checkpoint8`; dweight and
    dbias are float32 (C,) whether or not the norm has parameters."""
    slope = _act_slope(activation)
    src = _source(x)
    shape, dtype, device = x.shape, x.dtype, x.device
    mean, rstd, G = _stats(mean, rstd, shape[0], device)
    dims = _gn_dims(shape, G)
    C = dims[4]
    weight, bias, wp, bp = _affine(weight, bias, C, device)
    dy_ldc = _chk_any(dy, 'dy', shape, dtype, device)
    L = _lib.load()
    dx = _like(dy)
    dw = torch.empty(C, dtype=torch.float32, device=device)
    db = torch.empty_like(dw)
    nbytes = L.e3_group_norm_workspace_bytes(*dims, 1)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _call(device, L.e3_group_norm_act_bwd, _DT[dtype], *src, mean.data_ptr(), rstd.data_ptr(), wp, bp, slope, dy.data_ptr(), dy_ldc, dx.data_ptr(), C,
          dw.data_ptr(), db.data_ptr(), *dims, ws.data_ptr() if nbytes else None, nbytes)
    return dx, dw, db
