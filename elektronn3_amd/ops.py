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
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}       # E3_DT_*


def _chk_any(t, name, like=None):
    """An fp32 / bf16 / fp16 NDHWC view on a ROCm device (with the shape, type and device of `like`)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DT:
        raise ValueError(f'{name}: expected a float32, bfloat16 or float16 tensor')
    if not t.is_cuda:
        raise ValueError(f'{name}: expected a CUDA tensor (the HIP path has no CPU fallback)')
    if t.dim() != 5:
        raise ValueError(f'{name}: expected a 5D (N, D, H, W, C) tensor, got {t.dim()}D')
    if like is not None and (tuple(t.shape) != tuple(like.shape) or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f'{name}: expected shape {tuple(like.shape)}, {like.dtype} on {like.device}, got {tuple(t.shape)}, {t.dtype} on {t.device}')
    return _ldc(t) if t.numel() else max(t.shape[4], 1)


def _chk_out(out, ins, name='out'):
    """`out` may be one of the inputs itself (the same view); a view that overlaps one otherwise would be read after it was written."""
    lo = out.data_ptr()
    hi = lo + ((out.shape[0] - 1) * out.stride(0) + (out.shape[1] - 1) * out.stride(1) + (out.shape[2] - 1) * out.stride(2)
               + (out.shape[3] - 1) * out.stride(3) + out.shape[4]) * out.element_size() if out.numel() else lo
    for t in ins:
        if t is None or t.numel() == 0 or (t.data_ptr() == lo and t.dtype == out.dtype and t.stride() == out.stride()):
            continue
        a = t.data_ptr()
        b = a + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
        # (the two halves of a concat buffer interleave in memory without sharing an element: rows of the same buffer, other channels)
        if a < hi and lo < b and not _disjoint_channels(t, out):
            raise ValueError(f'{name} overlaps an input without being the same view')


def _disjoint_channels(t, out):
    if t.dtype != out.dtype or t.dim() != 5:
        return False
    ldc, d = _ldc(out), (t.data_ptr() - out.data_ptr())
    if _ldc(t) != ldc or d % t.element_size():
        return False
    d = (d // t.element_size()) % ldc
    return d >= out.shape[4] and d + t.shape[4] <= ldc


def _chk_vec(t, n, name, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.numel() != n or t.device != device:
        raise ValueError(f'{name}: expected {n} float32 values on {device}')
    return t.contiguous()


def _act_slope(activation):
    """Slope code of the C ABI from an activation's name or module (those of UNet(activation=...)); nn.PReLU and nn.RReLU are not covered."""
    from .unet import _activation_slope
    slope = _activation_slope(activation)
    if slope is None or slope == 3.0 or activation == 'rrelu' or isinstance(activation, torch.nn.RReLU):
        raise NotImplementedError(f"activation {activation!r}: 'relu', 'leaky', 'lin', 'silu' or their modules")
    return slope


class Checkpoint8:
    """An (N, D, H, W, C) activation kept in 8 bits: ``q`` (int8, one code per element in packed NDHWC order) and ``scale`` (float32, one per 64
    elements).  It stands for ``q * scale`` (3.76 times smaller than float32, 1.88 times than a 16-bit type); an element is off by at most half
    a step, ``amax / 254`` of its block's largest magnitude.  A block with a NaN or an infinity stands for NaNs.  Made by :func:`checkpoint8` or
    :func:`group_norm_act`; read by :func:`checkpoint8_restore`, :func:`group_norm_act_apply` and :func:`group_norm_act_bwd`."""
    __slots__ = ('q', 'scale', 'shape', 'dtype')

    def __init__(self, q, scale, shape, dtype):
        shape = torch.Size(int(s) for s in shape)
        n = shape.numel()
        if len(shape) != 5 or dtype not in _DT:
            raise ValueError('Checkpoint8: expected the (N, D, H, W, C) shape and the float32, bfloat16 or float16 type of the tensor it stands for')
        if q.dtype != torch.int8 or q.numel() != n or not q.is_contiguous():
            raise ValueError(f'Checkpoint8: q: expected {n} contiguous int8 codes')
        if scale.dtype != torch.float32 or scale.numel() != -(-n // 64) or not scale.is_contiguous() or scale.device != q.device:
            raise ValueError(f'Checkpoint8: scale: expected {-(-n // 64)} contiguous float32 values on {q.device}')
        if not q.is_cuda:
            raise ValueError('Checkpoint8: expected CUDA tensors (the HIP path has no CPU fallback)')
        self.q, self.scale, self.shape, self.dtype = q, scale, shape, dtype

    @property
    def device(self):
        return self.q.device

    @property
    def nbytes(self):
        return self.q.numel() + 4 * self.scale.numel()

    def numel(self):
        return self.q.numel()

    def __repr__(self):
        return f'Checkpoint8(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})'


def _new_checkpoint(x):
    n = x.numel()
    return Checkpoint8(torch.empty(n, dtype=torch.int8, device=x.device), torch.empty(-(-n // 64), dtype=torch.float32, device=x.device), x.shape, x.dtype)


def checkpoint8(x):
    """Keeps an activation (float32 / bfloat16 / float16 NDHWC view) in 8 bits; see :class:`Checkpoint8`."""
    ldc = _chk_any(x, 'x')
    ck = _new_checkpoint(x)
    with torch.cuda.device(x.device):
        check(_lib.load().e3_checkpoint8_pack(stream_ptr(x.device), _DT[x.dtype], ptr(x), ldc, x.numel() // max(x.shape[4], 1), x.shape[4] or 1, ptr(ck.q), ptr(ck.scale)))
    return ck


def checkpoint8_restore(ck, out=None):
    """The tensor that a :class:`Checkpoint8` stands for, rounded to its type (into ``out``, an NDHWC view, if given)."""
    if not isinstance(ck, Checkpoint8):
        raise ValueError('expected a Checkpoint8')
    y = out if out is not None else torch.empty(ck.shape, dtype=ck.dtype, device=ck.device)
    ldc = _chk_any(y, 'out', like=ck)
    with torch.cuda.device(ck.device):
        check(_lib.load().e3_checkpoint8_unpack(stream_ptr(ck.device), _DT[ck.dtype], ptr(ck.q), ptr(ck.scale), ck.numel() // max(ck.shape[4], 1), ck.shape[4] or 1,
                                                ptr(y), ldc))
    return y


def _source(x):
    """(x pointer, ldc, q pointer, scale pointer) of a tensor or a checkpoint of it."""
    if isinstance(x, Checkpoint8):
        return None, 0, ptr(x.q), ptr(x.scale)
    return ptr(x), _chk_any(x, 'x'), None, None


def _gn_dims(x, num_groups):
    N, D, H, W, C = x.shape
    if min(x.shape) < 1:
        raise ValueError(f'x: expected at least one element, got shape {tuple(x.shape)}')
    if num_groups < 1 or C % num_groups != 0:
        raise ValueError('num_channels must be divisible by num_groups')
    return N, D, H, W, C, num_groups


def _stats(x, mean, rstd):
    if mean.dim() != 2 or mean.shape[0] != x.shape[0]:
        raise ValueError(f'mean: expected shape ({x.shape[0]}, num_groups)')
    n = mean.numel()
    return _chk_vec(mean, n, 'mean', x.device), _chk_vec(rstd, n, 'rstd', x.device), mean.shape[1]


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation='relu', checkpoint=False, out=None):
    """``act(group_norm(x, num_groups, weight, bias, eps))`` over a float32 / bfloat16 / float16 NDHWC view (weight, bias: float32 (C,)), with the statistics
    that the backward needs: ``(y, mean, rstd)``, mean and rstd (N, num_groups) float32.  ``checkpoint=True`` also keeps ``x`` in 8 bits on the way:
    ``(y, mean, rstd, Checkpoint8)``.  ``out`` may be ``x`` itself."""
    slope = _act_slope(activation)
    ldc = _chk_any(x, 'x')
    dims = _gn_dims(x, num_groups)
    weight, bias = _chk_vec(weight, x.shape[4], 'weight', x.device), _chk_vec(bias, x.shape[4], 'bias', x.device)
    if not eps >= 0:
        raise ValueError('eps must not be negative')
    y = out if out is not None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y_ldc = _chk_any(y, 'out', like=x)
    if out is not None:
        _chk_out(out, (x,))
    L = _lib.load()
    mean, rstd = (torch.empty((x.shape[0], num_groups), dtype=torch.float32, device=x.device) for _ in range(2))
    ck = _new_checkpoint(x) if checkpoint else None
    ws = _ws(L.e3_group_norm_workspace_bytes(*dims), x.device)
    with torch.cuda.device(x.device):
        check(L.e3_group_norm_act_fwd(stream_ptr(x.device), _DT[x.dtype], ptr(x), ldc, ptr(weight), ptr(bias), float(eps), slope, ptr(y), y_ldc, ptr(mean), ptr(rstd),
                                      ptr(ck.q) if ck else None, ptr(ck.scale) if ck else None, *dims, ptr(ws), c_size_t(ws.numel())))
    return (y, mean, rstd, ck) if checkpoint else (y, mean, rstd)


def group_norm_act_apply(x, mean, rstd, weight=None, bias=None, activation='relu', out=None):
    """``y`` of :func:`group_norm_act` from its statistics and its input or the input's :class:`Checkpoint8` (the activation recomputed in a backward
    pass; a checkpoint's values enter in float32)."""
    slope = _act_slope(activation)
    src = _source(x)
    mean, rstd, G = _stats(x, mean, rstd)
    dims = _gn_dims(x, G)
    weight, bias = _chk_vec(weight, x.shape[4], 'weight', x.device), _chk_vec(bias, x.shape[4], 'bias', x.device)
    y = out if out is not None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y_ldc = _chk_any(y, 'out', like=x)
    if out is not None and not isinstance(x, Checkpoint8):
        _chk_out(out, (x,))
    with torch.cuda.device(x.device):
        check(_lib.load().e3_group_norm_act_apply(stream_ptr(x.device), _DT[x.dtype], *src, ptr(mean), ptr(rstd), ptr(weight), ptr(bias), slope, ptr(y), y_ldc, *dims))
    return y


def group_norm_act_bwd(x, mean, rstd, dy, weight=None, bias=None, activation='relu'):
    """Gradients ``(dx, dweight, dbias)`` of :func:`group_norm_act` from its statistics and its input or the input's :class:`Checkpoint8`; dweight and
    dbias are float32 (C,) whether or not the norm has parameters."""
    slope = _act_slope(activation)
    src = _source(x)
    mean, rstd, G = _stats(x, mean, rstd)
    dims = _gn_dims(x, G)
    C = x.shape[4]
    weight, bias = _chk_vec(weight, C, 'weight', x.device), _chk_vec(bias, C, 'bias', x.device)
    dy_ldc = _chk_any(dy, 'dy', like=x)
    L = _lib.load()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw, db = (torch.empty(C, dtype=torch.float32, device=x.device) for _ in range(2))
    ws = _ws(L.e3_group_norm_workspace_bytes(*dims), x.device)
    with torch.cuda.device(x.device):
        check(L.e3_group_norm_act_bwd(stream_ptr(x.device), _DT[x.dtype], *src, ptr(mean), ptr(rstd), ptr(weight), ptr(bias), slope, ptr(dy), dy_ldc, ptr(dx), C,
                                      ptr(dw), ptr(db), *dims, ptr(ws), c_size_t(ws.numel())))
    return dx, dw, db
