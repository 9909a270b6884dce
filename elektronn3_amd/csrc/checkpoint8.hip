// 8-bit activation checkpoints: a tensor into codes and block scales, and back (the format: checkpoint8.h).
//
// Both are one streaming pass: 4 + 1.06 bytes per fp32 element, 2 + 1.06 per 16-bit element, a few operations each: HBM-bound.  2 x 64 x 128 x 128 x 32 in fp32
// (268 MB + 71 MB): 67 us there, 61 us back (5.0, 5.5 TB/s).  A tensor of the memory-side cache's size or more is read / written past it (NT; 73 and 68 us without);
// smaller ones stay in it for their next reader (134 MB restored with NT: 31 us instead of 28).
#include "checkpoint8.h"

#include "../../include/e3unet.h"

using namespace e3n;

namespace {

constexpr int BT = 256;

// flat piece -> (voxel row, first channel).  DENSE: the rows follow each other without a gap, the view is one flat array.
template <int V, bool DENSE> __device__ __forceinline__ size_t piece_offset(size_t e, int C, int ldc) {
    if constexpr (DENSE) return e;
    else {
        const size_t v = e < 0xffffffffu ? (size_t)((unsigned)e / (unsigned)C) : e / (size_t)C;
        return v * (size_t)ldc + (e - v * (size_t)C);
    }
}

// Codes of flat elements e0 ... moved to their side
template <int V> __device__ __forceinline__ void to_side_exact(const Border& d, int C, size_t e0, const float (&f)[V], Codes<V>& q) {
    size_t v = e0 < 0xffffffffu ? (size_t)((unsigned)e0 / (unsigned)C) : e0 / (size_t)C;
    int c = (int)(e0 - v * (size_t)C);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const size_t g = (v / (size_t)d.S) * d.G + c / (C / d.G);
        const double mu = d.mean[g], rs = d.rstd[g], ga = d.gamma ? (double)d.gamma[c] : 1.0, be = d.beta ? (double)d.beta[c] : 0.0;
        const float w = code_value<V>(q, e);
        if ((((double)f[e] - mu) * rs * ga + be > 0.0) != (((double)w - mu) * rs * ga + be > 0.0)) q.q[e] = other_neighbour(q.q[e], f[e], w);
        if (++c == C) { c = 0; ++v; }
    }
}
// ... with the constants a, b of a piece's channels (C % V == 0: a piece lies in one voxel)
template <int V> struct Affine { float a[V], b[V]; };
template <int V> __device__ __forceinline__ Affine<V> affine_at(const Border& d, int C, size_t e0) {
    const int c = (int)(e0 < 0xffffffffu ? (unsigned)e0 % (unsigned)C : (unsigned)(e0 % (size_t)C));
    Affine<V> k;
#pragma unroll
    for (int e = 0; e < V; ++e) { k.a[e] = d.a[c + e]; k.b[e] = d.b[c + e]; }
    return k;
}
template <int V> __device__ __forceinline__ void to_side_affine(const Affine<V>& k, const float (&f)[V], Codes<V>& q) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float w = code_value<V>(q, e);
        if ((__builtin_fmaf(f[e], k.a[e], k.b[e]) > 0.f) != (__builtin_fmaf(w, k.a[e], k.b[e]) > 0.f)) q.q[e] = other_neighbour(q.q[e], f[e], w);
    }
}

template <int DT, int V, bool DENSE, bool NT, int RULE>
__global__ __launch_bounds__(BT) void checkpoint8_pack_kernel(const typename Elem<DT>::T* __restrict__ x, int ldc, int C, size_t n,
                                                              signed char* __restrict__ q, float* __restrict__ scale, const Border border) {
    constexpr int U = DT == DT_F32 ? 8 : 4;                  // pieces in flight per lane
    const size_t step = (size_t)gridDim.x * BT * V;
    // (where the grid's step is whole voxels a thread keeps its channels, and their constants)
    const bool same = RULE == 2 && step % (size_t)C == 0;
    Affine<V> k{};
    if constexpr (RULE == 2) k = affine_at<V>(border, C, ((size_t)blockIdx.x * BT + threadIdx.x) * V);
    // (the loop's condition is the workgroup's: every lane of a wave reaches the reduction inside encode_block)
    for (size_t b0 = (size_t)blockIdx.x * BT * V; b0 < n; b0 += U * step) {
        Raw<DT, V> raw[U]; bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t e = b0 + u * step + (size_t)threadIdx.x * V;
            ok[u] = e < n;
            raw[u] = Raw<DT, V>{};
            if (ok[u]) raw[u] = load_raw<DT, V, NT>(x + piece_offset<V, DENSE>(e, C, ldc));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V];
            unpack_raw<DT, V>(raw[u], f);
            Codes<V> c = encode_block<V>(f);
            const size_t e0 = b0 + u * step + (size_t)threadIdx.x * V;
            if constexpr (RULE == 1) if (ok[u] && c.scale > 0.f) to_side_exact<V>(border, C, e0, f, c);
            if constexpr (RULE == 2) if (ok[u] && c.scale > 0.f) {
                if (!same) k = affine_at<V>(border, C, e0);
                to_side_affine<V>(k, f, c);
            }
            if (ok[u]) store_codes<V>(c, q, scale, e0);
        }
    }
}

template <int DT, int V, bool DENSE, bool NT>
__global__ __launch_bounds__(BT) void checkpoint8_unpack_kernel(const signed char* __restrict__ q, const float* __restrict__ scale, size_t n, int C, int ldc,
                                                                typename Elem<DT>::T* __restrict__ y) {
    constexpr int U = DT == DT_F32 ? 8 : 4;
    const size_t step = (size_t)gridDim.x * BT * V;
    for (size_t e0 = ((size_t)blockIdx.x * BT + threadIdx.x) * V; e0 < n; e0 += U * step) {
        RawQ<V> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) { raw[u] = RawQ<V>{}; if (e0 + u * step < n) raw[u] = load_q<V>(q, scale, e0 + u * step); }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V];
            unpack_q<V>(raw[u], f);
            if (e0 + u * step < n) store_f32<DT, V, NT>(y + piece_offset<V, DENSE>(e0 + u * step, C, ldc), f);
        }
    }
}

constexpr size_t CACHE_BYTES = 256u << 20;

// A unit's raw tensor out of its checkpoint together with what the executor forms from it: the activation a = act(fmaf(raw, scale, shift)) into a view and, POOL, its
// ceil-mode max-pool -- the expressions and the order of elementwise.hip's passes, bit for bit.  One lane = one voxel (POOL: one window) x 4 channels.  (Restoring and
// those passes one after the other read every raw tensor once more.)  Network of 4 levels on 2 x 64 x 128 x 128: 602 us per step without pools, 174 with: HBM-bound.
template <bool POOL>
__global__ __launch_bounds__(BT) void checkpoint8_act_kernel(const RestoreArgs r) {
    const float slope = r.act.get();
    const int Q = r.C >> 2, kd = POOL ? r.kd : 1;
    const int Dp = (r.D + kd - 1) / kd, Hp = POOL ? (r.H + 1) >> 1 : r.H, Wp = POOL ? (r.W + 1) >> 1 : r.W;
    const size_t total = (size_t)r.N * Dp * Hp * Wp * Q;
    auto one = [&](size_t v, int q, const RawQ<4>& raw) {
        float f[4], o[4];
        unpack_q<4>(raw, f);
        const f32x4 sc = *reinterpret_cast<const f32x4*>(r.scale + 4 * q), sh = *reinterpret_cast<const f32x4*>(r.shift + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = act_fwd(__builtin_fmaf(f[e], sc[e], sh[e]), act_slope_at(r.act, slope, (unsigned)(v * r.C + 4 * q + e)));
        *reinterpret_cast<f32x4*>(r.raw + v * r.C + 4 * q) = f32x4{f[0], f[1], f[2], f[3]};
        const f32x4 y = {o[0], o[1], o[2], o[3]};
        *reinterpret_cast<f32x4*>(r.a + v * r.a_ldc + 4 * q) = y;
        return y;
    };
    for (size_t i = blockIdx.x * (size_t)BT + threadIdx.x; i < total; i += (size_t)gridDim.x * BT) {
        const int q = i % Q; size_t t = i / Q;
        if constexpr (!POOL) one(t, q, load_q<4>(r.q, r.qs, t * r.C + 4 * q));
        else {
            const int pw = t % Wp; t /= Wp; const int ph = t % Hp; t /= Hp; const int pd = t % Dp; const int n = t / Dp;
            RawQ<4> raw[8]; size_t vox[8]; bool ok[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int dz = k >> 2, d = pd * kd + dz, h = ph * 2 + ((k >> 1) & 1), w = pw * 2 + (k & 1);
                ok[k] = dz < kd && d < r.D && h < r.H && w < r.W;
                vox[k] = (((size_t)n * r.D + d) * r.H + h) * r.W + w;
                raw[k] = {};
                if (ok[k]) raw[k] = load_q<4>(r.q, r.qs, vox[k] * r.C + 4 * q);
            }
            f32x4 best = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (ok[k]) {
                    const f32x4 o = one(vox[k], q, raw[k]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) best[e] = (o[e] > best[e] || o[e] != o[e]) ? o[e] : best[e];
                }
            *reinterpret_cast<f32x4*>(r.pooled + ((((size_t)n * Dp + pd) * Hp + ph) * Wp + pw) * r.C + 4 * q) = best;
        }
    }
}

// The codes of a pooled unit's raw tensor (r.raw, read) adjusted so that a pooling window's first maximum is the one of the exact tensor: where the rounded values
// of a window have another, the maximum's code becomes the neighbour of its element that gives the larger activation, and the codes that still reach it the neighbours
// that give the smaller one -- an element stays at one of its two neighbours, and on its side of the border (SIDE).  Those two conditions win: where the neighbour that a window needs lies
// across the border (the elements within a step of it), or SiLU falls where its argument grows, the maximum moves after all (the headline network on random data: 68 of 11 million windows).
// Without it a few per cent of the windows hand their whole gradient to another voxel: 4 - 19 % of the encoder's gradients (random data, 4 levels), 2 % at most with it.
// One lane = one window x 4 channels.
// The same network: 156 us per step, one more read of the pooled units' raw tensors.
template <bool SIDE>
__global__ __launch_bounds__(BT) void checkpoint8_windows_kernel(const RestoreArgs r, signed char* __restrict__ codes) {
    const float slope = r.act.get();
    const int Q = r.C >> 2, kd = r.kd;
    const int Dp = (r.D + kd - 1) / kd, Hp = (r.H + 1) >> 1, Wp = (r.W + 1) >> 1;
    const size_t total = (size_t)r.N * Dp * Hp * Wp * Q;
    for (size_t i = blockIdx.x * (size_t)BT + threadIdx.x; i < total; i += (size_t)gridDim.x * BT) {
        const int q = i % Q; size_t t = i / Q;
        const int pw = t % Wp; t /= Wp; const int ph = t % Hp; t /= Hp; const int pd = t % Dp; const int n = t / Dp;
        f32x4 x[8]; RawQ<4> raw[8]; size_t at[8]; bool ok[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int dz = k >> 2, d = pd * kd + dz, h = ph * 2 + ((k >> 1) & 1), w = pw * 2 + (k & 1);
            ok[k] = dz < kd && d < r.D && h < r.H && w < r.W;
            at[k] = ((((size_t)n * r.D + d) * r.H + h) * r.W + w) * r.C + 4 * q;
            raw[k] = {}; x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (ok[k]) { x[k] = *reinterpret_cast<const f32x4*>(r.raw + at[k]); raw[k] = load_q<4>(codes, r.qs, at[k]); }
        }
        const f32x4 sc = *reinterpret_cast<const f32x4*>(r.scale + 4 * q), sh = *reinterpret_cast<const f32x4*>(r.shift + 4 * q);
        unsigned changed = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float best = -INFINITY, bq = -INFINITY, oq[8];
            int m = -1, mq = -1;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float sl = act_slope_at(r.act, slope, (unsigned)(at[k] + e));
                const float o = act_fwd(__builtin_fmaf(x[k][e], sc[e], sh[e]), sl);
                float v[4];
                unpack_q<4>(raw[k], v);
                oq[k] = act_fwd(__builtin_fmaf(v[e], sc[e], sh[e]), sl);
                if (ok[k] && o > best) { best = o; m = k; }
                if (ok[k] && oq[k] > bq) { bq = oq[k]; mq = k; }
            }
            if (m == mq) continue;
            float top = 0.f;
#pragma unroll
            for (int pass = 0; pass < 2; ++pass)             // the maximum up, then the others down
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const bool mine = pass == 0 ? k == m : ok[k] && k != m && (k < m ? oq[k] >= top : oq[k] > top);
                    if (mine && raw[k].s > 0.f) {
                        const float sl = act_slope_at(r.act, slope, (unsigned)(at[k] + e));
                        Codes<1> c; c.scale = raw[k].s; c.q[0] = (signed char)(raw[k].q[0] >> (8 * e));
                        const float v0 = code_value<1>(c, 0);
                        c.q[0] = other_neighbour(c.q[0], x[k][e], v0);
                        const float z0 = __builtin_fmaf(v0, sc[e], sh[e]), z1 = __builtin_fmaf(code_value<1>(c, 0), sc[e], sh[e]);
                        const float o1 = act_fwd(z1, sl);
                        if ((pass == 0 ? o1 > oq[k] : o1 < oq[k]) && (!SIDE || (z0 > 0.f) == (z1 > 0.f))) {
                            oq[k] = o1;
                            raw[k].q[0] = (raw[k].q[0] & ~(0xffu << (8 * e))) | ((unsigned)(unsigned char)c.q[0] << (8 * e));
                            changed |= 1u << k;
                        }
                    }
                    if (pass == 0 && k == m) top = oq[k];
                }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (changed >> k & 1) *reinterpret_cast<unsigned*>(codes + at[k]) = raw[k].q[0];
    }
}

unsigned grid_for(size_t n, int V) {
    const size_t blocks = (n + (size_t)BT * V - 1) / ((size_t)BT * V);
    return (unsigned)(blocks < 2048 ? blocks : 2048);       // 8 workgroups of 4 waves per CU, grid-stride beyond
}

template <int DT, int V, bool NT, int RULE>
void pack_nt(const void* x, int ldc, size_t n, int C, signed char* q, float* scale, const Border& b, hipStream_t s) {
    typedef const typename Elem<DT>::T* P;
    if (ldc == C) hipLaunchKernelGGL((checkpoint8_pack_kernel<DT, V, true, NT, RULE>), dim3(grid_for(n, V)), dim3(BT), 0, s, (P)x, ldc, C, n, q, scale, b);
    else hipLaunchKernelGGL((checkpoint8_pack_kernel<DT, V, false, NT, RULE>), dim3(grid_for(n, V)), dim3(BT), 0, s, (P)x, ldc, C, n, q, scale, b);
}
template <int DT, int V, bool NT>
void unpack_nt(const signed char* q, const float* scale, size_t n, int C, void* y, int ldc, hipStream_t s) {
    typedef typename Elem<DT>::T* P;
    if (ldc == C) hipLaunchKernelGGL((checkpoint8_unpack_kernel<DT, V, true, NT>), dim3(grid_for(n, V)), dim3(BT), 0, s, q, scale, n, C, ldc, (P)y);
    else hipLaunchKernelGGL((checkpoint8_unpack_kernel<DT, V, false, NT>), dim3(grid_for(n, V)), dim3(BT), 0, s, q, scale, n, C, ldc, (P)y);
}
template <int DT, int V>
void pack_typed(const void* x, int ldc, size_t n, int C, signed char* q, float* scale, const Border& b, hipStream_t s) {
    if (b.rule == 1) pack_nt<DT, V, false, 1>(x, ldc, n, C, q, scale, b, s);
    else if (b.rule == 2) pack_nt<DT, V, false, V == 4 ? 2 : 0>(x, ldc, n, C, q, scale, b, s);        // (the fp32 executor's)
    else if (V > 1 && n * sizeof(typename Elem<DT>::T) >= CACHE_BYTES) pack_nt<DT, V, (V > 1), 0>(x, ldc, n, C, q, scale, b, s);
    else pack_nt<DT, V, false, 0>(x, ldc, n, C, q, scale, b, s);
}
template <int DT, int V>
void unpack_typed(const signed char* q, const float* scale, size_t n, int C, void* y, int ldc, hipStream_t s) {
    if (V > 1 && n * sizeof(typename Elem<DT>::T) >= CACHE_BYTES) unpack_nt<DT, V, (V > 1)>(q, scale, n, C, y, ldc, s);
    else unpack_nt<DT, V, false>(q, scale, n, C, y, ldc, s);
}

// a flat tensor of rows without gaps is cut into pieces whatever its channel count
bool wide(int dt, const void* p, int ldc, int C, size_t n, const void* q) {
    return (uintptr_t)q % wide_of(dt) == 0 && (ldc == C ? n % wide_of(dt) == 0 && aligned16(p) : wide_rows(dt, p, ldc, C));
}

}  // namespace

int launch_checkpoint8_pack(int dt, const void* x, int x_ldc, long long vox, int C, signed char* q, float* scale, const Border& border, hipStream_t s) {
    const size_t n = (size_t)vox * C;
    if (n == 0) return E3_OK;
    E3_REQUIRE(border.rule != 2 || (dt == DT_F32 && C % 4 == 0 && x_ldc == C && wide(dt, x, x_ldc, C, n, q) && aligned16(border.a) && aligned16(border.b)), E3_ERR_INVALID,
               "a checkpoint with channel constants: packed fp32 tensor with 16-byte rows expected");
    switch (dt * 2 + wide(dt, x, x_ldc, C, n, q)) {
        case 0: pack_typed<DT_F32, 1>(x, x_ldc, n, C, q, scale, border, s); break;
        case 1: pack_typed<DT_F32, 4>(x, x_ldc, n, C, q, scale, border, s); break;
        case 2: pack_typed<DT_BF16, 1>(x, x_ldc, n, C, q, scale, border, s); break;
        case 3: pack_typed<DT_BF16, 8>(x, x_ldc, n, C, q, scale, border, s); break;
        case 4: pack_typed<DT_F16, 1>(x, x_ldc, n, C, q, scale, border, s); break;
        default: pack_typed<DT_F16, 8>(x, x_ldc, n, C, q, scale, border, s); break;
    }
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

int launch_checkpoint8_unpack(int dt, const signed char* q, const float* scale, long long vox, int C, void* y, int y_ldc, hipStream_t s) {
    const size_t n = (size_t)vox * C;
    if (n == 0) return E3_OK;
    switch (dt * 2 + wide(dt, y, y_ldc, C, n, q)) {
        case 0: unpack_typed<DT_F32, 1>(q, scale, n, C, y, y_ldc, s); break;
        case 1: unpack_typed<DT_F32, 4>(q, scale, n, C, y, y_ldc, s); break;
        case 2: unpack_typed<DT_BF16, 1>(q, scale, n, C, y, y_ldc, s); break;
        case 3: unpack_typed<DT_BF16, 8>(q, scale, n, C, y, y_ldc, s); break;
        case 4: unpack_typed<DT_F16, 1>(q, scale, n, C, y, y_ldc, s); break;
        default: unpack_typed<DT_F16, 8>(q, scale, n, C, y, y_ldc, s); break;
    }
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

int launch_checkpoint8_windows(const RestoreArgs& r, signed char* codes, bool side, hipStream_t s) {
    E3_REQUIRE(r.C % 4 == 0, E3_ERR_INVALID, "channel counts must be multiples of 4");
    const size_t items = (size_t)r.N * ((r.D + r.kd - 1) / r.kd) * ((r.H + 1) / 2) * ((r.W + 1) / 2) * (r.C / 4), blocks = (items + BT - 1) / BT;
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    if (side) hipLaunchKernelGGL(checkpoint8_windows_kernel<true>, grid, dim3(BT), 0, s, r, codes);
    else hipLaunchKernelGGL(checkpoint8_windows_kernel<false>, grid, dim3(BT), 0, s, r, codes);
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

int launch_checkpoint8_act(const RestoreArgs& r, hipStream_t s) {
    E3_REQUIRE(r.C % 4 == 0 && r.a_ldc % 4 == 0, E3_ERR_INVALID, "channel counts must be multiples of 4");
    const int kd = r.pooled ? r.kd : 1;
    const size_t items = (size_t)r.N * ((r.D + kd - 1) / kd) * (r.pooled ? (r.H + 1) / 2 : r.H) * (r.pooled ? (r.W + 1) / 2 : r.W) * (r.C / 4);
    const size_t blocks = (items + BT - 1) / BT;
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    if (r.pooled) hipLaunchKernelGGL(checkpoint8_act_kernel<true>, grid, dim3(BT), 0, s, r);
    else hipLaunchKernelGGL(checkpoint8_act_kernel<false>, grid, dim3(BT), 0, s, r);
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

extern "C" {

int e3_checkpoint8_pack(void* stream, int dtype, const void* x, int x_ldc, long long voxels, int C, signed char* q, float* scale) {
    E3_REQUIRE(dtype >= 0 && dtype <= 2, E3_ERR_INVALID, "dtype must be E3_DT_F32, E3_DT_BF16 or E3_DT_F16");
    E3_REQUIRE(C >= 1 && voxels >= 0 && x_ldc >= C, E3_ERR_INVALID, "bad sizes");
    E3_REQUIRE(voxels == 0 || (x && q && scale), E3_ERR_INVALID, "null argument");
    return launch_checkpoint8_pack(dtype, x, x_ldc, voxels, C, q, scale, Border(), (hipStream_t)stream);
}

int e3_checkpoint8_unpack(void* stream, int dtype, const signed char* q, const float* scale, long long voxels, int C, void* y, int y_ldc) {
    E3_REQUIRE(dtype >= 0 && dtype <= 2, E3_ERR_INVALID, "dtype must be E3_DT_F32, E3_DT_BF16 or E3_DT_F16");
    E3_REQUIRE(C >= 1 && voxels >= 0 && y_ldc >= C, E3_ERR_INVALID, "bad sizes");
    E3_REQUIRE(voxels == 0 || (y && q && scale), E3_ERR_INVALID, "null argument");
    return launch_checkpoint8_unpack(dtype, q, scale, voxels, C, y, y_ldc, (hipStream_t)stream);
}

}  // extern "C"
