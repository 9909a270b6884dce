// Group norm with an activation over channels-last tensors (N, D, H, W, C), its gradients, and the same from an 8-bit checkpoint of its input.
//
// A group is cg = C / G consecutive channels of ONE sample, m = S * cg elements (S = D H W voxels):
//     z = (x - mean) rstd gamma + beta,  y = act(z);   rstd = (var + eps)^-1/2, var the mean of (x - mean)^2
//     dz = dy act'(z),  h = (x - mean) rstd,  dgamma = sum dz h,  dbeta = sum dz  (over samples and voxels)
//     dx = rstd (gamma dz - m1 - h m2),  m1 = mean over the group of gamma dz,  m2 = of gamma dz h
//
// All kernels are streaming passes with one mapping: a thread keeps V consecutive channels (V = 8: 16-byte accesses; V = 1 for rows that do not allow them) and
// walks the voxels of its workgroup's chunk, so that the per-channel constants stay in registers; consecutive threads take consecutive pieces of a voxel, then
// consecutive voxels.  A workgroup works on one chunk of one sample and, for more than 512 pieces per voxel, on one tile of its channels.
//   forward:   statistics (read x) -> finalise -> apply (read x, write y [, write the checkpoint])
//   backward:  reduce (read x, dy) -> finalise -> apply (read x, dy, write dx)
// Sums leave a workgroup as fp64 records [sample][chunk][..], merged in a fixed order: results do not depend on timing.
#include "checkpoint8.h"

#include "../../include/e3unet.h"

using namespace e3n;

namespace {

constexpr int MAX_T = 512;                   // threads of a workgroup, at most

struct GnArgs {
    const void* x; int x_ldc;                // the input, or (x == nullptr) its checkpoint
    const signed char* q; const float* qs;
    const void* dy; int dy_ldc;
    void* out; int out_ldc;                  // y, or dx
    signed char* q_out; float* qs_out;       // forward: the checkpoint that the apply pass writes along (or nullptr)
    const float* gamma; const float* beta;   // [C] or nullptr: 1, 0
    const float* mean; const float* rstd;    // [N][G]
    const float* m1; const float* m2;        // [N][G] (backward apply)
    float slope;
    int N, C, G, cg; long long S;
    int P, PT, tiles, R;                     // pieces per voxel, pieces per tile, tiles, voxels per workgroup step
    int chunks; long long chunk;             // chunks of a sample, voxels of a chunk
    int unit;                                // channels that the statistics pass adds up before it writes them (divides cg and V)
    double* part;                            // records (sum, sum of squares) [N][chunks][C / unit] | (sum dz, sum dz h) [N][chunks][C]
};

struct Where { int n, tile, r, p, c; long long v0, v1; bool on; };
template <int V> __device__ __forceinline__ Where where(const GnArgs& a) {
    Where w;
    const unsigned b = blockIdx.x, t = b / a.tiles;
    w.tile = b % a.tiles;
    w.n = t / a.chunks;
    const int k = t % a.chunks;
    w.r = threadIdx.x / a.PT;
    w.p = w.tile * a.PT + threadIdx.x % a.PT;
    w.c = w.p * V;
    w.v0 = k * a.chunk;
    w.v1 = w.v0 + a.chunk < a.S ? w.v0 + a.chunk : a.S;
    w.on = w.r < a.R && w.p < a.P;
    return w;
}

// one piece of the input
template <int DT, int V, bool CK> struct In {
    Raw<DT, V> r;
    __device__ __forceinline__ void load(const GnArgs& a, long long row, int c) { r = load_raw<DT, V>((const typename Elem<DT>::T*)a.x + (size_t)row * a.x_ldc + c); }
    __device__ __forceinline__ void get(float (&f)[V]) const { unpack_raw<DT, V>(r, f); }
};
template <int DT, int V> struct In<DT, V, true> {
    RawQ<V> r;
    __device__ __forceinline__ void load(const GnArgs& a, long long row, int c) { r = load_q<V>(a.q, a.qs, (size_t)row * a.C + c); }
    __device__ __forceinline__ void get(float (&f)[V]) const { unpack_q<V>(r, f); }
};

// Sums of `rows` x `units` pairs in LDS over the rows: L lanes share a unit (fixed order), lane 0 hands the sums on.
template <typename T, typename F> __device__ __forceinline__ void sum_rows(const T* a, const T* b, int rows, int units, F done) {
    int L = 64;
    while (L > 1 && units * L > (int)blockDim.x) L >>= 1;
    const int l = threadIdx.x & (L - 1);
    for (int u0 = 0; u0 < units; u0 += blockDim.x / L) {
        const int u = u0 + threadIdx.x / L;
        double s = 0.0, t = 0.0;
        if (u < units)
            for (int r = l; r < rows; r += L) { s += (double)a[r * units + u]; t += (double)b[r * units + u]; }
        for (int o = L >> 1; o >= 1; o >>= 1) { s += __shfl_xor(s, o); t += __shfl_xor(t, o); }
        if (l == 0 && u < units) done(u, s, t);
    }
}

// ------------------------------------------------------------------------------------------------ forward
// Sums and sums of squares in fp64: the variance is then a difference that loses nothing an fp32 input holds, whatever its mean.
template <int DT, int V>
__global__ __launch_bounds__(MAX_T) void gn_stats_kernel(const GnArgs a) {
    extern __shared__ double sh[];
    const Where w = where<V>(a);
    constexpr int U = 4;
    double s[V], t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = t[e] = 0.0;
    if (w.on)
        for (long long v = w.v0 + w.r; v < w.v1; v += U * a.R) {
            In<DT, V, false> in[U]; bool ok[U];
#pragma unroll
            for (int u = 0; u < U; ++u) { ok[u] = v + u * a.R < w.v1; in[u].r = Raw<DT, V>{}; if (ok[u]) in[u].load(a, w.n * a.S + v + u * a.R, w.c); }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[V];
                in[u].get(f);
#pragma unroll
                for (int e = 0; e < V; ++e) { const double d = f[e]; s[e] += d; t[e] = fma(d, d, t[e]); }      // (a piece that is not there is zeros)
            }
        }
    // channels of one unit are added up in the thread (all of them belong to one group), then the rows of the workgroup
#pragma unroll
    for (int k = 1; k < V; k <<= 1)
        if (a.unit > k)
#pragma unroll
            for (int e = 0; e < V; e += 2 * k) { s[e] += s[e + k]; t[e] += t[e + k]; }
    const int K = V / a.unit, units = a.PT * K;
    double* s2 = sh + a.R * units;
    if (w.r < a.R) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e % a.unit == 0) { const int i = w.r * units + (int)(threadIdx.x % a.PT) * K + e / a.unit; sh[i] = s[e]; s2[i] = t[e]; }
    }
    __syncthreads();
    const int all = a.C / a.unit, first = w.tile * units;
    double* o = a.part + (size_t)(blockIdx.x / a.tiles) * all * 2;
    sum_rows(sh, s2, a.R, units, [&](int u, double x, double y) { if (first + u < all) { o[(first + u) * 2] = x; o[(first + u) * 2 + 1] = y; } });
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// one wave per (sample, group)
__global__ __launch_bounds__(256) void gn_finalize_kernel(const double* __restrict__ part, int chunks, int units, int per, int groups, double inv_m, float eps,
                                                          float* __restrict__ mean, float* __restrict__ rstd) {
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (i >= groups) return;
    const int G = units / per, n = i / G, g = i % G;
    double s = 0.0, t = 0.0;
    for (int k = lane; k < chunks * per; k += 64) {
        const double* r = part + ((size_t)(n * (size_t)chunks + k / per) * units + g * per + k % per) * 2;
        s += r[0]; t += r[1];
    }
    s = wave_sum(s); t = wave_sum(t);
    if (lane == 0) {
        const double m = s * inv_m;
        double var = t * inv_m - m * m;
        if (var < 0.0) var = 0.0;                    // (a constant group; NaN stays NaN)
        mean[i] = (float)m;
        rstd[i] = (float)(1.0 / sqrt(var + (double)eps));
    }
}

// act(z): slope 0 ReLU, (0, 1] LeakyReLU / identity, ACT_SILU z * sigmoid(z)
template <bool SILU> __device__ __forceinline__ float activate(float z, float slope) {
    if constexpr (SILU) return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
    else return z <= 0.f ? (slope == 0.f ? 0.f : slope * z) : z;       // NaN stays NaN
}

template <int V> struct Consts { float mu[V], a[V], b[V]; };
template <int V> __device__ __forceinline__ Consts<V> constants(const GnArgs& a, int n, int c) {
    Consts<V> k;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = n * a.G + (c + e) / a.cg;
        k.mu[e] = a.mean[g];
        k.a[e] = a.rstd[g] * (a.gamma ? a.gamma[c + e] : 1.f);
        k.b[e] = a.beta ? a.beta[c + e] : 0.f;
    }
    return k;
}

template <int DT, int V, bool CK, bool SILU, bool KEEP>
__global__ __launch_bounds__(MAX_T) void gn_apply_kernel(const GnArgs a) {
    const Where w = where<V>(a);
    constexpr int U = 4;
    typedef typename Elem<DT>::T T;
    Consts<V> k{};
    if (w.on) k = constants<V>(a, w.n, w.c);
    // (KEEP: every lane goes round together -- the checkpoint's blocks are 8 lanes)
    for (long long vb = w.v0; vb < w.v1; vb += U * a.R) {
        In<DT, V, CK> in[U]; bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = vb + w.r + u * a.R;
            ok[u] = w.on && v < w.v1;
            in[u].r = {};
            if (ok[u]) in[u].load(a, w.n * a.S + v, w.c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V], o[V];
            in[u].get(f);
            const size_t row = (size_t)(w.n * a.S + vb + w.r + u * a.R);
            if constexpr (KEEP) {
                const Codes<V> c = encode_block<V>(f);
                if (ok[u]) store_codes<V>(c, a.q_out, a.qs_out, row * a.C + w.c);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = activate<SILU>(__builtin_fmaf(f[e] - k.mu[e], k.a[e], k.b[e]), a.slope);
            if (ok[u]) store_f32<DT, V>((T*)a.out + row * a.out_ldc + w.c, o);
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward
// dz = dy act'(z).  On which side of 0 a ReLU's z falls is decided as in exact arithmetic: z's rounding error is below 2^-21 of |(x - mean) rstd gamma|, and a z
// that small is formed again in fp64 (one element in a few hundred thousand).
template <bool SILU> __device__ __forceinline__ float dz_of(float x, float g, float mu, float rstd, float gamma, float beta, float a, float slope) {
    const float p = (x - mu) * a, z = p + beta;
    if constexpr (SILU) {
        const float sg = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
        return g * (sg * (1.f + z * (1.f - sg)));
    } else {
        bool pos = z > 0.f;
        if (fabsf(z) < fabsf(p) * 0x1p-21f) pos = ((double)x - (double)mu) * (double)rstd * (double)gamma + (double)beta > 0.0;
        return pos ? g : (slope == 0.f ? 0.f : slope * g);
    }
}

template <int V> struct ConstsB { float mu[V], rs[V], ga[V], be[V]; };
template <int V> __device__ __forceinline__ ConstsB<V> constants_b(const GnArgs& a, int n, int c) {
    ConstsB<V> k;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = n * a.G + (c + e) / a.cg;
        k.mu[e] = a.mean[g]; k.rs[e] = a.rstd[g];
        k.ga[e] = a.gamma ? a.gamma[c + e] : 1.f;
        k.be[e] = a.beta ? a.beta[c + e] : 0.f;
    }
    return k;
}

// Per-thread sums in fp32 over at most a chunk's voxels / R, everything behind them in fp64.
template <int DT, int V, bool CK, bool SILU>
__global__ __launch_bounds__(MAX_T) void gn_bwd_reduce_kernel(const GnArgs a) {
    extern __shared__ float shf[];
    const Where w = where<V>(a);
    constexpr int U = 2;
    typedef typename Elem<DT>::T T;
    float s[V], t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = t[e] = 0.f;
    if (w.on) {
        const ConstsB<V> k = constants_b<V>(a, w.n, w.c);
        for (long long v = w.v0 + w.r; v < w.v1; v += U * a.R) {
            In<DT, V, CK> in[U]; Raw<DT, V> dy[U]; bool ok[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ok[u] = v + u * a.R < w.v1;
                in[u].r = {}; dy[u] = {};
                const long long row = w.n * a.S + v + u * a.R;
                if (ok[u]) { in[u].load(a, row, w.c); dy[u] = load_raw<DT, V>((const T*)a.dy + (size_t)row * a.dy_ldc + w.c); }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[V], g[V];
                in[u].get(f); unpack_raw<DT, V>(dy[u], g);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float dz = dz_of<SILU>(f[e], g[e], k.mu[e], k.rs[e], k.ga[e], k.be[e], k.rs[e] * k.ga[e], a.slope);
                    const float h = (f[e] - k.mu[e]) * k.rs[e];
                    if (ok[u]) { s[e] += dz; t[e] = __builtin_fmaf(dz, h, t[e]); }
                }
            }
        }
    }
    const int units = a.PT * V;
    float* t2 = shf + a.R * units;
    if (w.r < a.R)
#pragma unroll
        for (int e = 0; e < V; ++e) { const int i = w.r * units + (int)(threadIdx.x % a.PT) * V + e; shf[i] = s[e]; t2[i] = t[e]; }
    __syncthreads();
    const int first = w.tile * units;
    double* o = a.part + (size_t)(blockIdx.x / a.tiles) * a.C * 2;
    sum_rows(shf, t2, a.R, units, [&](int u, double x, double y) { if (first + u < a.C) { o[(first + u) * 2] = x; o[(first + u) * 2 + 1] = y; } });
}

// waves [0, N G): m1, m2 of a group; waves [N G, N G + C): dgamma, dbeta of a channel
__global__ __launch_bounds__(256) void gn_bwd_finalize_kernel(const double* __restrict__ part, int N, int chunks, int C, int G, const float* __restrict__ gamma, double inv_m,
                                                              float* __restrict__ m1, float* __restrict__ m2, float* __restrict__ dgamma, float* __restrict__ dbeta) {
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, cg = C / G;
    double s = 0.0, t = 0.0;
    if (i < N * G) {
        const int n = i / G, c0 = (i % G) * cg;
        for (long long k = lane; k < (long long)chunks * cg; k += 64) {
            const int c = c0 + (int)(k % cg);
            const double* r = part + ((size_t)((size_t)n * chunks + k / cg) * C + c) * 2;
            const double g = gamma ? (double)gamma[c] : 1.0;
            s += g * r[0]; t += g * r[1];
        }
        s = wave_sum(s); t = wave_sum(t);
        if (lane == 0) { m1[i] = (float)(s * inv_m); m2[i] = (float)(t * inv_m); }
    } else if (i < N * G + C) {
        const int c = i - N * G;
        for (int k = lane; k < N * chunks; k += 64) { const double* r = part + ((size_t)k * C + c) * 2; s += r[0]; t += r[1]; }
        s = wave_sum(s); t = wave_sum(t);
        if (lane == 0) { if (dbeta) dbeta[c] = (float)s; if (dgamma) dgamma[c] = (float)t; }
    }
}

template <int DT, int V, bool CK, bool SILU>
__global__ __launch_bounds__(MAX_T) void gn_bwd_apply_kernel(const GnArgs a) {
    const Where w = where<V>(a);
    constexpr int U = 2;
    typedef typename Elem<DT>::T T;
    if (!w.on) return;
    const ConstsB<V> k = constants_b<V>(a, w.n, w.c);
    float m1[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { const int g = w.n * a.G + (w.c + e) / a.cg; m1[e] = a.m1[g]; m2[e] = a.m2[g]; }
    for (long long v = w.v0 + w.r; v < w.v1; v += U * a.R) {
        In<DT, V, CK> in[U]; Raw<DT, V> dy[U]; bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ok[u] = v + u * a.R < w.v1;
            in[u].r = {}; dy[u] = {};
            const long long row = w.n * a.S + v + u * a.R;
            if (ok[u]) { in[u].load(a, row, w.c); dy[u] = load_raw<DT, V>((const T*)a.dy + (size_t)row * a.dy_ldc + w.c); }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V], g[V], o[V];
            in[u].get(f); unpack_raw<DT, V>(dy[u], g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float dz = dz_of<SILU>(f[e], g[e], k.mu[e], k.rs[e], k.ga[e], k.be[e], k.rs[e] * k.ga[e], a.slope);
                const float h = (f[e] - k.mu[e]) * k.rs[e];
                o[e] = k.rs[e] * (__builtin_fmaf(k.ga[e], dz, -m1[e]) - h * m2[e]);
            }
            if (ok[u]) store_f32<DT, V>((T*)a.out + (size_t)(w.n * a.S + v + u * a.R) * a.out_ldc + w.c, o);
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
struct Shape { int N; long long S; int C, G; };

// mapping of a pass; `target`: workgroups that it asks for (at least one per sample and tile)
template <int V> void map_pass(GnArgs& a, const Shape& sh, int target, int U, bool keep) {
    a.N = sh.N; a.S = sh.S; a.C = sh.C; a.G = sh.G; a.cg = sh.C / sh.G;
    a.P = sh.C / V;
    a.tiles = (a.P + MAX_T - 1) / MAX_T;
    a.PT = (a.P + a.tiles - 1) / a.tiles;
    a.R = 256 / a.PT > 0 ? 256 / a.PT : 1;
    if (keep) {                              // whole blocks of 64 elements per workgroup step
        int k = 8;
        for (int p = a.PT; k > 1 && p % 2 == 0; p /= 2) k /= 2;
        a.R = (a.R + k - 1) / k * k;
    }
    long long most = target / ((long long)sh.N * a.tiles);
    if (most < 1) most = 1;
    const long long step = (long long)a.R * U;
    long long chunks = (sh.S + step - 1) / step;
    if (chunks > most) chunks = most;
    a.chunk = (sh.S + chunks - 1) / chunks;
    a.chunk = (a.chunk + a.R - 1) / a.R * a.R;
    a.chunks = (int)((sh.S + a.chunk - 1) / a.chunk);
}
dim3 grid_of(const GnArgs& a) { return dim3((unsigned)((long long)a.N * a.chunks * a.tiles)); }
dim3 block_of(const GnArgs& a) { return dim3((unsigned)((a.R * a.PT + 63) / 64 * 64)); }

constexpr int STATS_WGS = 2048, APPLY_WGS = 2048;

template <int V> int unit_of(int cg) {
    int u = V;
    while (cg % u) u >>= 1;
    return u;
}

template <int V> size_t fwd_part_doubles(const Shape& sh) {
    GnArgs a{}; map_pass<V>(a, sh, STATS_WGS, 4, false);
    return (size_t)sh.N * a.chunks * (sh.C / unit_of<V>(sh.C / sh.G)) * 2;
}
template <int V> size_t bwd_part_doubles(const Shape& sh) {
    GnArgs a{}; map_pass<V>(a, sh, STATS_WGS, 2, false);
    return (size_t)sh.N * a.chunks * sh.C * 2;
}
size_t max2(size_t a, size_t b) { return a > b ? a : b; }
size_t workspace_bytes(const Shape& sh) {
    size_t d = max2(fwd_part_doubles<1>(sh), bwd_part_doubles<1>(sh));
    if (sh.C % 8 == 0) d = max2(d, max2(fwd_part_doubles<8>(sh), bwd_part_doubles<8>(sh)));
    return align_up(d * sizeof(double), 256) + align_up((size_t)2 * sh.N * sh.G * sizeof(float), 256);
}

template <int DT, int V, bool CK> void launch_apply(GnArgs a, const Shape& sh, hipStream_t s) {
    const bool keep = a.q_out != nullptr;
    map_pass<V>(a, sh, APPLY_WGS, 4, keep);
    if (a.slope == ACT_SILU) {
        if constexpr (V == 8 && !CK) if (keep) { hipLaunchKernelGGL((gn_apply_kernel<DT, V, CK, true, true>), grid_of(a), block_of(a), 0, s, a); return; }
        hipLaunchKernelGGL((gn_apply_kernel<DT, V, CK, true, false>), grid_of(a), block_of(a), 0, s, a);
    } else {
        if constexpr (V == 8 && !CK) if (keep) { hipLaunchKernelGGL((gn_apply_kernel<DT, V, CK, false, true>), grid_of(a), block_of(a), 0, s, a); return; }
        hipLaunchKernelGGL((gn_apply_kernel<DT, V, CK, false, false>), grid_of(a), block_of(a), 0, s, a);
    }
}

template <int DT, int V> int forward(GnArgs a, const Shape& sh, float eps, float* mean, float* rstd, void* ws, hipStream_t s) {
    GnArgs st = a;
    map_pass<V>(st, sh, STATS_WGS, 4, false);
    st.unit = unit_of<V>(st.cg);
    st.part = (double*)ws;
    const int units = sh.C / st.unit;
    hipLaunchKernelGGL((gn_stats_kernel<DT, V>), grid_of(st), block_of(st), (size_t)st.R * st.PT * (V / st.unit) * 2 * sizeof(double), s, st);
    hipLaunchKernelGGL(gn_finalize_kernel, dim3((sh.N * sh.G + 3) / 4), dim3(256), 0, s, st.part, st.chunks, units, st.cg / st.unit, sh.N * sh.G,
                       1.0 / ((double)sh.S * st.cg), eps, mean, rstd);
    a.mean = mean; a.rstd = rstd;
    // the checkpoint rides in the apply pass where its blocks are whole there; otherwise it is a pass of its own
    signed char* q = a.q_out; float* qs = a.qs_out;
    GnArgs m{}; map_pass<V>(m, sh, APPLY_WGS, 4, true);
    const bool fused = q && V == 8 && m.tiles == 1 && m.R * m.PT <= MAX_T && ((unsigned long long)sh.S * sh.C) % CK_BLOCK == 0 && ((uintptr_t)q & 7) == 0;
    if (q && !fused) { const int rc = launch_checkpoint8_pack(DT, a.x, a.x_ldc, (long long)sh.N * sh.S, sh.C, q, qs, s); if (rc) return rc; }
    if (!fused) a.q_out = nullptr;
    launch_apply<DT, V, false>(a, sh, s);
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

template <int DT, int V, bool CK> int backward(GnArgs a, const Shape& sh, float* dgamma, float* dbeta, void* ws, hipStream_t s) {
    GnArgs st = a;
    map_pass<V>(st, sh, STATS_WGS, 2, false);
    st.part = (double*)ws;
    float* m1 = (float*)((char*)ws + align_up((size_t)sh.N * st.chunks * sh.C * 2 * sizeof(double), 256));
    float* m2 = m1 + (size_t)sh.N * sh.G;
    const size_t lds = (size_t)st.R * st.PT * V * 2 * sizeof(float);
    if (a.slope == ACT_SILU) hipLaunchKernelGGL((gn_bwd_reduce_kernel<DT, V, CK, true>), grid_of(st), block_of(st), lds, s, st);
    else hipLaunchKernelGGL((gn_bwd_reduce_kernel<DT, V, CK, false>), grid_of(st), block_of(st), lds, s, st);
    hipLaunchKernelGGL(gn_bwd_finalize_kernel, dim3((sh.N * sh.G + sh.C + 3) / 4), dim3(256), 0, s, st.part, sh.N, st.chunks, sh.C, sh.G, a.gamma,
                       1.0 / ((double)sh.S * st.cg), m1, m2, dgamma, dbeta);
    map_pass<V>(a, sh, APPLY_WGS, 2, false);
    a.m1 = m1; a.m2 = m2;
    if (a.slope == ACT_SILU) hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, V, CK, true>), grid_of(a), block_of(a), 0, s, a);
    else hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, V, CK, false>), grid_of(a), block_of(a), 0, s, a);
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

bool act_ok(float slope) { return (slope >= 0.f && slope <= 1.f) || slope == ACT_SILU; }

// sizes of a call: 0, or the error that e3_last_error() describes
int check_shape(int dtype, int N, int D, int H, int W, int C, int G, float slope, Shape& sh) {
    E3_REQUIRE(dtype >= 0 && dtype <= 2, E3_ERR_INVALID, "dtype must be E3_DT_F32, E3_DT_BF16 or E3_DT_F16");
    E3_REQUIRE(N >= 1 && D >= 1 && H >= 1 && W >= 1 && C >= 1, E3_ERR_INVALID, "sizes must be at least 1");
    E3_REQUIRE(G >= 1 && C % G == 0, E3_ERR_INVALID, "num_groups must divide the channel count");
    E3_REQUIRE(act_ok(slope), E3_ERR_UNSUPPORTED, "activation slope must be in [0, 1], or 2 for SiLU");
    sh.N = N; sh.S = (long long)D * H * W; sh.C = C; sh.G = G;
    E3_REQUIRE((long long)N * ((C + MAX_T - 1) / MAX_T) <= (1ll << 30) && (long long)N * G + C < (1ll << 31), E3_ERR_UNSUPPORTED, "too many samples");
    return E3_OK;
}

}  // namespace

extern "C" {

size_t e3_group_norm_workspace_bytes(int N, int D, int H, int W, int C, int G) {
    Shape sh;
    if (check_shape(0, N, D, H, W, C, G, 0.f, sh)) return 0;
    return workspace_bytes(sh);
}

int e3_group_norm_act_fwd(void* stream, int dtype, const void* x, int x_ldc, const float* gamma, const float* beta, float eps, float act_slope, void* y, int y_ldc,
                          float* mean, float* rstd, signed char* q, float* q_scale, int N, int D, int H, int W, int C, int G, void* workspace, size_t workspace_bytes_) {
    Shape sh;
    const int rc = check_shape(dtype, N, D, H, W, C, G, act_slope, sh);
    if (rc) return rc;
    E3_REQUIRE(x && y && mean && rstd && workspace, E3_ERR_INVALID, "null argument");
    E3_REQUIRE((q == nullptr) == (q_scale == nullptr), E3_ERR_INVALID, "a checkpoint is codes and scales");
    E3_REQUIRE(x_ldc >= C && y_ldc >= C, E3_ERR_INVALID, "rows are shorter than the channel count");
    E3_REQUIRE(eps >= 0.f, E3_ERR_INVALID, "eps must not be negative");
    E3_REQUIRE(workspace_bytes_ >= workspace_bytes(sh), E3_ERR_WORKSPACE, "workspace too small");
    GnArgs a{};
    a.x = x; a.x_ldc = x_ldc; a.out = y; a.out_ldc = y_ldc; a.gamma = gamma; a.beta = beta; a.slope = act_slope; a.q_out = q; a.qs_out = q_scale;
    const bool v8 = rows_by_8(dtype, x, x_ldc, C) && rows_by_8(dtype, y, y_ldc, C);
    const hipStream_t s = (hipStream_t)stream;
    switch (dtype * 2 + v8) {
        case 0: return forward<DT_F32, 1>(a, sh, eps, mean, rstd, workspace, s);
        case 1: return forward<DT_F32, 8>(a, sh, eps, mean, rstd, workspace, s);
        case 2: return forward<DT_BF16, 1>(a, sh, eps, mean, rstd, workspace, s);
        case 3: return forward<DT_BF16, 8>(a, sh, eps, mean, rstd, workspace, s);
        case 4: return forward<DT_F16, 1>(a, sh, eps, mean, rstd, workspace, s);
        default: return forward<DT_F16, 8>(a, sh, eps, mean, rstd, workspace, s);
    }
}

int e3_group_norm_act_apply(void* stream, int dtype, const void* x, int x_ldc, const signed char* q, const float* q_scale, const float* mean, const float* rstd,
                            const float* gamma, const float* beta, float act_slope, void* y, int y_ldc, int N, int D, int H, int W, int C, int G) {
    Shape sh;
    const int rc = check_shape(dtype, N, D, H, W, C, G, act_slope, sh);
    if (rc) return rc;
    E3_REQUIRE(y && mean && rstd && (x || (q && q_scale)), E3_ERR_INVALID, "null argument");
    E3_REQUIRE((!x || x_ldc >= C) && y_ldc >= C, E3_ERR_INVALID, "rows are shorter than the channel count");
    GnArgs a{};
    a.x = x; a.x_ldc = x_ldc; a.q = q; a.qs = q_scale; a.out = y; a.out_ldc = y_ldc; a.mean = mean; a.rstd = rstd; a.gamma = gamma; a.beta = beta; a.slope = act_slope;
    const bool v8 = (x ? rows_by_8(dtype, x, x_ldc, C) : C % 8 == 0 && ((uintptr_t)q & 7) == 0) && rows_by_8(dtype, y, y_ldc, C);
    const hipStream_t s = (hipStream_t)stream;
    switch ((dtype * 2 + v8) * 2 + (x == nullptr)) {
        case 0: launch_apply<DT_F32, 1, false>(a, sh, s); break;
        case 1: launch_apply<DT_F32, 1, true>(a, sh, s); break;
        case 2: launch_apply<DT_F32, 8, false>(a, sh, s); break;
        case 3: launch_apply<DT_F32, 8, true>(a, sh, s); break;
        case 4: launch_apply<DT_BF16, 1, false>(a, sh, s); break;
        case 5: launch_apply<DT_BF16, 1, true>(a, sh, s); break;
        case 6: launch_apply<DT_BF16, 8, false>(a, sh, s); break;
        case 7: launch_apply<DT_BF16, 8, true>(a, sh, s); break;
        case 8: launch_apply<DT_F16, 1, false>(a, sh, s); break;
        case 9: launch_apply<DT_F16, 1, true>(a, sh, s); break;
        case 10: launch_apply<DT_F16, 8, false>(a, sh, s); break;
        default: launch_apply<DT_F16, 8, true>(a, sh, s); break;
    }
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

int e3_group_norm_act_bwd(void* stream, int dtype, const void* x, int x_ldc, const signed char* q, const float* q_scale, const float* mean, const float* rstd,
                          const float* gamma, const float* beta, float act_slope, const void* dy, int dy_ldc, void* dx, int dx_ldc, float* dgamma, float* dbeta,
                          int N, int D, int H, int W, int C, int G, void* workspace, size_t workspace_bytes_) {
    Shape sh;
    const int rc = check_shape(dtype, N, D, H, W, C, G, act_slope, sh);
    if (rc) return rc;
    E3_REQUIRE(dy && dx && mean && rstd && workspace && (x || (q && q_scale)), E3_ERR_INVALID, "null argument");
    E3_REQUIRE((!x || x_ldc >= C) && dy_ldc >= C && dx_ldc >= C, E3_ERR_INVALID, "rows are shorter than the channel count");
    E3_REQUIRE(workspace_bytes_ >= workspace_bytes(sh), E3_ERR_WORKSPACE, "workspace too small");
    GnArgs a{};
    a.x = x; a.x_ldc = x_ldc; a.q = q; a.qs = q_scale; a.dy = dy; a.dy_ldc = dy_ldc; a.out = dx; a.out_ldc = dx_ldc;
    a.mean = mean; a.rstd = rstd; a.gamma = gamma; a.beta = beta; a.slope = act_slope;
    const bool v8 = (x ? rows_by_8(dtype, x, x_ldc, C) : C % 8 == 0 && ((uintptr_t)q & 7) == 0) && rows_by_8(dtype, dy, dy_ldc, C) && rows_by_8(dtype, dx, dx_ldc, C);
    const hipStream_t s = (hipStream_t)stream;
    switch ((dtype * 2 + v8) * 2 + (x == nullptr)) {
        case 0: return backward<DT_F32, 1, false>(a, sh, dgamma, dbeta, workspace, s);
        case 1: return backward<DT_F32, 1, true>(a, sh, dgamma, dbeta, workspace, s);
        case 2: return backward<DT_F32, 8, false>(a, sh, dgamma, dbeta, workspace, s);
        case 3: return backward<DT_F32, 8, true>(a, sh, dgamma, dbeta, workspace, s);
        case 4: return backward<DT_BF16, 1, false>(a, sh, dgamma, dbeta, workspace, s);
        case 5: return backward<DT_BF16, 1, true>(a, sh, dgamma, dbeta, workspace, s);
        case 6: return backward<DT_BF16, 8, false>(a, sh, dgamma, dbeta, workspace, s);
        case 7: return backward<DT_BF16, 8, true>(a, sh, dgamma, dbeta, workspace, s);
        case 8: return backward<DT_F16, 1, false>(a, sh, dgamma, dbeta, workspace, s);
        case 9: return backward<DT_F16, 1, true>(a, sh, dgamma, dbeta, workspace, s);
        case 10: return backward<DT_F16, 8, false>(a, sh, dgamma, dbeta, workspace, s);
        default: return backward<DT_F16, 8, true>(a, sh, dgamma, dbeta, workspace, s);
    }
}

}  // extern "C"
