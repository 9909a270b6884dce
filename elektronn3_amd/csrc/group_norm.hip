// Group norm with an activation over channels-last tensors (N, D, H, W, C), its gradients, and the same from an 8-bit checkpoint of its input.
//
// A group is cg = C / G consecutive channels of ONE sample, m = S * cg elements (S = D H W voxels):
//     z = (x - mean) rstd gamma + beta,  y = act(z);   rstd = (var + eps)^-1/2, var the mean of (x - mean)^2
//     dz = dy act'(z),  h = (x - mean) rstd,  dgamma = sum dz h,  dbeta = sum dz  (over samples and voxels)
//     dx = rstd (gamma dz - m1 - h m2),  m1 = mean over the group of gamma dz,  m2 = of gamma dz h
//
// All kernels are streaming passes with one mapping: a thread keeps V consecutive channels (16 bytes: 4 fp32, 8 16-bit elements; V = 1 for rows that do not allow it) and
// walks the voxels of its workgroup's chunk, so that the per-channel constants stay in registers; consecutive threads take consecutive pieces of a voxel, then
// consecutive voxels.  A workgroup works on one chunk of one sample and, for more than 512 pieces per voxel, on one tile of its channels.  UN is the number of
// consecutive channels of a piece that surely share a group (8, 4 or 1): V / UN constants or sums per thread instead of V, which decides the register count.
//   forward:   statistics (read x) -> apply (read x, write y [, write the checkpoint])
//   backward:  reduce (read x, dy) -> apply (read x, dy, write dx)
//   small groups: one launch each way, the pieces held in registers in between (the forward's not where too many groups share a line: map_group_fwd)
// What bounds them: HBM, or the memory-side cache, for tensors above some 16 MB, where the second read of the inputs is the price of two passes; below, the latency of
// two dependent launches (4 - 6 us each), and of the calling program.  2 x 64 x 128 x 128 x 32, 8 groups:
//   fp32 forward 46 us (5.8 TB/s) + 83 (6.5), fp32 backward from a checkpoint 64 (5.3) + 97 (6.3), bf16 backward 51 (5.3) + 66 (6.1)
// Sums leave a workgroup as fp64 records [sample][chunk][..], merged in a fixed order: results do not depend on timing.  Every workgroup of the apply pass
// merges its sample's records itself (a few tens of KB out of L2, about 1 us) instead of waiting for a third launch in between; where the records of a
// sample are more than MERGE_MAX a finalising launch does it.
#include <type_traits>

#include "checkpoint8.h"

#include "../../include/e3unet.h"

using namespace e3n;

namespace {

constexpr int MAX_T = 512;                   // threads of a workgroup, at most
// pieces that a thread has in flight: a pass that reads one tensor, one that reads two
template <int V> constexpr int U1 = V == 8 ? 4 : 8;
template <int V> constexpr int U2 = V == 8 ? 2 : 4;

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
    // records: (sum, sum of squares) [N][chunks][G], or [C / UN] where groups lie across tiles | (sum dz, sum dz h) [N][chunks][C]
    double* part;
    double* gpart;                           // backward: (sum gamma dz, sum gamma dz h) [N][chunks][G], or nullptr where groups lie across tiles
    // apply passes that merge the records themselves (rec != nullptr)
    const double* rec; int rec_chunks;       // [N][rec_chunks][G] pairs
    double inv_m; float eps;
    float* mean_out; float* rstd_out;        // forward: the statistics, written by the first workgroup of a sample
    const double* cpart; float* dgamma; float* dbeta; int sum_wgs;      // backward: the first sum_wgs workgroups sum the channel records [N * rec_chunks][C]
};

struct Where { int n, tile, r, p, c; long long v0, v1; bool on; };
template <int V> __device__ __forceinline__ Where where(const GnArgs& a, unsigned b) {
    Where w;
    const unsigned t = b / a.tiles;
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
template <int DT, int V, bool CK, bool NT = false> struct In {
    Raw<DT, V> r;
    __device__ __forceinline__ void load(const GnArgs& a, long long row, int c) { r = load_raw<DT, V, NT>((const typename Elem<DT>::T*)a.x + (size_t)row * a.x_ldc + c); }
    __device__ __forceinline__ void get(float (&f)[V]) const { unpack_raw<DT, V>(r, f); }
};
template <int DT, int V, bool NT> struct In<DT, V, true, NT> {
    RawQ<V> r;
    __device__ __forceinline__ void load(const GnArgs& a, long long row, int c) { r = load_q<V>(a.q, a.qs, (size_t)row * a.C + c); }
    __device__ __forceinline__ void get(float (&f)[V]) const { unpack_q<V>(r, f); }
};

// v of the lane that a DPP control names
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, false);
    return __hiloint2double(hi, lo);
}
// inside a row of 16 lanes with DPP (pair, quad, half row, row: each step's partner holds the other half's sum), beyond with permutes
__device__ __forceinline__ double wave_sum(double v) {
    v += dpp<0xB1>(v); v += dpp<0x4E>(v); v += dpp<0x141>(v); v += dpp<0x140>(v);
    v += __shfl_xor(v, 16); v += __shfl_xor(v, 32);
    return v;
}

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

// Sums of `per` consecutive pairs in LDS for each of `groups` groups, in the same manner
template <typename F> __device__ __forceinline__ void sum_groups(const double* a, const double* b, int stride, int per, int groups, F done) {
    int L = 64;
    while (L > 1 && (groups * L > (int)blockDim.x || L >= 2 * per)) L >>= 1;
    const int l = threadIdx.x & (L - 1);
    for (int g0 = 0; g0 < groups; g0 += blockDim.x / L) {
        const int g = g0 + threadIdx.x / L;
        double s = 0.0, t = 0.0;
        if (g < groups)
            for (int k = l; k < per; k += L) { s += a[(g * per + k) * stride]; t += b[(g * per + k) * stride]; }
        for (int o = L >> 1; o >= 1; o >>= 1) { s += __shfl_xor(s, o); t += __shfl_xor(t, o); }
        if (l == 0 && g < groups) done(g, s, t);
    }
}

// Merges a sample's records [chunks][units] of pairs, a unit for each group, into sh[2 g], sh[2 g + 1].  Threads read the records in memory order and
// keep their unit; rows are added in a fixed order.  sh: 2 blockDim + 2 units doubles at least.
__device__ __forceinline__ void merge_records(const double* rec, int chunks, int units, double* sh) {
    const int rows = blockDim.x / units, T = rows * units, n = chunks * units;
    double s = 0.0, t = 0.0;
    constexpr int M = 8;                     // records in flight (4: 0.5 us more for 4096 records)
    if ((int)threadIdx.x < T)
        for (int j = threadIdx.x; j < n; j += M * T) {
            double2 v[M];
#pragma unroll
            for (int k = 0; k < M; ++k) { v[k] = make_double2(0.0, 0.0); if (j + k * T < n) v[k] = *reinterpret_cast<const double2*>(rec + 2 * (size_t)(j + k * T)); }
#pragma unroll
            for (int k = 0; k < M; ++k) { s += v[k].x; t += v[k].y; }
        }
    double* sums = sh + 2 * blockDim.x;
    if ((int)threadIdx.x < T) { sh[threadIdx.x] = s; sh[T + threadIdx.x] = t; }
    __syncthreads();
    sum_rows(sh, sh + T, rows, units, [&](int u, double x, double y) { sums[2 * u] = x; sums[2 * u + 1] = y; });
    __syncthreads();
    for (int g = threadIdx.x; g < 2 * units; g += blockDim.x) sh[g] = sums[g];
    __syncthreads();
}
// records of a sample that the apply pass merges itself (128 KB out of L2): at 5376 of them 22.0 us for a backward of 2 x 7 x 82 x 19 x 168 in 21 groups instead of 23.4 with a
// finaliser's launch in between, which costs the host 4 us more; 16384 (512 chunks of 32 groups) the same as the launch, 42.0 : 40.1 in fp32, 29.3 : 31.2 in fp16
constexpr int MERGE_MAX = 8192;
constexpr int MERGE_UNITS = 128;             // ... of at most so many units (a workgroup has 192 threads or more)

__device__ __forceinline__ void statistics_of(double s, double t, double inv_m, float eps, float& mean, float& rstd) {
    const double m = s * inv_m;
    double var = t * inv_m - m * m;
    if (var < 0.0) var = 0.0;                        // (a constant group; NaN stays NaN)
    mean = (float)m;
    rstd = (float)(1.0 / sqrt(var + (double)eps));
}

// sums of a workgroup of 256 threads, in thread 0
__device__ __forceinline__ void block_sum2(double& s, double& t) {
    __shared__ double sh[8];
    s = wave_sum(s); t = wave_sum(t);
    if ((threadIdx.x & 63) == 0) { sh[2 * (threadIdx.x >> 6)] = s; sh[2 * (threadIdx.x >> 6) + 1] = t; }
    __syncthreads();
    s = (sh[0] + sh[2]) + (sh[4] + sh[6]);
    t = (sh[1] + sh[3]) + (sh[5] + sh[7]);
}

// one workgroup per (sample, group)
__global__ __launch_bounds__(256) void gn_finalize_kernel(const double* __restrict__ part, int chunks, int units, int per, double inv_m, float eps,
                                                          float* __restrict__ mean, float* __restrict__ rstd) {
    const int i = blockIdx.x, G = units / per, n = i / G, g = i % G;
    double s = 0.0, t = 0.0;
    for (int k = threadIdx.x; k < chunks * per; k += 256) {
        const double* r = part + ((size_t)(n * (size_t)chunks + k / per) * units + g * per + k % per) * 2;
        s += r[0]; t += r[1];
    }
    block_sum2(s, t);
    if (threadIdx.x == 0) statistics_of(s, t, inv_m, eps, mean[i], rstd[i]);
}

// the constants of a piece: a = rstd gamma
template <int V, int UN> struct Consts { float mu[V / UN], rs[V / UN], a[V], b[V]; };
template <int V, int UN> __device__ __forceinline__ Consts<V, UN> constants(const GnArgs& a, const float* mean, const float* rstd, int c) {      // the sample's statistics
    Consts<V, UN> k;
#pragma unroll
    for (int e = 0; e < V; ++e) { k.a[e] = a.gamma ? a.gamma[c + e] : 1.f; k.b[e] = a.beta ? a.beta[c + e] : 0.f; }
#pragma unroll
    for (int u = 0; u < V / UN; ++u) { const int g = (c + u * UN) / a.cg; k.mu[u] = mean[g]; k.rs[u] = rstd[g]; }
#pragma unroll
    for (int e = 0; e < V; ++e) k.a[e] *= k.rs[e / UN];
    return k;
}

// act(z): slope 0 ReLU, (0, 1] LeakyReLU / identity, ACT_SILU z * sigmoid(z)
template <bool SILU> __device__ __forceinline__ float activate(float z, float slope) {
    if constexpr (SILU) return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
    else return z <= 0.f ? (slope == 0.f ? 0.f : slope * z) : z;       // NaN stays NaN
}

// |z| below which the fp32 evaluation of z may have the wrong sign: its rounding error is below 2^-21 of |(x - mean) a|, which is |beta| up to a factor 2 there
template <int V, int UN> __device__ __forceinline__ float border_of(const Consts<V, UN>& k) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) m = fmaxf(m, fabsf(k.b[e]));
    return m * 0x1p-20f;
}
__device__ __forceinline__ bool positive_exact(float x, float mu, float rs, double ga, double be) { return ((double)x - (double)mu) * (double)rs * ga + be > 0.0; }

// The codes of a piece moved to the side of the activation's border that their elements are on (see checkpoint8.h); pieces with an element at the border itself are
// decided again in fp64, in a rolled loop (unrolled, hipcc computes its operands in front of the voxel loop and keeps them in registers).
template <int V, int UN>
__device__ __forceinline__ void keep_side(const GnArgs& a, int c, const float (&x)[V], const Consts<V, UN>& k, float border, Codes<V>& q) {
    if (!(q.scale > 0.f)) return;
    float least = 3.4e38f, v[V];
    unsigned moved = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        v[e] = code_value<V>(q, e);
        const float z = __builtin_fmaf(x[e] - k.mu[e / UN], k.a[e], k.b[e]), zq = __builtin_fmaf(v[e] - k.mu[e / UN], k.a[e], k.b[e]);
        least = fminf(least, fminf(fabsf(z), fabsf(zq)));
        moved |= ((z > 0.f) != (zq > 0.f)) ? 1u << e : 0u;
    }
    if (least < border) {
        moved = 0;
#pragma unroll 1
        for (int e = 0; e < V; ++e) {
            float xe = x[0], ve = v[0], mu = k.mu[0], rs = k.rs[0];
#pragma unroll
            for (int j = 1; j < V; ++j) { xe = e == j ? x[j] : xe; ve = e == j ? v[j] : ve; mu = e == j ? k.mu[j / UN] : mu; rs = e == j ? k.rs[j / UN] : rs; }
            const double ga = a.gamma ? (double)a.gamma[c + e] : 1.0, be = a.beta ? (double)a.beta[c + e] : 0.0;
            moved |= positive_exact(xe, mu, rs, ga, be) != positive_exact(ve, mu, rs, ga, be) ? 1u << e : 0u;
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (moved >> e & 1) q.q[e] = other_neighbour(q.q[e], x[e], v[e]);
}

// ------------------------------------------------------------------------------------------------ forward
// One read of x: 46 us for 268 MB.  Sums and sums of squares in fp64 (the vector pipes have room: 8 operations per element): the variance is then a difference that is off by 1e-16 (mean / std)^2 -- less than the inputs' own rounding up to mean / std = 1e5.
template <int V, int UN> struct Moments {
    double s[V / UN], t[V / UN];
    __device__ __forceinline__ Moments() {
#pragma unroll
        for (int u = 0; u < V / UN; ++u) s[u] = t[u] = 0.0;
    }
    __device__ __forceinline__ void add(const float (&f)[V]) {
#pragma unroll
        for (int e = 0; e < V; ++e) { const double d = f[e]; s[e / UN] += d; t[e / UN] = fma(d, d, t[e / UN]); }
    }
};

template <int DT, int V, int UN>
__global__ __launch_bounds__(MAX_T) void gn_stats_kernel(const GnArgs a) {
    extern __shared__ double sh[];
    const Where w = where<V>(a, blockIdx.x);
    constexpr int U = U1<V>;
    Moments<V, UN> m;
    if (w.on)
        for (long long v = w.v0 + w.r; v < w.v1; v += U * a.R) {
            In<DT, V, false> in[U];
#pragma unroll
            for (int u = 0; u < U; ++u) { in[u].r = {}; if (v + u * a.R < w.v1) in[u].load(a, w.n * a.S + v + u * a.R, w.c); }
#pragma unroll
            for (int u = 0; u < U; ++u) { float f[V]; in[u].get(f); m.add(f); }        // (a piece that is not there is zeros)
        }
    constexpr int K = V / UN;
    const int units = a.PT * K;
    double* s2 = sh + a.R * units;
    if (w.r < a.R) {
#pragma unroll
        for (int u = 0; u < K; ++u) { const int i = w.r * units + (int)(threadIdx.x % a.PT) * K + u; sh[i] = m.s[u]; s2[i] = m.t[u]; }
    }
    __syncthreads();
    if (a.tiles > 1) {
        const int all = a.C / UN, first = w.tile * units;
        double* o = a.part + (size_t)(blockIdx.x / a.tiles) * all * 2;
        sum_rows(sh, s2, a.R, units, [&](int u, double x, double y) { if (first + u < all) { o[(first + u) * 2] = x; o[(first + u) * 2 + 1] = y; } });
    } else {
        double* o = a.part + (size_t)blockIdx.x * a.G * 2;
        sum_rows(sh, s2, a.R, units, [&](int u, double x, double y) { sh[u] = x; s2[u] = y; });      // (a unit's column is read by its own lanes only)
        __syncthreads();
        sum_groups(sh, s2, 1, a.cg / UN, a.G, [&](int g, double x, double y) { o[2 * g] = x; o[2 * g + 1] = y; });
    }
}

// NT: the input is read for the last time and the output written past the caches (non-temporal), which leaves the memory-side cache to what the statistics or
// reduce pass has just read: forward of 2 x 64 x 128 x 128 x 32 in fp32 168 -> 130 us, in bf16 92 -> 72, a pass from the checkpoint 84 -> 54; with the next reader of y
// timed along 233 -> 217, 133 -> 118, at 34 MB 38.2 -> 36.8.  From a tensor that no pass has read before it loses (bf16 53 -> 58): not there.
template <int DT, int V, int UN, bool CK, bool SILU, bool KEEP, bool NT>
__global__ __launch_bounds__(MAX_T) void gn_apply_kernel(const GnArgs a) {
    extern __shared__ double sh[];
    const Where w = where<V>(a, blockIdx.x);
    constexpr int U = U1<V>;
    typedef typename Elem<DT>::T T;
    In<DT, V, CK, NT> in[U]; bool ok[U];
    auto load = [&](long long vb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = vb + w.r + u * a.R;
            ok[u] = w.on && v < w.v1;
            in[u].r = {};
            if (ok[u]) in[u].load(a, w.n * a.S + v, w.c);
        }
    };
    // from the chunk's end to its start: what the statistics pass read last is still in the memory-side cache.  The first step is requested in front of the merge
    const int step = U * a.R;
    long long vb = w.v0 + (w.v1 - w.v0 - 1) / step * step;
    load(vb);
    const float* mean = a.mean + (size_t)w.n * a.G; const float* rstd = a.rstd + (size_t)w.n * a.G;
    if (a.rec) {                             // (uniform)
        merge_records(a.rec + (size_t)w.n * a.rec_chunks * a.G * 2, a.rec_chunks, a.G, sh);
        float* st = reinterpret_cast<float*>(sh + 2 * blockDim.x);
        for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
            statistics_of(sh[2 * g], sh[2 * g + 1], a.inv_m, a.eps, st[g], st[a.G + g]);
            if (w.v0 == 0 && w.tile == 0) { a.mean_out[(size_t)w.n * a.G + g] = st[g]; a.rstd_out[(size_t)w.n * a.G + g] = st[a.G + g]; }
        }
        __syncthreads();
        mean = st; rstd = st + a.G;
    }
    Consts<V, UN> k{};
    if (w.on) k = constants<V, UN>(a, mean, rstd, w.c);
    const float border = border_of<V, UN>(k);
    // (KEEP: every lane goes round together -- a checkpoint's block is 8 or 16 lanes)
    for (;;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V], o[V];
            in[u].get(f);
            const size_t row = (size_t)(w.n * a.S + vb + w.r + u * a.R);
            if constexpr (KEEP) {
                Codes<V> c = encode_block<V>(f);
                if constexpr (!SILU) if (ok[u] && a.slope != 1.f) keep_side<V, UN>(a, w.c, f, k, border, c);
                if (ok[u]) store_codes<V>(c, a.q_out, a.qs_out, row * a.C + w.c);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = activate<SILU>(__builtin_fmaf(f[e] - k.mu[e / UN], k.a[e], k.b[e]), a.slope);
            if (ok[u]) store_f32<DT, V, NT>((T*)a.out + row * a.out_ldc + w.c, o);
        }
        vb -= step;
        if (vb < w.v0) break;
        load(vb);
    }
}

// Small groups: a workgroup takes ONE sample's bundle of whole groups (one group, or the groups of a piece), keeps its pieces in registers from the
// statistics to the stores, and needs no records and no second launch.  HELD<V> pieces per thread; thread = (voxel r, piece p) as above, PT pieces to a bundle.
// 1 x 4 x 8 x 8 x 128 in 8 groups, fp16: 5.4 us (two launches take 10 - 12 for tensors of that size), the latency of a launch, one trip to memory and two barriers.
template <int V> constexpr int HELD = U1<V>;
template <int DT, int V, int UN, bool SILU, bool KEEP>
__global__ __launch_bounds__(MAX_T) void gn_fwd_group_kernel(const GnArgs a) {
    constexpr int K = V / UN;
    __shared__ double sh[2 * K * MAX_T / 64];
    __shared__ float st[2 * K];
    typedef typename Elem<DT>::T T;
    const int bundles = a.P / a.PT, n = blockIdx.x / bundles, c0 = (blockIdx.x % bundles) * a.PT * V;
    const int r = threadIdx.x / a.PT, c = c0 + (threadIdx.x % a.PT) * V;
    const bool on = r < a.R;
    In<DT, V, false> in[HELD<V>];
    Moments<V, UN> m;
#pragma unroll
    for (int k = 0; k < HELD<V>; ++k) { in[k].r = {}; if (on && r + k * a.R < a.S) in[k].load(a, n * a.S + r + k * a.R, c); }
#pragma unroll
    for (int k = 0; k < HELD<V>; ++k) { float f[V]; in[k].get(f); m.add(f); }
    // wave, then workgroup.  (K > 1: the bundle is one piece, its units are whole groups or quarters of one: merged by the thread that takes the group)
    const int G = a.PT * V / a.cg > 0 ? a.PT * V / a.cg : 1, per = K / G > 0 ? K / G : 1, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int u = 0; u < K; ++u) {
        const double x = wave_sum(m.s[u]), y = wave_sum(m.t[u]);
        if ((threadIdx.x & 63) == 0) { sh[2 * (wave * K + u)] = x; sh[2 * (wave * K + u) + 1] = y; }
    }
    __syncthreads();
    if ((int)threadIdx.x < G) {
        double x = 0.0, y = 0.0;
        for (int i = 0; i < waves; ++i)
            for (int u = threadIdx.x * per; u < (int)(threadIdx.x + 1) * per; ++u) { x += sh[2 * (i * K + u)]; y += sh[2 * (i * K + u) + 1]; }
        float mean, rstd;
        statistics_of(x, y, a.inv_m, a.eps, mean, rstd);
        st[threadIdx.x] = mean; st[K + threadIdx.x] = rstd;
        const size_t g = (size_t)n * a.G + c0 / a.cg + threadIdx.x;
        a.mean_out[g] = mean; a.rstd_out[g] = rstd;
    }
    __syncthreads();
    Consts<V, UN> k0{};
    if (on) k0 = constants<V, UN>(a, st - c0 / a.cg, st + K - c0 / a.cg, c);
#pragma unroll
    for (int k = 0; k < HELD<V>; ++k) {
        const int v = r + k * a.R;
        const bool ok = on && v < a.S;
        float f[V], o[V];
        in[k].get(f);
        const size_t row = (size_t)(n * a.S + v);
        if constexpr (KEEP) {                // (bundles of whole blocks)
            Codes<V> q = encode_block<V>(f);
            if constexpr (!SILU) if (ok && a.slope != 1.f) keep_side<V, UN>(a, c, f, k0, border_of<V, UN>(k0), q);
            if (ok) store_codes<V>(q, a.q_out, a.qs_out, row * a.C + c);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = activate<SILU>(__builtin_fmaf(f[e] - k0.mu[e / UN], k0.a[e], k0.b[e]), a.slope);
        if (ok && a.out) store_f32<DT, V>((T*)a.out + row * a.out_ldc + c, o);      // (no output: the statistics alone)
    }
}

// ------------------------------------------------------------------------------------------------ backward
// dz = dy act'(z) of a piece; t = x - mean.  On which side of 0 a ReLU's z falls is decided as in exact arithmetic: z's rounding error is below 2^-21 of
// |t a|, which is |beta| up to a factor 2 where z is that small, and a piece with such a z is decided again in fp64 (one in some ten thousand).  That branch
// is a loop over the elements with its constants from memory: unrolled, hipcc computes their addresses and conversions in front of the voxel loop and keeps 64 to
// 100 registers with them (reduce pass: 204 registers instead of 92, two waves per SIMD instead of five).
template <int V, int UN, bool SILU>
__device__ __forceinline__ void grad_piece(const GnArgs& a, int n, int c, const float (&x)[V], const float (&g)[V], const Consts<V, UN>& k, float border, float (&dz)[V], float (&t)[V]) {
    float least = 3.4e38f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        t[e] = x[e] - k.mu[e / UN];
        const float z = __builtin_fmaf(t[e], k.a[e], k.b[e]);
        if constexpr (SILU) {
            const float sg = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
            dz[e] = g[e] * (sg * (1.f + z * (1.f - sg)));
        } else {
            least = fminf(least, fabsf(z));
            dz[e] = z > 0.f ? g[e] : (a.slope == 0.f ? 0.f : a.slope * g[e]);
        }
    }
    if constexpr (!SILU) {
        if (least < border) {
#pragma unroll 1
            for (int e = 0; e < V; ++e) {
                const size_t i = (size_t)n * a.G + (c + e) / a.cg;
                const double ga = a.gamma ? (double)a.gamma[c + e] : 1.0, be = a.beta ? (double)a.beta[c + e] : 0.0;
                float xe = x[0], ge = g[0];
#pragma unroll
                for (int j = 1; j < V; ++j) { xe = e == j ? x[j] : xe; ge = e == j ? g[j] : ge; }
                const bool pos = positive_exact(xe, a.mean[i], a.rstd[i], ga, be);
                const float d = pos ? ge : (a.slope == 0.f ? 0.f : a.slope * ge);
#pragma unroll
                for (int j = 0; j < V; ++j) dz[j] = e == j ? d : dz[j];
            }
        }
    }
}
// Per-thread sums of dz and dz t (h = t rstd: the factor comes last) in fp32 over at most SUM_TERMS elements, everything behind them in fp64.  The first step is
// requested in front of the constants (rows of single 16-bit channels, 2.3 M elements: 19.1 -> 16.6 us for the whole backward, others -0.4 ... +0.6).
template <int DT, int V, int UN, bool CK, bool SILU>
__global__ __launch_bounds__(MAX_T) void gn_bwd_reduce_kernel(const GnArgs a) {
    extern __shared__ float shf[];
    const Where w = where<V>(a, blockIdx.x);
    constexpr int U = U2<V>;
    typedef typename Elem<DT>::T T;
    float s[V], t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = t[e] = 0.f;
    if (w.on) {
        In<DT, V, CK> in[U]; Raw<DT, V> dy[U];
        auto load = [&](long long v) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                in[u].r = {}; dy[u] = {};
                const long long row = w.n * a.S + v + u * a.R;
                if (v + u * a.R < w.v1) { in[u].load(a, row, w.c); dy[u] = load_raw<DT, V>((const T*)a.dy + (size_t)row * a.dy_ldc + w.c); }
            }
        };
        long long v = w.v0 + w.r;
        load(v);                             // (ahead of the constants)
        const Consts<V, UN> k = constants<V, UN>(a, a.mean + (size_t)w.n * a.G, a.rstd + (size_t)w.n * a.G, w.c);
        const float border = border_of<V, UN>(k);
        for (;;) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[V], g[V], dz[V], d[V];
                in[u].get(f); unpack_raw<DT, V>(dy[u], g);       // (a piece that is not there has dy = 0)
                grad_piece<V, UN, SILU>(a, w.n, w.c, f, g, k, border, dz, d);
#pragma unroll
                for (int e = 0; e < V; ++e) { s[e] += dz[e]; t[e] = __builtin_fmaf(dz[e], d[e], t[e]); }
            }
            v += U * a.R;
            if (v >= w.v1) break;
            load(v);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] *= k.rs[e / UN];
    }
    const int units = a.PT * V;
    float* t2 = shf + a.R * units;
    if (w.r < a.R)
#pragma unroll
        for (int e = 0; e < V; ++e) { const int i = w.r * units + (int)(threadIdx.x % a.PT) * V + e; shf[i] = s[e]; t2[i] = t[e]; }
    __syncthreads();
    const int first = w.tile * units;
    double* o = a.part + (size_t)(blockIdx.x / a.tiles) * a.C * 2;
    double* gs = reinterpret_cast<double*>(shf + ((2 * a.R * units + 1) & ~1));
    sum_rows(shf, t2, a.R, units, [&](int u, double x, double y) {
        if (first + u < a.C) {
            o[(first + u) * 2] = x; o[(first + u) * 2 + 1] = y;
            if (a.gpart) { const double g = a.gamma ? (double)a.gamma[first + u] : 1.0; gs[2 * u] = g * x; gs[2 * u + 1] = g * y; }
        }
    });
    if (a.gpart) {                           // (one tile: all channels of the sample's chunk are here)
        __syncthreads();
        double* p = a.gpart + (size_t)blockIdx.x * a.G * 2;
        sum_groups(gs, gs + 1, 2, a.cg, a.G, [&](int g, double x, double y) { p[2 * g] = x; p[2 * g + 1] = y; });
    }
}

// dgamma, dbeta of 16 channels from the channel records of all samples and chunks: thread = (channel, one of blockDim / 16 record rows)
__device__ __forceinline__ void sum_channels(const double* part, int records, int C, int c0, float* dgamma, float* dbeta, double* sh) {
    const int c = c0 + (threadIdx.x & 15), rows = blockDim.x / 16;
    double s = 0.0, t = 0.0;
    if (c < C)
        for (int k = threadIdx.x >> 4; k < records; k += 4 * rows) {
            double2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) { v[u] = make_double2(0.0, 0.0); if (k + u * rows < records) v[u] = *reinterpret_cast<const double2*>(part + ((size_t)(k + u * rows) * C + c) * 2); }
#pragma unroll
            for (int u = 0; u < 4; ++u) { s += v[u].x; t += v[u].y; }
        }
    sh[threadIdx.x] = s; sh[blockDim.x + threadIdx.x] = t;
    __syncthreads();
    sum_rows(sh, sh + blockDim.x, rows, 16, [&](int u, double x, double y) {
        if (c0 + u < C) { if (dbeta) dbeta[c0 + u] = (float)x; if (dgamma) dgamma[c0 + u] = (float)y; }
    });
}

// workgroups [0, N G): m1, m2 of a group, from its records or its channels' ones; the ones behind them: dgamma, dbeta of 16 channels each
__global__ __launch_bounds__(256) void gn_bwd_finalize_kernel(const double* __restrict__ part, const double* __restrict__ gpart, int N, int chunks, int C, int G, const float* __restrict__ gamma, double inv_m,
                                                              float* __restrict__ m1, float* __restrict__ m2, float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ double sh[512];
    const int i = blockIdx.x, cg = C / G;
    if (i < N * G) {
        double s = 0.0, t = 0.0;
        const int n = i / G, c0 = (i % G) * cg;
        if (gpart)
            for (int k = threadIdx.x; k < chunks; k += 256) {
                const double* r = gpart + ((size_t)((size_t)n * chunks + k) * G + i % G) * 2;
                s += r[0]; t += r[1];
            }
        else for (long long k = threadIdx.x; k < (long long)chunks * cg; k += 256) {
            const int c = c0 + (int)(k % cg);
            const double* r = part + ((size_t)((size_t)n * chunks + k / cg) * C + c) * 2;
            const double g = gamma ? (double)gamma[c] : 1.0;
            s += g * r[0]; t += g * r[1];
        }
        block_sum2(s, t);
        if (threadIdx.x == 0) { m1[i] = (float)(s * inv_m); m2[i] = (float)(t * inv_m); }
    } else sum_channels(part, N * chunks, C, (i - N * G) * 16, dgamma, dbeta, sh);
}

// dx = a dz - rstd m1 - t rstd^2 m2, from the chunk's end to its start; dgamma and dbeta in workgroups of their own in front of the others.  2 x 64 x 128 x 128 x 32: 97 us from a
// checkpoint in fp32 (608 MB), 66 in bf16 (403 MB)
template <int DT, int V, int UN, bool CK, bool SILU>
__global__ __launch_bounds__(MAX_T) void gn_bwd_apply_kernel(const GnArgs a) {
    extern __shared__ double sh[];
    if ((int)blockIdx.x < a.sum_wgs) { sum_channels(a.cpart, a.N * a.rec_chunks, a.C, blockIdx.x * 16, a.dgamma, a.dbeta, sh); return; }
    const Where w = where<V>(a, blockIdx.x - a.sum_wgs);
    constexpr int U = U2<V>;
    typedef typename Elem<DT>::T T;
    constexpr bool NT = V > 1;               // (as in the forward: 255 -> 230 us, bf16 131 -> 115)
    In<DT, V, CK, NT> in[U]; Raw<DT, V> dy[U]; bool ok[U];
    auto load = [&](long long vb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long v = vb + w.r + u * a.R, row = w.n * a.S + v;
            ok[u] = w.on && v < w.v1;
            in[u].r = {}; dy[u] = {};
            if (ok[u]) { in[u].load(a, row, w.c); dy[u] = load_raw<DT, V, NT>((const T*)a.dy + (size_t)row * a.dy_ldc + w.c); }
        }
    };
    const int step = U * a.R;                // (from the end, as in the forward)
    long long vb = w.v0 + (w.v1 - w.v0 - 1) / step * step;
    load(vb);
    if (a.rec) merge_records(a.rec + (size_t)w.n * a.rec_chunks * a.G * 2, a.rec_chunks, a.G, sh);
    if (!w.on) return;
    const Consts<V, UN> k = constants<V, UN>(a, a.mean + (size_t)w.n * a.G, a.rstd + (size_t)w.n * a.G, w.c);
    const float border = border_of<V, UN>(k);
    float c1[V / UN], c2[V / UN];
#pragma unroll
    for (int u = 0; u < V / UN; ++u) {
        const int g = (w.c + u * UN) / a.cg;
        const float m1 = a.rec ? (float)(sh[2 * g] * a.inv_m) : a.m1[(size_t)w.n * a.G + g], m2 = a.rec ? (float)(sh[2 * g + 1] * a.inv_m) : a.m2[(size_t)w.n * a.G + g];
        c1[u] = k.rs[u] * m1; c2[u] = k.rs[u] * k.rs[u] * m2;
    }
    for (;;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V], g[V], dz[V], d[V], o[V];
            in[u].get(f); unpack_raw<DT, V>(dy[u], g);
            grad_piece<V, UN, SILU>(a, w.n, w.c, f, g, k, border, dz, d);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = __builtin_fmaf(k.a[e], dz[e], -__builtin_fmaf(d[e], c2[e / UN], c1[e / UN]));
            if (ok[u]) store_f32<DT, V, NT>((T*)a.out + (size_t)(w.n * a.S + vb + w.r + u * a.R) * a.out_ldc + w.c, o);
        }
        vb -= step;
        if (vb < w.v0) break;
        load(vb);
    }
}

// Small groups: a workgroup takes a bundle of whole groups (as in gn_fwd_group_kernel), keeps its pieces of x and dy in registers from the sums to dx, and walks the
// samples, which gives it its channels' dgamma and dbeta: no records, no second launch.
template <int DT, int V, int UN, bool CK, bool SILU>
__global__ __launch_bounds__(MAX_T) void gn_bwd_group_kernel(const GnArgs a) {
    extern __shared__ double sh[];
    __shared__ float st[2 * V];
    typedef typename Elem<DT>::T T;
    constexpr int H = HELD<V>;
    const int units = a.PT * V, c0 = blockIdx.x * units, groups = units > a.cg ? units / a.cg : 1;
    const int r = threadIdx.x / a.PT, p = threadIdx.x % a.PT, c = c0 + p * V;
    const bool on = r < a.R;
    double *gs = sh, *all = sh + 2 * units;
    float *fs = reinterpret_cast<float*>(all + 2 * units), *ft = fs + a.R * units;
    for (int u = threadIdx.x; u < 2 * units; u += blockDim.x) all[u] = 0.0;
    for (int n = 0; n < a.N; ++n) {
        In<DT, V, CK> in[H]; Raw<DT, V> dy[H];
#pragma unroll
        for (int k = 0; k < H; ++k) {
            const long long row = n * a.S + r + k * a.R;
            in[k].r = {}; dy[k] = {};
            if (on && r + k * a.R < a.S) { in[k].load(a, row, c); dy[k] = load_raw<DT, V>((const T*)a.dy + (size_t)row * a.dy_ldc + c); }
        }
        Consts<V, UN> k0{};
        if (on) k0 = constants<V, UN>(a, a.mean + (size_t)n * a.G, a.rstd + (size_t)n * a.G, c);
        const float border = border_of<V, UN>(k0);
        float s[V], t[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = t[e] = 0.f;
#pragma unroll
        for (int k = 0; k < H; ++k) {
            float f[V], g[V], dz[V], d[V];
            in[k].get(f); unpack_raw<DT, V>(dy[k], g);           // (a piece that is not there has dy = 0)
            grad_piece<V, UN, SILU>(a, n, c, f, g, k0, border, dz, d);
#pragma unroll
            for (int e = 0; e < V; ++e) { s[e] += dz[e]; t[e] = __builtin_fmaf(dz[e], d[e], t[e]); }
        }
        if (on)
#pragma unroll
            for (int e = 0; e < V; ++e) { const int i = r * units + p * V + e; fs[i] = s[e]; ft[i] = t[e] * k0.rs[e / UN]; }
        __syncthreads();
        sum_rows(fs, ft, a.R, units, [&](int u, double x, double y) {
            const double g = a.gamma ? (double)a.gamma[c0 + u] : 1.0;
            all[2 * u] += x; all[2 * u + 1] += y;                // (a unit is the same thread's for every sample)
            gs[2 * u] = g * x; gs[2 * u + 1] = g * y;
        });
        __syncthreads();
        if (groups > 1) {
            if ((int)threadIdx.x < groups) {
                double x = 0.0, y = 0.0;
                for (int e = threadIdx.x * a.cg; e < (int)(threadIdx.x + 1) * a.cg; ++e) { x += gs[2 * e]; y += gs[2 * e + 1]; }
                st[threadIdx.x] = (float)(x * a.inv_m); st[V + threadIdx.x] = (float)(y * a.inv_m);
            }
        } else if (threadIdx.x < 64) {
            double x = 0.0, y = 0.0;
            for (int e = threadIdx.x; e < units; e += 64) { x += gs[2 * e]; y += gs[2 * e + 1]; }
            x = wave_sum(x); y = wave_sum(y);
            if (threadIdx.x == 0) { st[0] = (float)(x * a.inv_m); st[V] = (float)(y * a.inv_m); }
        }
        __syncthreads();
        float c1[V / UN], c2[V / UN];
#pragma unroll
        for (int u = 0; u < V / UN; ++u) {
            const int g = groups > 1 ? u * UN / a.cg : 0;
            c1[u] = k0.rs[u] * st[g]; c2[u] = k0.rs[u] * k0.rs[u] * st[V + g];
        }
#pragma unroll
        for (int k = 0; k < H; ++k) {
            float f[V], g[V], dz[V], d[V], o[V];
            in[k].get(f); unpack_raw<DT, V>(dy[k], g);
            grad_piece<V, UN, SILU>(a, n, c, f, g, k0, border, dz, d);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = __builtin_fmaf(k0.a[e], dz[e], -__builtin_fmaf(d[e], c2[e / UN], c1[e / UN]));
            if (on && r + k * a.R < a.S) store_f32<DT, V>((T*)a.out + (size_t)(n * a.S + r + k * a.R) * a.out_ldc + c, o);
        }
    }
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
        if (a.dbeta) a.dbeta[c0 + u] = (float)all[2 * u];
        if (a.dgamma) a.dgamma[c0 + u] = (float)all[2 * u + 1];
    }
}

// ------------------------------------------------------------------------------------------------ host side
struct Shape { int N; long long S; int C, G; };

constexpr int PASS_WGS = 512;                // workgroups of a pass: two per CU (256 threads each); 1024 cost the merges of mid-sized tensors 2 - 8 us and gain nothing
constexpr int PASS_T = 256;
constexpr int SUM_TERMS = 512;               // fp32 terms of a sum: their rounding stays below 512 2^-24 of the sum of magnitudes, with more chunks for samples of more voxels

void set_shape(GnArgs& a, const Shape& sh) { a.N = sh.N; a.S = sh.S; a.C = sh.C; a.G = sh.G; a.cg = sh.C / sh.G; a.inv_m = 1.0 / ((double)sh.S * a.cg); }

// Twice as many where a backward's workgroups have 16 steps or more and a sample's records stay few (us of a call in a replayed graph, two -> four workgroups per CU.  2 x 64 x 128 x 128 x 32 in 8 groups: fp32
// 234 -> 219, from a checkpoint 169 -> 164, bf16 from a checkpoint 111 -> 106, but bf16 129 -> 131; 4 x 64 x 64 x 64 x 64 in 8: fp32 233 -> 218, bf16 from a checkpoint 123 -> 112; one sample
// 64 x 128 x 128 x 32 in 32, bf16 from a checkpoint, would lose 65 -> 71), or for rows of single elements, whose loads are small (bf16 forward of 1 x 19 x 27 x 89 x 65 in 1 group 28 -> 22,
// 1 x 41 x 64 x 65 x 33 in 3 41 -> 30, 2 x 30 x 100 x 101 x 7 in 7 31 -> 25; their backwards with two, three, four per CU: 23.3, 20.0, 20.2; 30.1, 25.5, 24.8; 24.8, 22.2, 22.5, and 20.2,
// 18.3, 19.3 for 3 x 17 x 45 x 51 x 25 in 5)
template <int V> int workgroups(const Shape& sh, bool backward, bool ck = true) {
    const long long steps = sh.N * sh.S * (sh.C / V) / (PASS_T * U2<V>);
    if (V == 1) return !backward ? 2 * PASS_WGS : steps >= 2 * PASS_WGS ? PASS_WGS * 3 / 2 : PASS_WGS;
    return backward && (ck || V < 8) && steps >= 16 * PASS_WGS && 2ll * PASS_WGS * sh.G <= 4096ll * sh.N ? 2 * PASS_WGS : PASS_WGS;
}

// mapping of a pass; `target`: workgroups that it asks for (at least one per sample and tile); `terms`: voxels of a thread at most, or 0
template <int V> void map_pass(GnArgs& a, const Shape& sh, int target, int U, bool keep, int terms = 0) {
    set_shape(a, sh);
    a.P = sh.C / V;
    a.tiles = (a.P + MAX_T - 1) / MAX_T;
    a.PT = (a.P + a.tiles - 1) / a.tiles;
    a.R = PASS_T / a.PT > 0 ? PASS_T / a.PT : 1;
    if (keep) {                              // whole blocks of 64 elements per workgroup step
        int k = CK_BLOCK / V;
        for (int p = a.PT; k > 1 && p % 2 == 0; p /= 2) k /= 2;
        a.R = (a.R + k - 1) / k * k;
    }
    long long most = target / ((long long)sh.N * a.tiles);
    if (most < 1) most = 1;
    if (terms && most < (sh.S + (long long)terms * a.R - 1) / ((long long)terms * a.R)) most = (sh.S + (long long)terms * a.R - 1) / ((long long)terms * a.R);
    const long long step = (long long)a.R * U;
    long long chunks = (sh.S + step - 1) / step;
    if (chunks > most) chunks = most;
    a.chunk = (sh.S + chunks - 1) / chunks;
    a.chunk = (a.chunk + a.R - 1) / a.R * a.R;
    a.chunks = (int)((sh.S + a.chunk - 1) / a.chunk);
}
dim3 grid_of(const GnArgs& a) { return dim3((unsigned)((long long)a.N * a.chunks * a.tiles)); }
dim3 block_of(const GnArgs& a) { return dim3((unsigned)((a.R * a.PT + 63) / 64 * 64)); }

// UN of the kernels
int unit_of(int V, int cg) { return V >= 8 && cg % 8 == 0 ? 8 : V >= 4 && cg % 4 == 0 ? 4 : 1; }

// units of a statistics record
int units_of(const GnArgs& a, int un) { return a.tiles > 1 ? a.C / un : a.G; }
template <int V> size_t fwd_part_doubles(const Shape& sh) {
    GnArgs a{}; map_pass<V>(a, sh, workgroups<V>(sh, false), U1<V>, false);
    return (size_t)sh.N * a.chunks * units_of(a, unit_of(V, a.cg)) * 2;
}
// what lies in the workspace of a backward pass: channel records, group records where a workgroup holds whole groups, and, where no apply pass merges those, m1 and m2
struct BwdSpace { size_t channels, groups, behind; bool merge; };
BwdSpace bwd_space(const GnArgs& a, const Shape& sh) {
    BwdSpace b;
    const bool whole = a.tiles == 1 && sh.C <= 2048;         // (16 bytes of LDS per channel beside the sums' 32 KB)
    b.merge = whole && sh.G <= MERGE_UNITS && (long long)a.chunks * sh.G <= MERGE_MAX;
    b.groups = whole ? align_up((size_t)sh.N * a.chunks * sh.G * 2 * sizeof(double), 256) : 0;
    b.channels = align_up((size_t)sh.N * a.chunks * sh.C * 2 * sizeof(double), 256);
    b.behind = b.merge ? 0 : (size_t)2 * sh.N * sh.G * sizeof(float);
    return b;
}
size_t max2(size_t a, size_t b) { return a > b ? a : b; }
// One workgroup per group where the pieces of a bundle fit its threads' registers: fills in PT and R
template <int V> bool map_group(GnArgs& a, const Shape& sh) {
    set_shape(a, sh);
    if (a.cg % V != 0 && V % a.cg != 0) return false;
    a.P = sh.C / V;
    a.PT = a.cg > V ? a.cg / V : 1;
    if (a.PT > MAX_T || sh.S > (long long)HELD<V> * (MAX_T / a.PT)) return false;
    a.R = MAX_T / a.PT;
    for (int t = MAX_T / 2; t >= 64; t /= 2)             // no more threads than pieces
        if (t / a.PT > 0 && sh.S <= t / a.PT) a.R = t / a.PT;
    return true;
}
// ... of the forward, for elements of `size` bytes.  A bundle narrower than a 128-byte line moves every line once per bundle in it, to as many workgroups on other XCDs: what that moves is
// limited.  us of a call in a replayed graph, two launches : one, 16-bit types unless said, by megabytes moved so (two launches and their workspace cost an eager call 4 us of the host's time
// besides, which shows where the GPU takes less than some 15 us: 15.5 : 14.6 for 24 x 2048 x 64, 15.5 : 11.6 for 2 x 4096 x 64, but 17.0 : 17.7 for 4 x 2048 x 512):
//   pieces: 32: 14.3 : 12.8 (2 x 2048 voxels x 512 in 64 groups), 11.7 : 11.7 (16 x 2048 x 64 in 8), fp32 12.5 : 13.6 (4 x 4096 x 64 in 16); 40: 15.0 : 13.9 (5 x 2048 x 256 in 32);
//     48: 13.4 : 16.6 (24 x 2048 x 64 in 8); 64: 17.5 : 19.6 (4 x 2048 x 512 in 64); 1024: 76 : 236 (64 of these)
//   single elements instead of two launches with pieces: 16: 10.7 : 9.1 (2 x 4096 x 32 in 32); 21: 14.6 : 11.9 (16 x 105 x 1200 in 100); 31: 15.0 : 16.6 (300 x 105 x 96 in 8);
//     41: 15.8 : 21.4 (32 x 105 x 1200 in 100); one-channel groups 32: 11.2 : 10.7 (1 x 4096 x 64 in 64); 64: 11.4 : 12.1 (2 x 4096 x 64 in 64); 256: 16.1 : 24.3 (4 x 4096 x 128 in 128);
//     1024: 34 : 88 (8 x 4096 x 256 in 256)
//   single elements in either form: 5 bundles to a line 385: 130 : 113 (400 x 315 x 300 in 25); 21 and 33 of them 41: 15.0 : 10.9 (16 x 315 x 201 in 67), 12.6 : 12.2 (64 x 315 x 33 in 33),
//     165: 26 : 31, 18 : 33 (four times these)
// Bundles of whole lines have no limit (1024 x 256 x 512 in 8: 150 : 142).
template <int V> bool map_group_fwd(GnArgs& a, const Shape& sh, int size, bool rows_of_pieces) {
    if (!map_group<V>(a, sh)) return false;
    const long long row = (long long)sh.C * size, width = (long long)a.PT * V * size, line = row < 128 ? row : 128;
    if (width >= line || (!rows_of_pieces && line <= 8 * width)) return true;
    const int piece = 16 / size;
    const bool cut = a.cg % piece != 0 && piece % a.cg != 0;
    return sh.N * sh.S * (row / width) * line <= (V > 1 ? 48ll : !rows_of_pieces ? 96ll : cut ? 32ll : 64ll) << 20;
}
// ... and of the backward, whose workgroups walk the samples: 6 us for the first and 3 - 9 for each other one (a workgroup's 16-byte pieces lie C elements apart) against
// 9 - 13 for two launches, which cost the host 5 us more.  1 x 4 x 8 x 8 x 128 in 8 groups, fp16: 8.4 us instead of 12.2, eagerly 13 instead of 18; two samples of it 14.2
// instead of 12.3, eagerly 14 instead of 18; four 25.8; 16384 elements to a group 15.4 instead of 14.0
constexpr int GROUP_SAMPLES = 2, GROUP_ELEMS = 8192, GROUP_CHANNELS = 512;         // samples, elements of a group in all of them, channels of a bundle (48 KB of LDS)
template <int V> bool map_group_bwd(GnArgs& a, const Shape& sh) {
    return sh.N <= GROUP_SAMPLES && map_group<V>(a, sh) && a.PT * V <= GROUP_CHANNELS && sh.N * sh.S * a.cg <= GROUP_ELEMS;
}
// single elements instead of two launches with pieces: where groups cut the pieces, or (one-channel groups of more voxels than pieces can hold) for one sample: 1 x 4096 voxels x 8, 16, 32,
// 64, 256 channels in 16 bits 7.2, 10.4, 11.5, 14.4, 21.7 us against 10.5, 10.9, 11.0, 13.6, 23.3 for two launches, but two samples x 16, 64 channels 18.0, 26.3 against 11.0, 13.9
template <int V> bool map_single_bwd(GnArgs& a, const Shape& sh) {
    const int cg = sh.C / sh.G;
    return (sh.N == 1 || (cg % V != 0 && V % cg != 0)) && map_group_bwd<1>(a, sh);
}
template <int V> size_t space_of(const Shape& sh, bool backward) {
    if (sh.C % V != 0) return 0;
    GnArgs a{};
    if (backward && (map_group_bwd<V>(a, sh) || (V > 1 && map_single_bwd<V>(a, sh)))) return 0;
    if (!backward) {
        const int size = V == 8 ? 2 : 4;
        const bool one = V > 1 ? map_group_fwd<V>(a, sh, size, true) || map_group_fwd<1>(a, sh, size, true)
                               : map_group_fwd<1>(a, sh, 2, false) && map_group_fwd<1>(a, sh, 4, false);       // (single elements: of every type)
        return one ? 0 : fwd_part_doubles<V>(sh) * sizeof(double);
    }
    map_pass<V>(a, sh, workgroups<V>(sh, true), U2<V>, false, SUM_TERMS);        // (the most that a backward takes)
    const BwdSpace b = bwd_space(a, sh);
    return b.channels + b.groups + b.behind;
}
size_t workspace_bytes(const Shape& sh, bool backward) {      // (for every type and alignment)
    return max2(space_of<1>(sh, backward), max2(space_of<4>(sh, backward), space_of<8>(sh, backward)));
}
size_t merge_lds(const GnArgs& a, int units) { return (size_t)2 * (block_of(a).x + units) * sizeof(double); }

#define GN_LAUNCH(KERNEL, GRID, BLOCK, LDS, S, A)                                                                                       \
    do {                                                                                                                                \
        if ((A).slope == ACT_SILU) { constexpr bool SILU = true; hipLaunchKernelGGL((KERNEL), GRID, BLOCK, LDS, S, A); }                \
        else { constexpr bool SILU = false; hipLaunchKernelGGL((KERNEL), GRID, BLOCK, LDS, S, A); }                                     \
    } while (0)

// BEHIND: behind a statistics pass of the same call
template <int DT, int V, int UN, bool CK, bool BEHIND> void launch_apply(GnArgs a, const Shape& sh, hipStream_t s) {
    const bool keep = a.q_out != nullptr;
    // (merging the records costs a workgroup 1 - 2 us: twice the workgroups without it, 74 -> 53 us for 2 x 64 x 128 x 128 x 32 in bf16)
    map_pass<V>(a, sh, a.rec ? workgroups<V>(sh, false) : 2 * PASS_WGS, U1<V>, keep);
    const size_t lds = a.rec ? merge_lds(a, sh.G) : 0;
    constexpr bool NT = V > 1 && (BEHIND || CK);
    if constexpr (V > 1 && BEHIND) {
        if (keep) { GN_LAUNCH((gn_apply_kernel<DT, V, UN, CK, SILU, true, NT>), grid_of(a), block_of(a), lds, s, a); return; }
    }
    GN_LAUNCH((gn_apply_kernel<DT, V, UN, CK, SILU, false, NT>), grid_of(a), block_of(a), lds, s, a);
}

// the checkpoint as a pass of its own, behind the one that has written mean and rstd
int pack_behind(int dt, const GnArgs& a, const Shape& sh, hipStream_t s) {
    Border b;
    if (a.slope != 1.f && a.slope != ACT_SILU) { b.rule = 1; b.mean = a.mean_out; b.rstd = a.rstd_out; b.gamma = a.gamma; b.beta = a.beta; b.S = sh.S; b.G = sh.G; }
    return launch_checkpoint8_pack(dt, a.x, a.x_ldc, (long long)sh.N * sh.S, sh.C, a.q_out, a.qs_out, b, s);
}

template <int DT, int V, int UN> int forward_group(GnArgs a, const Shape& sh, hipStream_t s) {
    const dim3 grid((unsigned)((long long)sh.N * (a.P / a.PT)));
    if constexpr (V > 1 && UN == V) {
        if (a.q_out && a.PT * V % CK_BLOCK == 0 && (uintptr_t)a.q_out % V == 0) {      // bundles of whole blocks
            GN_LAUNCH((gn_fwd_group_kernel<DT, V, UN, SILU, true>), grid, block_of(a), 0, s, a);
            return E3_OK;
        }
    }
    if (a.q_out && a.out == a.x) {           // in place: the checkpoint, which needs the statistics, in front of the output
        GnArgs st = a;
        st.out = nullptr;
        GN_LAUNCH((gn_fwd_group_kernel<DT, V, UN, SILU, false>), grid, block_of(a), 0, s, st);
        const int rc = pack_behind(DT, a, sh, s);
        if (rc) return rc;
        a.q_out = nullptr;
    }
    GN_LAUNCH((gn_fwd_group_kernel<DT, V, UN, SILU, false>), grid, block_of(a), 0, s, a);
    return a.q_out ? pack_behind(DT, a, sh, s) : E3_OK;
}

template <int DT, int V, int UN> int forward(GnArgs a, const Shape& sh, void* ws, hipStream_t s) {
    constexpr int size = sizeof(typename Elem<DT>::T);
    if (map_group_fwd<V>(a, sh, size, V > 1)) {
        const int rc = forward_group<DT, V, UN>(a, sh, s);
        E3_CHECK_HIP(hipGetLastError());
        return rc;
    }
    if constexpr (V > 1) {                   // (groups that cut the pieces, or one-channel groups of more voxels than pieces can hold: element by element)
        if (map_group_fwd<1>(a, sh, size, true)) return forward<DT, 1, 1>(a, sh, ws, s);
    }
    E3_REQUIRE(ws, E3_ERR_WORKSPACE, "workspace too small");         // (where workspace_bytes() and this dispatch disagree)
    GnArgs st = a;
    map_pass<V>(st, sh, workgroups<V>(sh, false), U1<V>, false);
    st.part = (double*)ws;
    const int units = units_of(st, UN);
    hipLaunchKernelGGL((gn_stats_kernel<DT, V, UN>), grid_of(st), block_of(st), (size_t)st.R * st.PT * (V / UN) * 2 * sizeof(double), s, st);
    a.mean = a.mean_out; a.rstd = a.rstd_out;
    // the checkpoint rides in the apply pass where its blocks are whole there; otherwise it is a pass of its own: behind the apply pass, or, in place, in front of it
    GnArgs m{}; map_pass<V>(m, sh, workgroups<V>(sh, false), U1<V>, true);
    const bool fused = a.q_out && V > 1 && m.tiles == 1 && m.R * m.PT <= MAX_T && ((unsigned long long)sh.S * sh.C) % CK_BLOCK == 0 && (uintptr_t)a.q_out % V == 0;
    const bool before = a.q_out && !fused && a.out == a.x;
    if (!before && st.tiles == 1 && (long long)st.chunks * sh.G <= MERGE_MAX && sh.G <= MERGE_UNITS) { a.rec = st.part; a.rec_chunks = st.chunks; }
    else hipLaunchKernelGGL(gn_finalize_kernel, dim3(sh.N * sh.G), dim3(256), 0, s, st.part, st.chunks, units, units / sh.G, st.inv_m, a.eps, a.mean_out, a.rstd_out);
    if (before) { const int rc = pack_behind(DT, a, sh, s); if (rc) return rc; }
    GnArgs ap = a;
    if (!fused) ap.q_out = nullptr;
    launch_apply<DT, V, UN, false, true>(ap, sh, s);
    E3_CHECK_HIP(hipGetLastError());
    return a.q_out && !fused && !before ? pack_behind(DT, a, sh, s) : E3_OK;
}

template <int DT, int V, int UN, bool CK> int backward(GnArgs a, const Shape& sh, void* ws, hipStream_t s) {
    if (map_group_bwd<V>(a, sh)) {
        const int units = a.PT * V;
        GN_LAUNCH((gn_bwd_group_kernel<DT, V, UN, CK, SILU>), dim3(a.P / a.PT), block_of(a), (size_t)4 * units * sizeof(double) + (size_t)2 * a.R * units * sizeof(float), s, a);
        E3_CHECK_HIP(hipGetLastError());
        return E3_OK;
    }
    if constexpr (V > 1) {
        if (map_single_bwd<V>(a, sh)) return backward<DT, 1, 1, CK>(a, sh, ws, s);
    }
    E3_REQUIRE(ws, E3_ERR_WORKSPACE, "workspace too small");
    GnArgs st = a;
    map_pass<V>(st, sh, workgroups<V>(sh, true, CK), U2<V>, false, SUM_TERMS);
    st.part = (double*)ws;
    const BwdSpace space = bwd_space(st, sh);
    if (space.groups) st.gpart = (double*)((char*)ws + space.channels);
    const size_t lds = align_up((size_t)st.R * st.PT * V * 2 * sizeof(float), 8) + (space.groups ? (size_t)sh.C * 2 * sizeof(double) : 0);
    GN_LAUNCH((gn_bwd_reduce_kernel<DT, V, UN, CK, SILU>), grid_of(st), block_of(st), lds, s, st);
    map_pass<V>(a, sh, workgroups<V>(sh, true, CK), U2<V>, false);
    size_t alds = 0;
    const int sums = (a.dgamma || a.dbeta) ? (sh.C + 15) / 16 : 0;
    if (space.merge) {
        a.rec = st.gpart; a.rec_chunks = st.chunks;
        a.cpart = st.part; a.sum_wgs = sums;
        alds = merge_lds(a, sh.G);
    } else {
        float* m1 = (float*)((char*)ws + space.channels + space.groups);
        float* m2 = m1 + (size_t)sh.N * sh.G;
        hipLaunchKernelGGL(gn_bwd_finalize_kernel, dim3(sh.N * sh.G + sums), dim3(256), 0, s, st.part, st.gpart, sh.N, st.chunks, sh.C, sh.G, a.gamma, a.inv_m, m1, m2, a.dgamma, a.dbeta);
        a.m1 = m1; a.m2 = m2;
    }
    const dim3 grid(grid_of(a).x + a.sum_wgs);
    GN_LAUNCH((gn_bwd_apply_kernel<DT, V, UN, CK, SILU>), grid, block_of(a), alds, s, a);
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

// f(DT, V, UN) as compile-time constants
template <int I> using Int = std::integral_constant<int, I>;
template <int DT, typename F> int by_pieces(bool wide, int cg, F f) {
    constexpr int V = wide_of(DT);
    if (!wide) return f(Int<DT>(), Int<1>(), Int<1>());
    if (cg % V == 0) return f(Int<DT>(), Int<V>(), Int<V>());
    if constexpr (V == 8) if (cg % 4 == 0) return f(Int<DT>(), Int<V>(), Int<4>());
    return f(Int<DT>(), Int<V>(), Int<1>());
}
template <typename F> int by_type(int dtype, bool wide, int cg, F f) {
    return dtype == DT_F32 ? by_pieces<DT_F32>(wide, cg, f) : dtype == DT_BF16 ? by_pieces<DT_BF16>(wide, cg, f) : by_pieces<DT_F16>(wide, cg, f);
}

bool act_ok(float slope) { return (slope >= 0.f && slope <= 1.f) || slope == ACT_SILU; }

// sizes of a call: 0, or the error that e3_last_error() describes
int check_shape(int dtype, int N, int D, int H, int W, int C, int G, float slope, Shape& sh) {
    E3_REQUIRE(dtype >= 0 && dtype <= 2, E3_ERR_INVALID, "dtype must be E3_DT_F32, E3_DT_BF16 or E3_DT_F16");
    E3_REQUIRE(N >= 1 && D >= 1 && H >= 1 && W >= 1 && C >= 1, E3_ERR_INVALID, "sizes must be at least 1");
    E3_REQUIRE(G >= 1 && C % G == 0, E3_ERR_INVALID, "num_groups must divide the channel count");
    E3_REQUIRE(act_ok(slope), E3_ERR_UNSUPPORTED, "activation slope must be in [0, 1], or 2 for SiLU");
    sh.N = N; sh.S = (long long)D * H * W; sh.C = C; sh.G = G;
    // (a launch has fewer than 2^32 threads: 512 per group or tile, 256 per 16 channels)
    E3_REQUIRE((long long)N * G < (1ll << 23) && (long long)N * ((C + MAX_T - 1ll) / MAX_T) < (1ll << 23) && C <= (1 << 26), E3_ERR_UNSUPPORTED, "more than 2^23 groups or 2^26 channels");
    return E3_OK;
}

}  // namespace

extern "C" {

size_t e3_group_norm_workspace_bytes(int N, int D, int H, int W, int C, int G, int backward) {
    Shape sh;
    if (check_shape(0, N, D, H, W, C, G, 0.f, sh)) return 0;
    return workspace_bytes(sh, backward != 0);
}

int e3_group_norm_act_fwd(void* stream, int dtype, const void* x, int x_ldc, const float* gamma, const float* beta, float eps, float act_slope, void* y, int y_ldc,
                          float* mean, float* rstd, signed char* q, float* q_scale, int N, int D, int H, int W, int C, int G, void* workspace, size_t workspace_bytes_) {
    Shape sh;
    const int rc = check_shape(dtype, N, D, H, W, C, G, act_slope, sh);
    if (rc) return rc;
    E3_REQUIRE(x && y && mean && rstd, E3_ERR_INVALID, "null argument");
    E3_REQUIRE((q == nullptr) == (q_scale == nullptr), E3_ERR_INVALID, "a checkpoint is codes and scales");
    E3_REQUIRE(x_ldc >= C && y_ldc >= C, E3_ERR_INVALID, "rows are shorter than the channel count");
    E3_REQUIRE(eps >= 0.f, E3_ERR_INVALID, "eps must not be negative");
    const size_t need = workspace_bytes(sh, false);
    E3_REQUIRE(workspace_bytes_ >= need && (workspace || !need), E3_ERR_WORKSPACE, "workspace too small");
    E3_REQUIRE(aligned16(workspace), E3_ERR_INVALID, "the workspace must be aligned to 16 bytes");
    GnArgs a{};
    a.x = x; a.x_ldc = x_ldc; a.out = y; a.out_ldc = y_ldc; a.gamma = gamma; a.beta = beta; a.slope = act_slope; a.q_out = q; a.qs_out = q_scale;
    a.eps = eps; a.mean_out = mean; a.rstd_out = rstd;
    const bool wide = wide_rows(dtype, x, x_ldc, C) && wide_rows(dtype, y, y_ldc, C);
    return by_type(dtype, wide, C / G, [&](auto dt, auto v, auto un) { return forward<dt.value, v.value, un.value>(a, sh, workspace, (hipStream_t)stream); });
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
    const bool wide = (x ? wide_rows(dtype, x, x_ldc, C) : wide_codes(dtype, q, C)) && wide_rows(dtype, y, y_ldc, C);
    by_type(dtype, wide, C / G, [&](auto dt, auto v, auto un) {
        if (x) launch_apply<dt.value, v.value, un.value, false, false>(a, sh, (hipStream_t)stream);
        else launch_apply<dt.value, v.value, un.value, true, false>(a, sh, (hipStream_t)stream);
        return E3_OK;
    });
    E3_CHECK_HIP(hipGetLastError());
    return E3_OK;
}

int e3_group_norm_act_bwd(void* stream, int dtype, const void* x, int x_ldc, const signed char* q, const float* q_scale, const float* mean, const float* rstd,
                          const float* gamma, const float* beta, float act_slope, const void* dy, int dy_ldc, void* dx, int dx_ldc, float* dgamma, float* dbeta,
                          int N, int D, int H, int W, int C, int G, void* workspace, size_t workspace_bytes_) {
    Shape sh;
    const int rc = check_shape(dtype, N, D, H, W, C, G, act_slope, sh);
    if (rc) return rc;
    E3_REQUIRE(dy && dx && mean && rstd && (x || (q && q_scale)), E3_ERR_INVALID, "null argument");
    E3_REQUIRE((!x || x_ldc >= C) && dy_ldc >= C && dx_ldc >= C, E3_ERR_INVALID, "rows are shorter than the channel count");
    const size_t need = workspace_bytes(sh, true);
    E3_REQUIRE(workspace || !need, E3_ERR_INVALID, "null argument");
    E3_REQUIRE(workspace_bytes_ >= need, E3_ERR_WORKSPACE, "workspace too small");
    E3_REQUIRE(aligned16(workspace), E3_ERR_INVALID, "the workspace must be aligned to 16 bytes");
    GnArgs a{};
    a.x = x; a.x_ldc = x_ldc; a.q = q; a.qs = q_scale; a.dy = dy; a.dy_ldc = dy_ldc; a.out = dx; a.out_ldc = dx_ldc;
    a.mean = mean; a.rstd = rstd; a.gamma = gamma; a.beta = beta; a.slope = act_slope; a.dgamma = dgamma; a.dbeta = dbeta;
    const bool wide = (x ? wide_rows(dtype, x, x_ldc, C) : wide_codes(dtype, q, C)) && wide_rows(dtype, dy, dy_ldc, C) && wide_rows(dtype, dx, dx_ldc, C);
    return by_type(dtype, wide, C / G, [&](auto dt, auto v, auto un) {
        return x ? backward<dt.value, v.value, un.value, false>(a, sh, workspace, (hipStream_t)stream)
                 : backward<dt.value, v.value, un.value, true>(a, sh, workspace, (hipStream_t)stream);
    });
}

}  // extern "C"
