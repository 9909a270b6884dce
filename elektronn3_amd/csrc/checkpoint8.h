// Element access of the normalisation kernels (group_norm.hip) and the 8-bit activation checkpoints (checkpoint8.hip).
//
// An 8-bit checkpoint of a channels-last tensor cuts its packed [N][D][H][W][C] elements into blocks of 64.  A block keeps
//     q = round_to_even(x * (127 / amax))  in int8,   scale = amax * (1 / 127)  in fp32,   and stands for  fp32(q * scale),
// with amax the block's largest magnitude and every operation rounded to fp32 (so that two implementations agree bit for bit).  Symmetric, because zero has to
// stay zero (a ReLU's border); 64 elements, because a block is then 8 lanes of 8 elements (16-byte pieces of a 16-bit tensor) and the scales cost 1/16 of the
// codes.  The step is amax / 127, the error of an element at most half of it.  amax < 2^-110: the block is kept as zeros (scale 0; 127 / amax would
// overflow).  A block that holds a NaN or an infinity gets scale NaN: all of it comes back as NaN, so that a diverged activation stays visible.
//
// A checkpoint of the input of a norm with ReLU / LeakyReLU is rounded TO ITS SIDE: where x and its rounded value lie on different sides of the activation's border
// (z = 0), the code is the other neighbour of x, which lies on x's side.  The error there is up to a whole step, but the backward then takes exactly the forward's
// branch.  (Not where x is its block's largest and the border lies between it and 127 scale, a rounding apart: the neighbour of +-127 beyond it is no code.)
// Rounded to nearest, 1 element in 400 of a Gaussian changes sides, and each contributes its whole gradient: 7 % of a layer's gradient norm.
#pragma once
#include "common.h"

namespace e3n {

constexpr int DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2;         // E3_DT_* of include/e3unet.h
constexpr int CK_BLOCK = 64;
constexpr float CK_TINY = 0x1p-110f;

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

template <int DT> struct Elem { typedef unsigned short T; };
template <> struct Elem<DT_F32> { typedef float T; };

template <int DT> __device__ __forceinline__ float to_f32(typename Elem<DT>::T v) {
    if constexpr (DT == DT_F32) return v;
    else if constexpr (DT == DT_BF16) return __uint_as_float((unsigned)v << 16);
    else return (float)__builtin_bit_cast(_Float16, v);
}
template <int DT> __device__ __forceinline__ typename Elem<DT>::T from_f32(float f) {       // round to nearest even; NaN stays NaN
    if constexpr (DT == DT_F32) return f;
    else if constexpr (DT == DT_BF16) return __builtin_bit_cast(unsigned short, (__bf16)f);
    else {
        asm("" : "+v"(f));       // (the fp32 value is the result: hipcc otherwise rounds some forms of its last operation straight to 16 bits, v_fma_mixlo_f16, and forms differ)
        return __builtin_bit_cast(unsigned short, (_Float16)f);
    }
}

// V consecutive channels of a voxel as they lie in memory: a piece of 16 bytes (V = wide_of(type): 4 fp32, 8 16-bit elements; C, row length and address in
// multiples of it), or V = 1.  (8 fp32 elements per lane, two accesses that each fill half of every line: the pass that restores a checkpoint 89 us instead of
// 62 for 268 MB of output.)
template <int DT, int V> struct Raw { typename Elem<DT>::T v; };
template <> struct Raw<DT_F32, 4> { f32x4 v; };
template <> struct Raw<DT_BF16, 8> { u16x8 v; };
template <> struct Raw<DT_F16, 8> { u16x8 v; };

// NT: non-temporal, for data that nobody reads again
template <int DT, int V, bool NT = false> __device__ __forceinline__ Raw<DT, V> load_raw(const typename Elem<DT>::T* p) {
    typedef decltype(Raw<DT, V>::v) P;
    Raw<DT, V> r;
    if constexpr (NT) r.v = __builtin_nontemporal_load(reinterpret_cast<const P*>(p));
    else r.v = *reinterpret_cast<const P*>(p);
    return r;
}
template <int DT, int V> __device__ __forceinline__ void unpack_raw(const Raw<DT, V>& r, float (&f)[V]) {
    if constexpr (V == 1) f[0] = to_f32<DT>(r.v);
    else if constexpr (DT == DT_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = r.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = to_f32<DT>(r.v[e]);
    }
}
template <int DT, int V, bool NT = false> __device__ __forceinline__ void store_f32(typename Elem<DT>::T* p, const float (&f)[V]) {
    typedef decltype(Raw<DT, V>::v) P;
    P o;
    if constexpr (V == 1) o = from_f32<DT>(f[0]);
    else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = from_f32<DT>(f[e]);
    }
    if constexpr (NT) __builtin_nontemporal_store(o, reinterpret_cast<P*>(p));
    else *reinterpret_cast<P*>(p) = o;
}

// V codes of a checkpoint and their scale
template <int V> struct RawQ { signed char q; float s; };
template <> struct RawQ<4> { unsigned q[1]; float s; };
template <> struct RawQ<8> { unsigned q[2]; float s; };
template <int V> __device__ __forceinline__ RawQ<V> load_q(const signed char* q, const float* scale, size_t e) {       // e: flat element, a multiple of V
    RawQ<V> r;
    if constexpr (V == 1) r.q = q[e];
    else if constexpr (V == 4) r.q[0] = *reinterpret_cast<const unsigned*>(q + e);
    else { const uint2 t = *reinterpret_cast<const uint2*>(q + e); r.q[0] = t.x; r.q[1] = t.y; }
    r.s = scale[e / CK_BLOCK];
    return r;
}
template <int V> __device__ __forceinline__ void unpack_q(const RawQ<V>& r, float (&f)[V]) {
#pragma clang fp contract(off)          // (the value is the ROUNDED product wherever it is used: fused into a reader's x - mean it would be another one)
    if constexpr (V == 1) f[0] = (float)r.q * r.s;
    else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (float)(signed char)(r.q[e / 4] >> (8 * (e % 4))) * r.s;
    }
}

// maximum over groups of 2^k consecutive lanes: inside a row of 16 lanes with DPP (neighbour, pair, half row, row; each step's partner holds the other half's
// maximum), beyond with permutes
template <int LANES> __device__ __forceinline__ unsigned group_max(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));               // quad_perm 1 0 3 2
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));               // quad_perm 2 3 0 1
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, false));              // row_half_mirror
    if constexpr (LANES >= 16) m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xf, 0xf, false));      // row_mirror
    if constexpr (LANES == 64) { m = max(m, (unsigned)__shfl_xor((int)m, 16)); m = max(m, (unsigned)__shfl_xor((int)m, 32)); }
    return m;
}

// A block's scale and codes from the values of its lanes: 64 / V consecutive lanes of a wave hold one block, V consecutive elements each (lanes outside the tensor
// pass zeros).  Magnitudes are compared as integers, where infinities and NaNs are the largest.  EVERY lane of the wave has to get here.
template <int V> struct Codes { signed char q[V]; float scale; };
template <int V> __device__ __forceinline__ Codes<V> encode_block(const float (&f)[V]) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) m = max(m, __float_as_uint(f[e]) & 0x7fffffffu);
    m = group_max<CK_BLOCK / V>(m);
    const float amax = __uint_as_float(m);
    const bool none = m < __float_as_uint(CK_TINY), bad = m >= 0x7f800000u;
    const float inv = (none || bad) ? 0.f : 127.f / amax;
    Codes<V> c;
    c.scale = none ? 0.f : (bad ? __uint_as_float(0x7fc00000u) : amax * (1.f / 127.f));
#pragma unroll
    for (int e = 0; e < V; ++e) c.q[e] = (none || bad) ? (signed char)0 : (signed char)(int)rintf(f[e] * inv);
    return c;
}
// the value of code e
template <int V> __device__ __forceinline__ float code_value(const Codes<V>& c, int e) {
#pragma clang fp contract(off)
    return (float)c.q[e] * c.scale;
}
// code q of x with value v, moved to the other neighbour of x
__device__ __forceinline__ signed char other_neighbour(signed char q, float x, float v) {
    const int m = (int)q + (x > v ? 1 : -1);
    return (signed char)(m > 127 ? 127 : m < -127 ? -127 : m);
}

template <int V> __device__ __forceinline__ void store_codes(const Codes<V>& c, signed char* q, float* scale, size_t e) {
    if constexpr (V == 1) q[e] = c.q[0];
    else {
        unsigned w[V / 4];
#pragma unroll
        for (int k = 0; k < V; ++k) { const unsigned b = (unsigned)(unsigned char)c.q[k] << (8 * (k % 4)); w[k / 4] = k % 4 ? w[k / 4] | b : b; }
        if constexpr (V == 4) *reinterpret_cast<unsigned*>(q + e) = w[0];
        else *reinterpret_cast<uint2*>(q + e) = make_uint2(w[0], w[V / 4 - 1]);
    }
    if (e % CK_BLOCK == 0) scale[e / CK_BLOCK] = c.scale;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int wide_of(int dt) { return dt == DT_F32 ? 4 : 8; }
// whether the rows of a view, or the codes of a checkpoint, allow 16-byte pieces
inline bool wide_rows(int dt, const void* p, int ldc, int C) { return C % wide_of(dt) == 0 && aligned16(p) && ldc % wide_of(dt) == 0; }
inline bool wide_codes(int dt, const void* q, int C) { return C % wide_of(dt) == 0 && (uintptr_t)q % wide_of(dt) == 0; }

}  // namespace e3n

// Which side of the border an element is on, for the pass that writes a checkpoint by itself.  rule 0: no border; 1: the exact sign of (x - mean) rstd gamma + beta
// with mean, rstd [N][G] and gamma, beta [C] or nullptr (what group_norm.hip decides by), S voxels to a sample; 2: the sign of fmaf(x, a[c], b[c]) (elementwise.hip)
struct Border { int rule = 0; const float *mean = nullptr, *rstd = nullptr, *gamma = nullptr, *beta = nullptr; const float *a = nullptr, *b = nullptr; long long S = 1; int G = 1; };

// launchers shared with the fused forms
int launch_checkpoint8_pack(int dt, const void* x, int x_ldc, long long vox, int C, signed char* q, float* scale, const Border& border, hipStream_t s);
int launch_checkpoint8_unpack(int dt, const signed char* q, const float* scale, long long vox, int C, void* y, int y_ldc, hipStream_t s);
// the fp32 executor's: raw [N][D][H][W][C], a with rows of a_ldc, pooled (or nullptr) with windows of (kd, 2, 2)
struct RestoreArgs {
    const signed char* q; const float* qs; float* raw; const float *scale, *shift; float* a; int a_ldc; float* pooled; int kd; int N, D, H, W, C; ActArg act;
};
int launch_checkpoint8_act(const RestoreArgs& r, hipStream_t s);
int launch_checkpoint8_windows(const RestoreArgs& r, signed char* codes, bool side, hipStream_t s);      // (reads r.raw; r.q, r.a, r.pooled are not used)
