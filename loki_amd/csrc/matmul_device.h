// matmul_device.h -- what the kernels of the 16-bit products share: types, activations, expert lookup, epilogues.
#pragma once
#include "moe_common.h"
#include "moe_kernels.h"
#include <algorithm>
#include <type_traits>

namespace lk {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
template <class T> struct Vec;
template <> struct Vec<__bf16> { typedef bf16x8 v8; typedef bf16x4 v4; };
template <> struct Vec<_Float16> { typedef f16x8 v8; typedef f16x4 v4; };
template <class T> using V8 = typename Vec<T>::v8;
template <class T> using V4 = typename Vec<T>::v4;

// D[16][16] += A[16][32] B[32][16]: lane (r, g) = 16 g + r holds A[r][8 g ..] and B[8 g ..][r], and D[4 g + i][r]
__device__ __forceinline__ f32x4 mfma32(bf16x8 a, bf16x8 b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
    (void) a; (void) b; return c;
#endif
}
__device__ __forceinline__ f32x4 mfma32(f16x8 a, f16x8 b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
    (void) a; (void) b; return c;
#endif
}

// ---------------------------------------------------------------- activations z s(g(z)), s(t) = 1 / (1 + e^-t)
// silu: g = z; gelu: g = 2 sqrt(2 / pi) (z + 0.044715 z^3), the tanh form. In fp32: e^-t and the reciprocal by their instructions (a division's ten
// cost 8192 x 16384 results 100 us). e^-t is 2^(-t log2 e): the constant's and the product's rounding, 1.22 * 2^-24 of the exponent, come to
// 1.3 |t| 2^-24 of it, and the two instructions and the sum to 5 * 2^-24. What that does to s is (1 - s) of the former: s is within
// (1.3 |t| (1 - s) + 5) 2^-24 of itself, 5 * 2^-24 where t is large, 120 * 2^-24 at t = -87, where s is 2^-126. A factor below 2^-126 is 0.
constexpr float GELU_C = 1.5957691216057308f, GELU_A = 0.044715f;
__device__ __forceinline__ float sigma(float t) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * t)); }
template <int ACT> __device__ __forceinline__ float act_arg(float z) { return ACT == ACT_GELU ? GELU_C * (z + GELU_A * z * z * z) : z; }
template <int ACT> __device__ __forceinline__ float act_fn(float z) { return ACT == ACT_NONE ? z : z * sigma(act_arg<ACT>(z)); }
__device__ __forceinline__ void activate8(int act, const float (&z)[8], float (&y)[8]) {   // (act is the launch's)
    if (act == ACT_SILU) {
#pragma unroll
        for (int u = 0; u < 8; ++u) { y[u] = act_fn<ACT_SILU>(z[u]); }
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int u = 0; u < 8; ++u) { y[u] = act_fn<ACT_GELU>(z[u]); }
    } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) { y[u] = z[u]; }
    }
}
// the derivative: s(g) + z g' s(g) s(-g)
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
    if (ACT == ACT_NONE) { return 1.f; }
    const float t = act_arg<ACT>(z), s = sigma(t), r = sigma(-t), d = ACT == ACT_GELU ? GELU_C * (1.f + 3.f * GELU_A * z * z) : 1.f;
    const float q = s * r;
    return q > 0.f ? s + z * d * q : s;   // (z d may be infinite where s or r has vanished)
}

// ---------------------------------------------------------------- slots
struct Span { int begin, end; };
// expert e's slots, inside 0 .. n whatever the offsets say
__device__ __forceinline__ Span span_of(const int * offsets, int n, int e) {
    if (!offsets) { return { 0, n }; }
    const int a = min(max(offsets[e], 0), n), b = min(max(offsets[e + 1], 0), n);
    return { a, max(a, b) };
}
// the pair's row: perm[slot] / topk by a product with 2^32 / topk rounded up (exact below 2^28 for topk <= 8); rows outside 0 .. xrows - 1
// come out as xrows or more
__device__ __forceinline__ uint32_t pair_row(uint32_t pair, uint32_t magic) { return magic ? __umulhi(pair, magic) : pair; }

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uni64(const void * p) {
    const uint64_t v = (uint64_t) p;
    return ((uint64_t) (uint32_t) uni((int) (uint32_t) (v >> 32)) << 32) | (uint32_t) uni((int) (uint32_t) v);
}

// m-tiles of the experts before e, lane l's of experts 4 l .. 4 l + 3 (no LDS: the operands may fill it); all: of all experts
struct Tiles {
    int first[4], all;
    __device__ __forceinline__ Tiles(const int * offsets, int n, int n_exp, int bm) {
        const int l = lane_id();
        int c[4], s = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = 4 * l + j;
            c[j] = 0;
            if (e < n_exp) { const Span sp = span_of(offsets, n, e); c[j] = (sp.end - sp.begin + bm - 1) / bm; }
            s += c[j];
        }
        int si = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int v = __shfl_up(si, o); if (l >= o) { si += v; } }
        int at = si - s;
#pragma unroll
        for (int j = 0; j < 4; ++j) { first[j] = at; at += c[j]; }
        all = __builtin_amdgcn_readlane(at, 63);
    }
    __device__ __forceinline__ int before(int e) const {   // (e uniform)
        int v = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { const int w = __builtin_amdgcn_readlane(first[j], (e >> 2) & 63); v = (e & 3) == j ? w : v; }
        return e >= NEXP_MAX ? all : v;
    }
    // the expert of m-tile i, i < all: the last one whose tiles begin at or before it
    __device__ __forceinline__ int expert(int i) const {
        int e = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { e += __popcll(__ballot(first[j] <= i)); }
        return uni(e) - 1;
    }
};

// ---------------------------------------------------------------- 8 values next to each other
template <class T> __device__ __forceinline__ V8<T> rounded(const float (&v)[8]) {
    V8<T> u;
#pragma unroll
    for (int i = 0; i < 8; ++i) { u[i] = (T) v[i]; }
    return u;
}
template <class T> __device__ __forceinline__ void put8(T * p, const float (&v)[8]) { *(LK_GLOBAL V8<T> *) p = rounded<T>(v); }
__device__ __forceinline__ void put8(float * p, const float (&v)[8]) {
    *(LK_GLOBAL f32x4 *) p = (f32x4) { v[0], v[1], v[2], v[3] };
    *(LK_GLOBAL f32x4 *) (p + 4) = (f32x4) { v[4], v[5], v[6], v[7] };
}
template <class T> __device__ __forceinline__ void add8(const T * p, float (&v)[8]) {
    const V8<T> u = *(const LK_GLOBAL V8<T> *) p;
#pragma unroll
    for (int i = 0; i < 8; ++i) { v[i] += (float) u[i]; }
}
__device__ __forceinline__ void add8(const float * p, float (&v)[8]) {
    const f32x4 a = *(const LK_GLOBAL f32x4 *) p, b = *(const LK_GLOBAL f32x4 *) (p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] += a[i]; v[4 + i] += b[i]; }
}

}  // namespace lk
