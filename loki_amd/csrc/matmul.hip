// matmul.hip -- products of bfloat16 / float16 matrices, dense or grouped by expert, and their backward pass.
//
//   forward  y[s][r]  = sum_k x[row(s)][k] W[e][r][k], with an epilogue     s: expert e's slots
//   dx       dx[s][k] = sum_r dz[s][r] W[e][r][k] (+ dz2 W2)
//   dW       dW[e][r][k] = sum over e's slots of dz[s][r] x[row(s)][k]
//
// All three are D[m][n] = sum_k A[m][k] B[n][k] with D's rows along n in memory. The matrix cores take B as their first operand, so that a
// lane's four results lie next to each other in a row of D.
#include "matmul_device.h"

namespace lk {
namespace {

constexpr int TM = 64, TN = 64, TK = 32, LDK = TK + 8;

// the expert and first slot of the launch's m-tile `mt` of `tm` slots; false: there is no such tile
__device__ bool find_tile(const int * offsets, int n, int n_exp, int tm, int mt, int & e, Span & s) {
    for (e = 0; e < n_exp; ++e) {
        s = span_of(offsets, n, e);
        const int tiles = (s.end - s.begin + tm - 1) / tm;
        if (mt < tiles) { s.begin += mt * tm; return true; }
        mt -= tiles;
    }
    return false;
}

// rows 0 .. nr - 1 of `p` (row i at p + at(i) * ld), columns k0 .. min(k0 + TK, K) - 1, as lds[i][k]; what is not there is 0
template <class T, class At> __device__ __forceinline__ void stage_rows(T (*lds)[LDK], const T * p, size_t ld, int nr, int k0, int K, At at) {
    for (int i = threadIdx.x; i < 64 * TK; i += 256) {
        const int r = i / TK, k = i % TK;
        T v = (T) 0.f;
        if (r < nr && k0 + k < K) { const int64_t row = at(r); if (row >= 0) { v = p[(size_t) row * ld + k0 + k]; } }
        lds[r][k] = v;
    }
}
// rows k0 .. min(k0 + TK, K) - 1 of `p`, columns c0 .. c0 + nc - 1, as lds[column][row]
template <class T, class At> __device__ __forceinline__ void stage_cols(T (*lds)[LDK], const T * p, size_t ld, int c0, int nc, int k0, int K, At at) {
    for (int i = threadIdx.x; i < 64 * TK; i += 256) {
        const int k = i / 64, c = i % 64;
        T v = (T) 0.f;
        if (c < nc && k0 + k < K) { const int64_t row = at(k0 + k); if (row >= 0) { v = p[(size_t) row * ld + c0 + c]; } }
        lds[c][k] = v;
    }
}
// a wave's 64 x 16 of the tile's products of one TK: n-rows 16 w .. of lb, all m of la
template <class T> __device__ __forceinline__ void products(const T (*la)[LDK], const T (*lb)[LDK], f32x4 (&acc)[4]) {
    const int w = threadIdx.x >> 6, lane = lane_id(), r = lane & 15, g = lane >> 4;
    const V8<T> b = *reinterpret_cast<const V8<T> *>(&lb[16 * w + r][8 * g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) { acc[i] = mfma32(b, *reinterpret_cast<const V8<T> *>(&la[16 * i + r][8 * g]), acc[i]); }
}

template <class T, int ACT> __global__ void __launch_bounds__(256) k_mm(MatmulArgs a) {
    __shared__ __attribute__((aligned(16))) T la[TM][LDK], lb[TN][LDK], lc[TN][LDK];
    int e; Span s;
    if (!find_tile(a.offsets, a.n, a.n_exp, TM, blockIdx.x, e, s)) { return; }
    const int n0 = blockIdx.y * TN, nm = min(TM, s.end - s.begin), nn = min(TN, a.R - n0);
    const T * W = (const T *) a.W + ((size_t) e * a.R + n0) * a.K, * W2 = a.W2 ? (const T *) a.W2 + ((size_t) e * a.R + n0) * a.K : nullptr;
    auto row = [&](int i) -> int64_t {
        if (!a.perm) { return s.begin + i; }
        const uint32_t t = pair_row((uint32_t) a.perm[s.begin + i], a.magic);
        return t < (uint32_t) a.xrows ? (int64_t) t : -1;
    };
    f32x4 acc[4] = {}, acc2[4] = {};
    for (int k0 = 0; k0 < a.K; k0 += TK) {
        __syncthreads();
        stage_rows(la, (const T *) a.x, a.K, nm, k0, a.K, row);
        stage_rows(lb, W, a.K, nn, k0, a.K, [](int i) -> int64_t { return i; });
        if (W2) { stage_rows(lc, W2, a.K, nn, k0, a.K, [](int i) -> int64_t { return i; }); }
        __syncthreads();
        products<T>(la, lb, acc);
        if (W2) { products<T>(la, lc, acc2); }
    }
    const int w = threadIdx.x >> 6, lane = lane_id(), r = lane & 15, g = lane >> 4;
    for (int i = 0; i < 4; ++i) {
        for (int u = 0; u < 4; ++u) {
            const int m = 16 * i + r, nc = n0 + 16 * w + 4 * g + u;
            if (m >= nm || nc >= a.R) { continue; }
            const size_t at = (size_t) (s.begin + m) * a.R + nc;
            const float z = acc[i][u] + (a.bias ? a.bias[(size_t) e * a.R + nc] : 0.f), z2 = acc2[i][u];
            float y = act_fn<ACT>(z);
            if (W2) { y *= z2; }
            if (a.residual) { y += (float) ((const T *) a.residual)[at]; }
            if (a.y_f32) { ((float *) a.y)[at] = y; } else { ((T *) a.y)[at] = (T) y; }
            if (a.z) { ((T *) a.z)[at] = (T) z; }
            if (a.z2) { ((T *) a.z2)[at] = (T) z2; }
        }
    }
}

template <class T> __global__ void __launch_bounds__(256) k_mm_dx(MatmulGradArgs a) {
    __shared__ __attribute__((aligned(16))) T la[TM][LDK], lb[TN][LDK];
    int e; Span s;
    if (!find_tile(a.offsets, a.n, a.n_exp, TM, blockIdx.x, e, s)) { return; }
    const int n0 = blockIdx.y * TN, nm = min(TM, s.end - s.begin), nn = min(TN, a.K - n0);
    auto same = [](int i) -> int64_t { return i; };
    f32x4 acc[4] = {};
    for (int src = 0; src < (a.dz2 ? 2 : 1); ++src) {
        const T * dz = (const T *) (src ? a.dz2 : a.dz) + (size_t) s.begin * a.R, * W = (const T *) (src ? a.W2 : a.W) + (size_t) e * a.R * a.K;
        for (int k0 = 0; k0 < a.R; k0 += TK) {
            __syncthreads();
            stage_rows(la, dz, a.R, nm, k0, a.R, same);
            stage_cols(lb, W, a.K, n0, nn, k0, a.R, same);
            __syncthreads();
            products<T>(la, lb, acc);
        }
    }
    const int w = threadIdx.x >> 6, lane = lane_id(), r = lane & 15, g = lane >> 4;
    for (int i = 0; i < 4; ++i) {
        for (int u = 0; u < 4; ++u) {
            const int m = 16 * i + r, nc = n0 + 16 * w + 4 * g + u;
            if (m < nm && nc < a.K) { ((T *) a.dx)[(size_t) (s.begin + m) * a.K + nc] = (T) acc[i][u]; }
        }
    }
}

template <class T> __global__ void __launch_bounds__(256) k_mm_dw(MatmulGradArgs a) {
    __shared__ __attribute__((aligned(16))) T la[TM][LDK], lb[TN][LDK];
    const int e = blockIdx.z % a.n_exp, second = blockIdx.z / a.n_exp;
    const Span s = span_of(a.offsets, a.n, e);
    const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN, nm = min(TM, a.R - m0), nn = min(TN, a.K - n0), len = s.end - s.begin;
    const T * dz = (const T *) (second ? a.dz2 : a.dz) + (size_t) s.begin * a.R;
    auto row = [&](int i) -> int64_t {
        if (!a.perm) { return s.begin + i; }
        const uint32_t t = pair_row((uint32_t) a.perm[s.begin + i], a.magic);
        return t < (uint32_t) a.xrows ? (int64_t) t : -1;
    };
    f32x4 acc[4] = {};
    for (int k0 = 0; k0 < len; k0 += TK) {
        __syncthreads();
        stage_cols(la, dz, a.R, m0, nm, k0, len, [](int i) -> int64_t { return i; });
        stage_cols(lb, (const T *) a.x, a.K, n0, nn, k0, len, row);
        __syncthreads();
        products<T>(la, lb, acc);
    }
    const int w = threadIdx.x >> 6, lane = lane_id(), r = lane & 15, g = lane >> 4;
    for (int i = 0; i < 4; ++i) {
        for (int u = 0; u < 4; ++u) {
            const int m = m0 + 16 * i + r, nc = n0 + 16 * w + 4 * g + u;
            if (m >= a.R || nc >= a.K) { continue; }
            const size_t at = ((size_t) e * a.R + m) * a.K + nc;
            float v = acc[i][u];
            if (a.dw_f32) { float * d = (float *) (second ? a.dW2 : a.dW) + at; *d = a.accumulate ? *d + v : v; }
            else { T * d = (T *) (second ? a.dW2 : a.dW) + at; *d = (T) (a.accumulate ? (float) *d + v : v); }
        }
    }
}

constexpr unsigned ceil_div(int64_t a, int64_t b) { return (unsigned) ((a + b - 1) / b); }

template <class T> hipError_t go_fwd(const MatmulArgs & a, hipStream_t st) {
    const dim3 grid(ceil_div(a.n, TM) + (a.offsets ? a.n_exp : 0), ceil_div(a.R, TN));
    if (a.act == ACT_SILU) { k_mm<T, ACT_SILU><<<grid, 256, 0, st>>>(a); }
    else if (a.act == ACT_GELU) { k_mm<T, ACT_GELU><<<grid, 256, 0, st>>>(a); }
    else { k_mm<T, ACT_NONE><<<grid, 256, 0, st>>>(a); }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_matmul(const MatmulArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? go_fwd<__bf16>(a, st) : go_fwd<_Float16>(a, st); }
hipError_t launch_matmul_dx(const MatmulGradArgs & a, hipStream_t st) {
    const dim3 grid(ceil_div(a.n, TM) + (a.offsets ? a.n_exp : 0), ceil_div(a.K, TN));
    if (a.type == TYPE_BF16) { k_mm_dx<__bf16><<<grid, 256, 0, st>>>(a); } else { k_mm_dx<_Float16><<<grid, 256, 0, st>>>(a); }
    return hipGetLastError();
}
hipError_t launch_matmul_dw(const MatmulGradArgs & a, hipStream_t st) {
    const dim3 grid(ceil_div(a.K, TN), ceil_div(a.R, TM), a.n_exp * (a.dW2 ? 2 : 1));
    if (a.type == TYPE_BF16) { k_mm_dw<__bf16><<<grid, 256, 0, st>>>(a); } else { k_mm_dw<_Float16><<<grid, 256, 0, st>>>(a); }
    return hipGetLastError();
}

}  // namespace lk
