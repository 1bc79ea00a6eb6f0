// matmul_rows.hip -- what goes over rows beside the 16-bit products: the epilogue's gradient with the bias's, the sum of a row's picks
// under the routing weights and the gradients of both. Many rows are bound by memory: every value is read and written once, 16 bytes a lane.
// A few rows of picks are bound by loads that wait for each other: 8 picks of 7168, 6 rows, 5.0 and 7.6 us.
#include "matmul_device.h"

namespace lk {
namespace {

constexpr int RT = 256;   // threads of a workgroup

template <class T> struct Row8 { float v[8]; };
template <class T> __device__ __forceinline__ Row8<T> load8(const T * p) {
    const V8<T> u = *(const LK_GLOBAL V8<T> *) p;
    Row8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) { r.v[i] = (float) u[i]; }
    return r;
}
template <class T> __device__ __forceinline__ void store8(T * p, const float (&v)[8]) {
    V8<T> u;
#pragma unroll
    for (int i = 0; i < 8; ++i) { u[i] = (T) v[i]; }
    *(LK_GLOBAL V8<T> *) p = u;
}
__device__ __forceinline__ void store8(float * p, const float (&v)[8]) {
    *(LK_GLOBAL f32x4 *) p = (f32x4) { v[0], v[1], v[2], v[3] };
    *(LK_GLOBAL f32x4 *) (p + 4) = (f32x4) { v[4], v[5], v[6], v[7] };
}

// dz (and dz2) of 8 values; returns dz in fp32
template <class T, int ACT> __device__ __forceinline__ void back8(const ActGradArgs & a, size_t at, float (&d)[8]) {
    const Row8<T> dy = load8((const T *) a.dy + at);
    if (ACT == ACT_NONE && !a.z2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) { d[i] = dy.v[i]; }
    } else {
        const Row8<T> z = load8((const T *) a.z + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) { d[i] = dy.v[i] * act_slope<ACT>(z.v[i]); }
        if (a.z2) {
            const Row8<T> z2 = load8((const T *) a.z2 + at);
            float d2[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) { d2[i] = dy.v[i] * act_fn<ACT>(z.v[i]); d[i] *= z2.v[i]; }
            if (a.dz2) { store8((T *) a.dz2 + at, d2); }
        }
    }
    if (a.dz) { store8((T *) a.dz + at, d); }
}

// without a bias the slots are one flat array (rows are next to each other): 8 values a thread
template <class T, int ACT> __global__ void __launch_bounds__(RT) k_act_grad(ActGradArgs a) {
    int first = 0, last = a.n;
    if (a.offsets) { first = min(max(a.offsets[0], 0), a.n); last = min(max(a.offsets[a.n_exp], 0), a.n); }
    const int64_t end = (int64_t) last * (a.R / 8);
    for (int64_t i = (int64_t) first * (a.R / 8) + (int64_t) blockIdx.x * RT + threadIdx.x; i < end; i += (int64_t) gridDim.x * RT) {
        float d[8];
        back8<T, ACT>(a, (size_t) i * 8, d);
    }
}
// with it, a workgroup takes `cw` threads' columns (8 each) of one chunk of an expert's rows and sums what it makes of them: RT / cw rows at
// a time, each thread its rows in order, then the threads of a column in order
template <class T, int ACT> __global__ void __launch_bounds__(RT) k_act_grad_bias(ActGradArgs a, int cw, int cb) {
    __shared__ float lds[RT][9];
    const int e = blockIdx.y, chunk = blockIdx.x / cb, col = (blockIdx.x % cb) * cw + threadIdx.x % cw, lane = threadIdx.x / cw, step = RT / cw;
    const Span s = span_of(a.offsets, a.n, e);
    const int64_t len = s.end - s.begin;
    const int r0 = s.begin + (int) (len * chunk / a.chunks), r1 = s.begin + (int) (len * (chunk + 1) / a.chunks);
    const bool on = col < a.R / 8;
    float sum[8] = {};
    if (on) {
#pragma unroll 4
        for (int r = r0 + lane; r < r1; r += step) {
            float d[8];
            back8<T, ACT>(a, (size_t) r * a.R + 8 * col, d);
#pragma unroll
            for (int i = 0; i < 8; ++i) { sum[i] += d[i]; }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) { lds[threadIdx.x][i] = sum[i]; }
    __syncthreads();
    if (lane == 0 && on) {
        for (int l = 1; l < step; ++l) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { sum[i] += lds[l * cw + threadIdx.x][i]; }
        }
        const size_t at = (size_t) 8 * col;
        if (a.chunks > 1) { store8(a.part + ((size_t) e * a.chunks + chunk) * a.R + at, sum); return; }
        float * d = a.dbias + (size_t) e * a.R + at;
        if (a.accumulate) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { sum[i] += d[i]; }
        }
        store8(d, sum);
    }
}
// the chunks' sums, in order
__global__ void __launch_bounds__(RT) k_bias_join(const float * __restrict__ part, int chunks, int R, int64_t all, int accumulate, float * __restrict__ dbias) {
    const int64_t i = (int64_t) blockIdx.x * RT + threadIdx.x;
    if (i >= all) { return; }
    const float * p = part + (i / R) * chunks * R + i % R;
    float v = 0.f;
#pragma unroll 8
    for (int c = 0; c < chunks; ++c) { v += p[(size_t) c * R]; }
    dbias[i] = accumulate ? dbias[i] + v : v;
}

// the slot of pair (t, k), or -1
__device__ __forceinline__ int slot_of(const CombineArgs & a, int64_t i) {
    if (a.sel) { const int e = a.sel[i]; if (e < 0 || e >= a.n_exp) { return -1; } }
    const int s = a.inv[i];
    return (unsigned) s < (unsigned) a.P ? s : -1;
}

// y = residual + sum over the picks, in their order, 8 columns a thread; a workgroup takes RT / cw rows of cw threads
template <class T> __global__ void __launch_bounds__(RT) k_combine16(CombineArgs a, int cw, int cb, int t0) {   // (rows from t0 on)
    const int col = (blockIdx.x % cb) * cw + threadIdx.x % cw;
    const int64_t t = t0 + (int64_t) (blockIdx.x / cb) * (RT / cw) + threadIdx.x / cw;
    if (t >= a.n || col >= a.E / 8) { return; }
    const size_t at = (size_t) t * a.E + 8 * col;
    V8<T> o[MAXK];
    float w[MAXK];
#pragma unroll
    for (int k = 0; k < MAXK; ++k) {   // (the rows' loads before the sums; a pick's expert and slot are waited for before the next one's are asked for)
        const int s = k < a.topk ? slot_of(a, t * a.topk + k) : -1;
        w[k] = s >= 0 ? (a.w ? a.w[t * a.topk + k] : 1.f) : 0.f;
        o[k] = (V8<T>) {};
        if (s >= 0) { o[k] = *(const LK_GLOBAL V8<T> *) ((const T *) a.o + (size_t) s * a.E + 8 * col); }
    }
    float y[8] = {};
    if (a.residual) {
        const Row8<T> r = load8((const T *) a.residual + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) { y[i] = r.v[i]; }
    }
#pragma unroll
    for (int k = 0; k < MAXK; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) { y[i] = __builtin_fmaf(w[k], (float) o[k][i], y[i]); }
    }
    if (a.y_f32) { store8((float *) a.y + at, y); } else { store8((T *) a.y + at, y); }
}

// d_o and dw of one row: W waves, each its columns, then the waves' sums in order. d_o may be o, so a pick's row is read, waited for and its gradient
// written before the next pick's is asked for
template <class T, int W> __global__ void __launch_bounds__(64 * W) k_combine16_grad(CombineArgs a, int t0) {
    __shared__ float lds[W][MAXK];
    const int64_t t = t0 + (int64_t) blockIdx.x;
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    int s[MAXK];
    float w[MAXK], dot[MAXK];
#pragma unroll
    for (int k = 0; k < MAXK; ++k) {
        s[k] = k < a.topk ? slot_of(a, t * a.topk + k) : -1;
        w[k] = s[k] >= 0 && a.w ? a.w[t * a.topk + k] : 1.f;
        dot[k] = 0.f;
    }
    for (int col = threadIdx.x; col < a.E / 8; col += 64 * W) {
        const Row8<T> d = load8((const T *) a.dy + (size_t) t * a.E + 8 * col);
#pragma unroll
        for (int k = 0; k < MAXK; ++k) {
            if (s[k] < 0) { continue; }
            const size_t at = (size_t) s[k] * a.E + 8 * col;
            if (a.dw) {
                const Row8<T> o = load8((const T *) a.o + at);
#pragma unroll
                for (int i = 0; i < 8; ++i) { dot[k] = __builtin_fmaf(o.v[i], d.v[i], dot[k]); }
            }
            if (a.d_o) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) { v[i] = w[k] * d.v[i]; }
                store8((T *) a.d_o + at, v);
            }
        }
    }
    if (!a.dw) { return; }
#pragma unroll
    for (int k = 0; k < MAXK; ++k) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { dot[k] += __shfl_xor(dot[k], o); }
    }
    if (W > 1) {
        if (lane == 0) {
#pragma unroll
            for (int k = 0; k < MAXK; ++k) { lds[wave][k] = dot[k]; }
        }
        __syncthreads();
    }
    if ((int) threadIdx.x < a.topk) {
        float v = 0.f;
        if (W > 1) { for (int i = 0; i < W; ++i) { v += lds[i][threadIdx.x]; } }
        else {
#pragma unroll
            for (int k = 0; k < MAXK; ++k) { v = (int) threadIdx.x == k ? dot[k] : v; }
        }
        a.dw[t * a.topk + threadIdx.x] = v;
    }
}

constexpr unsigned blocks(int64_t n, int64_t per) { return (unsigned) ((n + per - 1) / per); }
constexpr int MOST = 1 << 22;   // workgroups of a launch, which has fewer than 2^32 threads (more rows: more launches)
// threads along a row of `nc` pieces of 8: a power of two, at most RT
constexpr int row_threads(int nc) { int w = 1; while (w < nc && w < RT) { w *= 2; } return w; }

// with a bias's gradient: a line of a row (8 threads) where experts have few rows, so that a workgroup takes them all and nothing is left to join
// (gelu, us, against whole rows in chunks: 37 rows of 7168 5.9 / 8.5; 64 experts of 94, 1024 12 / 14; 256 of 128, 2048 83 / 92; 64 of 512, 2048 98 / 92; 501 of
// 7168 16 / 14; 1000 36 / 22)
constexpr int FEW_ROWS = 128;
int bias_threads(int n, int R, int n_exp) { return n / n_exp <= FEW_ROWS ? std::min(row_threads(R / 8), 8) : row_threads(R / 8); }
template <class T, int ACT> hipError_t go_act(const ActGradArgs & a, hipStream_t st) {
    if (!a.dbias) {
        const int64_t all = (int64_t) a.n * (a.R / 8);
        k_act_grad<T, ACT><<<blocks(all, RT) < 16384 ? blocks(all, RT) : 16384, RT, 0, st>>>(a);
        return hipGetLastError();
    }
    const int cw = bias_threads(a.n, a.R, a.n_exp), cb = (int) blocks(a.R / 8, cw);
    k_act_grad_bias<T, ACT><<<dim3(cb * a.chunks, a.n_exp), RT, 0, st>>>(a, cw, cb);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.chunks > 1) {
        const int64_t all = (int64_t) a.n_exp * a.R;
        k_bias_join<<<blocks(all, RT), RT, 0, st>>>(a.part, a.chunks, a.R, all, a.accumulate, a.dbias);
        e = hipGetLastError();
    }
    return e;
}
template <class T> hipError_t go_act(const ActGradArgs & a, hipStream_t st) {
    return a.act == ACT_SILU ? go_act<T, ACT_SILU>(a, st) : a.act == ACT_GELU ? go_act<T, ACT_GELU>(a, st) : go_act<T, ACT_NONE>(a, st);
}
template <class T> hipError_t go_combine(const CombineArgs & a, hipStream_t st) {
    const int cw = row_threads(a.E / 8), cb = (int) blocks(a.E / 8, cw);
    const int most = MOST / cb * (RT / cw);
    for (int t0 = 0; t0 < a.n; t0 += most) { k_combine16<T><<<blocks(std::min(a.n - t0, most), RT / cw) * cb, RT, 0, st>>>(a, cw, cb, t0); }
    return hipGetLastError();
}
template <class T> hipError_t go_combine_grad(const CombineArgs & a, hipStream_t st) {
    for (int t0 = 0; t0 < a.n; t0 += MOST) {
        const unsigned rows = (unsigned) std::min(a.n - t0, MOST);
        if (a.E <= 512) { k_combine16_grad<T, 1><<<rows, 64, 0, st>>>(a, t0); }
        else if (a.n > 512) { k_combine16_grad<T, 4><<<rows, 256, 0, st>>>(a, t0); }
        else { k_combine16_grad<T, 16><<<rows, 1024, 0, st>>>(a, t0); }
    }
    return hipGetLastError();
}

}  // namespace

int act_grad_chunks(int n, int R, int n_exp) {
    if (n / n_exp <= FEW_ROWS) { return 1; }
    const int cw = row_threads(R / 8), cb = (int) blocks(R / 8, cw), rows = n / n_exp / (RT / cw);   // rows a thread sums, on average
    int c = 1;
    while (c < 128 && cb * n_exp * c < 1024 && rows > 8 * c) { c *= 2; }
    return c;
}
hipError_t launch_act_grad(const ActGradArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? go_act<__bf16>(a, st) : go_act<_Float16>(a, st); }
hipError_t launch_combine16(const CombineArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? go_combine<__bf16>(a, st) : go_combine<_Float16>(a, st); }
hipError_t launch_combine16_grad(const CombineArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? go_combine_grad<__bf16>(a, st) : go_combine_grad<_Float16>(a, st); }

}  // namespace lk
