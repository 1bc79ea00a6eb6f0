// balance.hip -- the balance loss of routed rows with its per-expert counts, and its gradient to the router's logits.
//
// Per sequence of T rows (s = sigmoid(z), p_te = s_te / sum_j s_tj, c_e = picks of expert e):
//   P_e = mean_t p_te,   f_e = n_exp c_e / (topk T),   loss = alpha sum_e f_e P_e
//   d loss / d z_te = alpha / T  p_te (1 - s_te) (f_e - sum_j f_j p_tj)              (the counts are constants)
// (the sequence-wise loss of the DeepSeek-V3 report, whose router this library has.) p does not change when a row's s are
// all scaled, so a row whose sigmoids are all tiny takes exp(z - max z) in their place; a row of -inf has p = 0.
#include "moe_device.h"
#include "moe_kernels.h"

#include <algorithm>

namespace lk {

namespace {

constexpr int BL_W = 16, BL_T = BL_W * 64;   // waves / threads per workgroup: a wave takes a row at a time
constexpr int BL_ROWS = 128;                 // rows per workgroup that a sequence is cut into, at least
constexpr float BL_TINY = 1e-10f;            // a row's sigmoid sum below which 1 + exp(-z) is exp(-z) to fp32 in every column

template <int CTRL> __device__ __forceinline__ float dppf(float v) { return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v))); }
__device__ __forceinline__ float rdlanef(float v, int l) { return __builtin_bit_cast(float, rdlane(__builtin_bit_cast(uint32_t, v), l)); }
__device__ __forceinline__ float wave_sum(float v) {
    v += dppf<DPP_XOR1>(v); v += dppf<DPP_XOR2>(v); v += dppf<DPP_HALF_MIRROR>(v); v += dppf<DPP_MIRROR>(v);
    return (rdlanef(v, 0) + rdlanef(v, 16)) + (rdlanef(v, 32) + rdlanef(v, 48));
}
__device__ __forceinline__ float wave_maxf(float v) {
    v = fmaxf(v, dppf<DPP_XOR1>(v)); v = fmaxf(v, dppf<DPP_XOR2>(v)); v = fmaxf(v, dppf<DPP_HALF_MIRROR>(v)); v = fmaxf(v, dppf<DPP_MIRROR>(v));
    return fmaxf(fmaxf(rdlanef(v, 0), rdlanef(v, 16)), fmaxf(rdlanef(v, 32), rdlanef(v, 48)));
}

// rows [a, b) of chunk c of sequence s
__device__ __forceinline__ void bl_rows(const BalanceArgs & g, int s, int c, int & a, int & b, int & T) {
    int lo = 0, hi = g.n;
    if (g.seq) { lo = min(max(g.seq[s], 0), g.n); hi = min(max(g.seq[s + 1], lo), g.n); }
    T = hi - lo;
    a = lo + (int) ((int64_t) T * c / g.chunks); b = lo + (int) ((int64_t) T * (c + 1) / g.chunks);
}

// a row's sigmoids: lane l holds the columns e = l + 64 j. q: the sigmoids (or their scaled stand-ins), om: 1 - sigmoid;
// returns 1 / sum q (0 where the row is all -inf)
template <int J> __device__ __forceinline__ float bl_sigmoids(const float (&z)[J], float (&q)[J], float (&om)[J]) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const float t = expf(-fabsf(z[j])), r = 1.f / (1.f + t);
        q[j] = z[j] >= 0.f ? r : t * r;
        om[j] = z[j] >= 0.f ? t * r : r;
        sum += q[j];
    }
    sum = wave_sum(sum);
    if (sum < BL_TINY) {
        float m = z[0];
#pragma unroll
        for (int j = 1; j < J; ++j) { m = fmaxf(m, z[j]); }
        m = wave_maxf(m);
        if (m == -INFINITY) { return 0.f; }
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) { q[j] = expf(z[j] - m); sum += q[j]; }
        sum = wave_sum(sum);
    }
    return 1.f / sum;
}

// f_e from a count (exact below 2^24)
__device__ __forceinline__ float bl_f(int cnt, const BalanceArgs & g, int T) { return (float) cnt * ((float) g.n_exp / ((float) g.topk * (float) T)); }

// the loss of one sequence from its sums: threads of a workgroup hold expert e = threadIdx.x (< n_exp); fixed order
__device__ __forceinline__ void bl_finish(const BalanceArgs & g, int s, int T, float psum, int cnt, float * scr) {
    const int e = threadIdx.x;
    float v = 0.f;
    if (e < g.n_exp) {
        g.counts[(size_t) s * g.n_exp + e] = cnt;
        if (T > 0) { v = bl_f(cnt, g, T) * (psum / (float) T); }
    }
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) { scr[threadIdx.x >> 6] = v; }
    __syncthreads();
    if (threadIdx.x == 0) {
        float tot = 0.f;
        for (int w = 0; w < NEXP_MAX / 64; ++w) { tot += scr[w]; }
        g.loss[s] = g.alpha * tot;
    }
}

template <int J>
__global__ void __launch_bounds__(BL_T) k_balance(BalanceArgs g) {
    __shared__ float s_p[BL_W][64 * J];
    __shared__ int s_c[NEXP_MAX];
    __shared__ float s_f[BL_W];
    const int s = blockIdx.y, c = blockIdx.x, lane = lane_id(), w = threadIdx.x >> 6, ne = g.n_exp;
    int a, b, T;
    bl_rows(g, s, c, a, b, T);
    if (threadIdx.x < NEXP_MAX) { s_c[threadIdx.x] = 0; }
    __syncthreads();
    for (int64_t i = (int64_t) a * g.topk + threadIdx.x; i < (int64_t) b * g.topk; i += BL_T) {
        const int e = g.sel[i];
        if ((unsigned) e < (unsigned) ne) { atomicAdd(&s_c[e], 1); }
    }
    float acc[J];
#pragma unroll
    for (int j = 0; j < J; ++j) { acc[j] = 0.f; }
    for (int t = a + w; t < b; t += BL_W) {
        float z[J], q[J], om[J];
#pragma unroll
        for (int j = 0; j < J; ++j) { const int e = lane + 64 * j; z[j] = e < ne ? g.logits[(size_t) t * ne + e] : -INFINITY; }
        const float inv = bl_sigmoids<J>(z, q, om);
#pragma unroll
        for (int j = 0; j < J; ++j) { acc[j] += q[j] * inv; }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) { s_p[w][lane + 64 * j] = acc[j]; }
    __syncthreads();
    const int e = threadIdx.x;
    float psum = 0.f; int cnt = 0;
    if (e < ne) {
        for (int v = 0; v < BL_W; ++v) { psum += s_p[v][e]; }
        cnt = s_c[e];
    }
    if (g.chunks == 1) { bl_finish(g, s, T, psum, cnt, s_f); return; }
    if (e < ne) {
        const size_t o = ((size_t) s * g.chunks + c) * ne + e;
        g.part[o] = psum; g.pcnt[o] = cnt;
    }
}

// chunks > 1: a sequence's sums over its chunks, four slices of them side by side and then in order, and its loss
__global__ void __launch_bounds__(BL_T) k_balance_join(BalanceArgs g) {
    __shared__ float s_p[4][NEXP_MAX];
    __shared__ int s_c[4][NEXP_MAX];
    __shared__ float s_f[BL_W];
    const int s = blockIdx.x, e = threadIdx.x & 255, k = threadIdx.x >> 8;
    int a, b, T;
    bl_rows(g, s, 0, a, b, T);
    float psum = 0.f; int cnt = 0;
    if (e < g.n_exp) {
        for (int c = k; c < g.chunks; c += 4) {
            const size_t o = ((size_t) s * g.chunks + c) * g.n_exp + e;
            psum += g.part[o]; cnt += g.pcnt[o];
        }
    }
    s_p[k][e] = psum; s_c[k][e] = cnt;
    __syncthreads();
    if (k == 0) {
        for (int i = 1; i < 4; ++i) { psum += s_p[i][e]; cnt += s_c[i][e]; }
    }
    bl_finish(g, s, T, k == 0 ? psum : 0.f, cnt, s_f);
}

template <int J>
__global__ void __launch_bounds__(BL_T) k_balance_grad(BalanceArgs g) {
    const int s = blockIdx.y, lane = lane_id(), w = threadIdx.x >> 6, ne = g.n_exp;
    if (s == g.nseq) {   // rows of no sequence: their gradient is 0
        const int64_t lo = min(max(g.seq[0], 0), g.n), hi = min(max(g.seq[g.nseq], 0), g.n);
        const int64_t gap = hi > lo ? hi - lo : 0, rest = ((int64_t) g.n - gap) * ne;
        for (int64_t i = (int64_t) blockIdx.x * BL_T + threadIdx.x; i < rest; i += (int64_t) gridDim.x * BL_T) {
            g.dlogits[i < lo * ne ? i : i + gap * ne] = 0.f;
        }
        return;
    }
    int a, b, T;
    bl_rows(g, s, blockIdx.x, a, b, T);
    if (a >= b) { return; }
    const float k = (g.gloss ? g.gloss[s] : 1.f) * g.alpha / (float) T;
    float f[J];
#pragma unroll
    for (int j = 0; j < J; ++j) { const int e = lane + 64 * j; f[j] = e < ne ? bl_f(g.counts[(size_t) s * ne + e], g, T) : 0.f; }
    for (int t = a + w; t < b; t += BL_W) {
        float z[J], q[J], om[J];
#pragma unroll
        for (int j = 0; j < J; ++j) { const int e = lane + 64 * j; z[j] = e < ne ? g.logits[(size_t) t * ne + e] : -INFINITY; }
        const float inv = bl_sigmoids<J>(z, q, om);
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) { d += f[j] * q[j]; }
        d = wave_sum(d) * inv;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = lane + 64 * j;
            if (e < ne) {
                float * o = g.dlogits + (size_t) t * ne + e;
                const float v = (k * (q[j] * inv)) * (om[j] * (f[j] - d));
                *o = g.accumulate ? *o + v : v;
            }
        }
    }
}

}  // namespace

int balance_chunks(int n, int nseq) {
    return std::max(1, std::min((int) (((int64_t) n + (int64_t) nseq * BL_ROWS - 1) / ((int64_t) nseq * BL_ROWS)), 256 / nseq));
}

hipError_t launch_balance(const BalanceArgs & a, hipStream_t st) {
    if (a.n < 0 || a.nseq < 1 || a.nseq > 65535 || a.n_exp < 1 || a.n_exp > NEXP_MAX || a.topk < 1 || a.chunks < 1 || (!a.seq && a.nseq != 1)) { return hipErrorInvalidValue; }
    const dim3 grid(a.chunks, a.nseq);
    switch ((a.n_exp + 63) / 64) {
    case 1: k_balance<1><<<grid, BL_T, 0, st>>>(a); break;
    case 2: k_balance<2><<<grid, BL_T, 0, st>>>(a); break;
    case 3: k_balance<3><<<grid, BL_T, 0, st>>>(a); break;
    default: k_balance<4><<<grid, BL_T, 0, st>>>(a); break;
    }
    if (const hipError_t e = hipGetLastError()) { return e; }
    if (a.chunks > 1) { k_balance_join<<<a.nseq, BL_T, 0, st>>>(a); }
    return hipGetLastError();
}

hipError_t launch_balance_grad(const BalanceArgs & a, hipStream_t st) {
    if (a.n < 0 || a.nseq < 1 || a.nseq >= 65535 || a.n_exp < 1 || a.n_exp > NEXP_MAX || a.topk < 1 || a.chunks < 1 || (!a.seq && a.nseq != 1)) { return hipErrorInvalidValue; }
    if (a.n == 0) { return hipSuccess; }
    const dim3 grid(a.chunks, a.nseq + (a.seq && !a.accumulate ? 1 : 0));
    switch ((a.n_exp + 63) / 64) {
    case 1: k_balance_grad<1><<<grid, BL_T, 0, st>>>(a); break;
    case 2: k_balance_grad<2><<<grid, BL_T, 0, st>>>(a); break;
    case 3: k_balance_grad<3><<<grid, BL_T, 0, st>>>(a); break;
    default: k_balance_grad<4><<<grid, BL_T, 0, st>>>(a); break;
    }
    return hipGetLastError();
}

}  // namespace lk
