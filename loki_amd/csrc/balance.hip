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
#include <type_traits>

namespace lk {

namespace {

#pragma clang fp contract(fast)   // (no bit contract here: fewer and larger steps)

constexpr int BL_B = 4, BL_W = 16;           // rows a wave takes at a time (their loads and reductions overlap), waves of the sums' workgroups
constexpr int BL_JOIN = 1024;                // threads of the joining workgroups
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
    const int per = (int) (((uint32_t) T + (uint32_t) g.chunks - 1) / (uint32_t) g.chunks);   // (T <= 2^24)
    a = min(lo + per * c, hi); b = min(a + per, hi);
}

// exp(x) for x <= 0: 2^h with h = x log2 e rounded, times what the rounding left out (v_exp_f32 and two products: 3 half steps
// of fp32; below 2^-126 the result is 0)
__device__ __forceinline__ float bl_exp(float x) {
    const float h = x * 0x1.715476p+0f, l = __builtin_fmaf(x, 0x1.715476p+0f, -h) + x * 0x1.4ae0cp-26f;
    const float p = __builtin_amdgcn_exp2f(h);
    return x < -126.f ? 0.f : __builtin_fmaf(p, l * 0x1.62e43p-1f, p);
}

// B rows' columns: lane l holds the columns e = l + 64 j of row t0 + i (rows from `end` on: the last row again, for the caller to
// leave out; columns past n_exp: -inf). The last columns' mask is opaque to the compiler, which would otherwise put each load
// behind a branch and wait for it there.
template <int J, int B> __device__ __forceinline__ void bl_load(const BalanceArgs & g, int t0, int end, float (&z)[B][J]) {
    const int lane = lane_id();
    uint32_t off = lane + 64 * (J - 1) < g.n_exp ? 0u : ~0u;
    __asm__ volatile("" : "+v"(off));
    const uint32_t last = (uint32_t) min(lane + 64 * (J - 1), g.n_exp - 1);
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const float * row = g.logits + (size_t) min(t0 + i, end - 1) * g.n_exp;
#pragma unroll
        for (int j = 0; j < J - 1; ++j) { z[i][j] = row[lane + 64 * j]; }
        z[i][J - 1] = row[last];
    }
#pragma unroll
    for (int i = 0; i < B; ++i) { z[i][J - 1] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, z[i][J - 1]) & ~off) | (0xff800000u & off)); }
}
// their sigmoids q (or the scaled stand-ins), om = 1 - sigmoid, and inv = 1 / sum q (0 where the row is all -inf)
template <int J, int B> __device__ __forceinline__ void bl_sigmoids(const float (&z)[B][J], float (&q)[B][J], float (&om)[B][J], float (&inv)[B]) {
    float sum[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        sum[i] = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float t = bl_exp(-fabsf(z[i][j])), r = __builtin_amdgcn_rcpf(1.f + t), tr = t * r;
            q[i][j] = z[i][j] >= 0.f ? r : tr;
            om[i][j] = z[i][j] >= 0.f ? tr : r;
            sum[i] += q[i][j];
        }
    }
#pragma unroll
    for (int i = 0; i < B; ++i) { sum[i] = wave_sum(sum[i]); }
#pragma unroll
    for (int i = 0; i < B; ++i) {
        inv[i] = __builtin_amdgcn_rcpf(sum[i]);
        if (sum[i] < BL_TINY) {
            float m = z[i][0];
#pragma unroll
            for (int j = 1; j < J; ++j) { m = fmaxf(m, z[i][j]); }
            m = wave_maxf(m);
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j) { q[i][j] = m == -INFINITY ? 0.f : bl_exp(z[i][j] - m); s += q[i][j]; }
            s = wave_sum(s);
            inv[i] = m == -INFINITY ? 0.f : __builtin_amdgcn_rcpf(s);
        }
    }
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
        for (int w = 0; w < NEXP_MAX / 64; ++w) { tot += scr[w]; }   // (the waves that hold experts)
        g.loss[s] = g.alpha * tot;
    }
}

// The sums: one read of the logits, P's parts in registers, counts by integer LDS atomics (exact in any order). 65536 rows of 256
// experts in 16 sequences, logits from memory: 21 us, 3.2 TB/s, and 4 for the join (17.8 together when the same call runs again and
// again, its logits then in the last-level cache). The vector units are busy 76 % of the cycles, and a wave has no load out while
// they are. Few rows: the launch (70 rows 5.5 us).
template <int J>
__global__ void __launch_bounds__(64 * BL_W) k_balance(BalanceArgs g) {
    constexpr int BL_T = 64 * BL_W;
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
    for (int t = a + __builtin_amdgcn_readfirstlane(w) * BL_B; t < b; t += BL_W * BL_B) {
        float z[BL_B][J], q[BL_B][J], om[BL_B][J], inv[BL_B];
        bl_load<J, BL_B>(g, t, b, z);
        bl_sigmoids<J, BL_B>(z, q, om, inv);
#pragma unroll
        for (int i = 0; i < BL_B; ++i) {
            if (t + i < b) {
#pragma unroll
                for (int j = 0; j < J; ++j) { acc[j] += q[i][j] * inv[i]; }
            }
        }
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

// chunks > 1: a sequence's sums over its chunks, four slices of them side by side and then in order, and its loss. A slice's loads
// are AHEAD chunks at once: one after the other they took 17 us for the 256 chunks of one sequence of 16384 rows, now 6.
__global__ void __launch_bounds__(BL_JOIN) k_balance_join(BalanceArgs g) {
    constexpr int AHEAD = 8;
    __shared__ float s_p[4][NEXP_MAX];
    __shared__ int s_c[4][NEXP_MAX];
    __shared__ float s_f[BL_JOIN / 64];
    const int s = blockIdx.x, e = threadIdx.x & 255, k = threadIdx.x >> 8;
    int a, b, T;
    bl_rows(g, s, 0, a, b, T);
    float psum = 0.f; int cnt = 0;
    if (e < g.n_exp) {
        for (int c0 = k; c0 < g.chunks; c0 += 4 * AHEAD) {
            float p[AHEAD]; int n[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {   // (past the last chunk: it again, left out below)
                const size_t o = ((size_t) s * g.chunks + min(c0 + 4 * i, g.chunks - 1)) * g.n_exp + e;
                p[i] = g.part[o]; n[i] = g.pcnt[o];
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const bool in = c0 + 4 * i < g.chunks;
                psum += in ? p[i] : 0.f; cnt += in ? n[i] : 0;
            }
        }
    }
    s_p[k][e] = psum; s_c[k][e] = cnt;
    __syncthreads();
    if (k == 0) {
        for (int i = 1; i < 4; ++i) { psum += s_p[i][e]; cnt += s_c[i][e]; }
    }
    bl_finish(g, s, T, k == 0 ? psum : 0.f, cnt, s_f);
}

// The gradient: a row's sigmoids once more (reading them back would cost what reading the logits costs, and the sums would have to
// write them), its weighted sum of f by the wave, one write. 65536 rows of 256 in 16 sequences, from memory: 29.5 us, 4.6 TB/s read and
// written (25 when the same call is repeated), vector units 76 % busy.
template <int J, int W>
__global__ void __launch_bounds__(64 * W) k_balance_grad(BalanceArgs g) {
    constexpr int BL_T = 64 * W;
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
    for (int t = a + __builtin_amdgcn_readfirstlane(w) * BL_B; t < b; t += W * BL_B) {
        float z[BL_B][J], q[BL_B][J], om[BL_B][J], inv[BL_B], d[BL_B];
        bl_load<J, BL_B>(g, t, b, z);
        bl_sigmoids<J, BL_B>(z, q, om, inv);
#pragma unroll
        for (int i = 0; i < BL_B; ++i) {
            d[i] = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j) { d[i] += f[j] * q[i][j]; }
        }
#pragma unroll
        for (int i = 0; i < BL_B; ++i) { d[i] = wave_sum(d[i]) * inv[i]; }
#pragma unroll
        for (int i = 0; i < BL_B; ++i) {
            if (t + i < b) {
                float * o = g.dlogits + (size_t) (t + i) * ne + lane;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (j < J - 1 || lane + 64 * j < ne) {
                        const float v = (k * (q[i][j] * inv[i])) * (om[i][j] * (f[j] - d[i]));
                        o[64 * j] = g.accumulate ? o[64 * j] + v : v;
                    }
                }
            }
        }
    }
}

}  // namespace

// Workgroups a sequence, each wave with a batch of BL_B rows at a time. Sums: 16 waves, so that there are few partial sums to join; up to
// 128 rows one workgroup, which needs no second launch (128 rows 6.9 us, and so 256 rows in 4 workgroups). The gradient has nothing to
// join: 4 waves up to 8192 rows (4100 rows 5.3 us, with 16 waves 6.3), 16 above (16384 rows 8.4 us, with 4 waves 10.9). (One sequence, the
// same call repeated.) The sequences' lengths are known on the device alone, so the cut is by their mean: one sequence with nine tenths
// of the rows is slow (8192 rows in 64 sequences: loss 8.8 -> 288 us, gradient 7.9 -> 88).
static int grad_waves(int n) { return n <= 8192 ? 4 : 16; }
static int chunks_of(int n, int nseq, bool grad) {
    const int w = grad ? grad_waves(n) : BL_W, rows = w * BL_B, most = w == 4 ? BALANCE_PARTS : BALANCE_PARTS / 2;
    if (!grad && n <= 128 * nseq) { return 1; }
    return std::max(1, std::min({ (int) (((int64_t) n + (int64_t) nseq * rows - 1) / ((int64_t) nseq * rows)), most / nseq, 256 }));
}
int balance_chunks(int n, int nseq) { return chunks_of(n, nseq, false); }

// go at the columns a lane holds
template <class F> static hipError_t by_columns(int n_exp, F && go) {
    switch ((n_exp + 63) / 64) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 2: go(std::integral_constant<int, 2>{}); break;
    case 3: go(std::integral_constant<int, 3>{}); break;
    default: go(std::integral_constant<int, 4>{}); break;
    }
    return hipGetLastError();
}

hipError_t launch_balance(const BalanceArgs & a, hipStream_t st) {
    if (a.n < 0 || a.nseq < 1 || a.nseq > 65535 || a.n_exp < 1 || a.n_exp > NEXP_MAX || a.topk < 1 || a.chunks < 1 || (!a.seq && a.nseq != 1)) { return hipErrorInvalidValue; }
    const hipError_t e = by_columns(a.n_exp, [&](auto j) { k_balance<decltype(j)::value><<<dim3(a.chunks, a.nseq), 64 * BL_W, 0, st>>>(a); });
    if (e != hipSuccess || a.chunks == 1) { return e; }
    k_balance_join<<<a.nseq, BL_JOIN, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_balance_grad(const BalanceArgs & args, hipStream_t st) {
    BalanceArgs a = args;
    a.chunks = chunks_of(a.n, std::max(1, a.nseq), true);
    if (a.n < 0 || a.nseq < 1 || a.nseq >= 65535 || a.n_exp < 1 || a.n_exp > NEXP_MAX || a.topk < 1 || a.chunks < 1 || (!a.seq && a.nseq != 1)) { return hipErrorInvalidValue; }
    if (a.n == 0) { return hipSuccess; }
    const dim3 grid(a.chunks, a.nseq + (a.seq && !a.accumulate ? 1 : 0));
    if (grad_waves(a.n) == 4) { return by_columns(a.n_exp, [&](auto j) { k_balance_grad<decltype(j)::value, 4><<<grid, 64 * 4, 0, st>>>(a); }); }
    return by_columns(a.n_exp, [&](auto j) { k_balance_grad<decltype(j)::value, 16><<<grid, 64 * 16, 0, st>>>(a); });
}

}  // namespace lk
