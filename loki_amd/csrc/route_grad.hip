// route_grad.hip -- the router's backward pass: from the gradients of the routing weights (and of the logits themselves) to
// the logits, the router weight and the rows.
//
// z = x W^T, s = sigmoid(z), S = sum_j s_j over the row's picks, w_k = scale s_k / max(S, 2^-14) (router.hip), so
//   S > 2^-14:  ds_k = scale / S (dw_k - sum_j dw_j s_j / S),  else  ds_k = scale / 2^-14 dw_k
//   dz = dz_in + sum over the picks of ds_k s_k (1 - s_k),   dW = dz^T x,   dx = dz W
// The bias only takes part in the selection and has no gradient.
//
// The two products run on the fp16 matrix cores at fp32's precision: an operand v is taken as v 2^k = hi + lo, two fp16 of 11 bits
// each, and a product is hi hi + hi lo + lo hi in fp32 sums; what is left out, lo lo, and each half's own rounding are below 2^-22 of
// the product. Three fp16 products cost a third of what the fp32 matrix cores take. k puts the largest finite |v| of those that share
// it at 2^14 .. 2^15, so that values down to 2^-18 of it keep both halves whole and smaller ones an absolute error of 2^-39 of it:
//   dx   dz: one k per row t (dx's row t is scaled back by 2^-k_t). W: one k per 64 columns, found by the kernel that splits it
//   dW   dz: one k per expert. What a row's picks get is a million times and more what the balance loss gives the other experts, and
//        an expert that is picked in few rows or none gets nothing else: on the row's scale its whole row of dW would be lost. It
//        comes in two steps, since nobody knows an expert's maximum when dz is split: the halves are made with a k per expert and 8
//        rows (the maximum at 2^2 .. 2^3: below it an absolute error of 2^-27 of these 8 rows' maximum), and a lane brings its operands
//        to the smallest k of its run's rows by one fp16 factor of 2^12 .. 2^-24 (rows below 2^-36 of the expert's largest become 0).
//        x: one k per column, running: a slab's maximum that passes the present range lowers k, and the accumulators of that column
//        follow (as the running maximum of an online softmax). Rows without any gradient have no part in it: what padding holds
//        there must not cost the others their bits.
// Non-finite values take no part in the maxima of dz and W; they make the outputs that they enter non-finite.
#include "moe_device.h"
#include "moe_kernels.h"

#include <algorithm>

namespace lk {

namespace {

constexpr float RG_CLAMP = 0x1p-14f;   // select_token_p's
constexpr int RG_NONE = 1000;          // k of a row without gradient: dx's is 0
constexpr int RG_ZK = 113, RG_ZNONE = 142, RG_ZUP = 12;   // dW's dz: k + RG_ZK is a byte; k of 8 rows without gradient; halves are made with k - RG_ZUP
typedef float gf4 __attribute__((ext_vector_type(4)));
typedef _Float16 gh8 __attribute__((ext_vector_type(8)));

// the k that puts m > 0 at 2^14 .. 2^15 (m finite; subnormals as the smallest normal number), at most MOST
template <int MOST = 126> __device__ __forceinline__ int rg_k(float m) { return min(MOST, 141 - max(1, (int) (__builtin_bit_cast(uint32_t, m) >> 23))); }
__device__ __forceinline__ float rg_pow2(int k) { return __builtin_bit_cast(float, (uint32_t) (min(max(k, -126), 127) + 127) << 23); }
__device__ __forceinline__ float rg_mag(float v) { const float a = fabsf(v); return a < INFINITY ? a : 0.f; }
__device__ __forceinline__ void rg_split(float v, _Float16 & hi, _Float16 & lo) { hi = (_Float16) v; lo = (_Float16) (v - (float) hi); }
template <int CTRL> __device__ __forceinline__ float rg_dpp(float v) { return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v))); }
__device__ __forceinline__ float rg_lane(float v, int l) { return __builtin_bit_cast(float, rdlane(__builtin_bit_cast(uint32_t, v), l)); }
__device__ __forceinline__ float rg_wave_max(float v) {
    v = fmaxf(v, rg_dpp<DPP_XOR1>(v)); v = fmaxf(v, rg_dpp<DPP_XOR2>(v)); v = fmaxf(v, rg_dpp<DPP_HALF_MIRROR>(v)); v = fmaxf(v, rg_dpp<DPP_MIRROR>(v));
    return fmaxf(fmaxf(rg_lane(v, 0), rg_lane(v, 16)), fmaxf(rg_lane(v, 32), rg_lane(v, 48)));
}
// the largest of the four lanes that share lane % 16
__device__ __forceinline__ float rg_max_rows(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t a = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    const uint32_t b = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, (uint32_t) p[0]), __builtin_bit_cast(float, (uint32_t) p[1])));
    const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t) q[0]), __builtin_bit_cast(float, (uint32_t) q[1]));
#else
    return v;
#endif
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rg_rsrc(const void * p, uint32_t bytes) {
    const uint64_t v = (uint64_t) p;
    const uint32_t hi = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) (v >> 32)), lo = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) v);
    return __builtin_amdgcn_make_buffer_rsrc((void *) (((uint64_t) hi << 32) | lo), (short) 0, __builtin_amdgcn_readfirstlane((int) bytes), 0x00020000);
}
// 16 bytes per lane from a buffer straight into LDS, lane L at dst + 16 L; the builtin exists for the device pass only
__device__ __forceinline__ void rg_lds16(__amdgpu_buffer_rsrc_t r, LK_LOCAL uint8_t * dst, uint32_t voff, uint32_t soff) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LK_LOCAL void *) dst, 16, voff, soff, 0, 0);
#else
    (void) r; (void) dst; (void) voff; (void) soff;
#endif
}

// The operands in memory, halves of 16 bytes = 8 consecutive K values:
//   zs [t / 16][K / 32][hi, lo][K / 8 % 4][t % 16][8]   dz, K = experts (n_exp up to a multiple of 32, zeros): the order of a wave's lanes
//   kt [t]                      the rows' k (zs)
//   zt [t / 8][hi, lo][ea][8]   dz of 8 rows, K = rows (ea: n_exp up to 64, 128 or 256, zeros; rows up to a multiple of 32, zeros)
//   zk [t / 8][ea / 64][16]     x: the k of experts r, r + 16, r + 32, r + 48 of the 64, bytes; y: bit i: row i of the 8 has a gradient
//   wt [hi, lo][kp / 8][E][8]   W, K = experts; kw [E / 64] its k
struct Ops { _Float16 * zs, * zt, * wt; short * kt; uint2 * zk; int * kw; int kp, ea, np; };

// The first nw workgroups split 64 columns of W each (all experts in registers between the maximum and the split). The others take 8
// rows, two a wave: lane k < topk holds pick k, then the columns e = lane + 64 j of the row.
__global__ void __launch_bounds__(256) k_route_prep(RouteGradArgs g, Ops o, int nw) {
    __shared__ _Float16 s_h[2][8][NEXP_MAX];
    __shared__ float s_v[8][NEXP_MAX], s_m[4];
    __shared__ uint8_t s_k[NEXP_MAX], s_on[8];
    const int lane = lane_id(), wv = threadIdx.x >> 6, ne = g.n_exp;
    if ((int) blockIdx.x < nw) {
        constexpr int NB = NEXP_MAX / 32;   // experts 8 (wv + 4 i) .. + 7 a wave
        const int c = (int) blockIdx.x * 64 + lane;
        float v[NB][8], m = 0.f;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int u = 0; u < 8; ++u) { const int e = 8 * (wv + 4 * i) + u; v[i][u] = g.W[(size_t) min(e, ne - 1) * g.E + c]; }   // (all loads out before the first use)
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int u = 0; u < 8; ++u) { v[i][u] = 8 * (wv + 4 * i) + u < ne ? v[i][u] : 0.f; }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int u = 0; u < 8; ++u) { m = fmaxf(m, rg_mag(v[i][u])); }
        }
        m = rg_wave_max(m);
        if (lane == 0) { s_m[wv] = m; }
        __syncthreads();
        const int k = rg_k(fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])));
        const float sc = rg_pow2(k);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int b = wv + 4 * i;
            if (b < o.kp / 8) {
                gh8 hi, lo;
#pragma unroll
                for (int u = 0; u < 8; ++u) { _Float16 h, l; rg_split(v[i][u] * sc, h, l); hi[u] = h; lo[u] = l; }
                *reinterpret_cast<gh8 *>(o.wt + ((size_t) b * g.E + c) * 8) = hi;
                *reinterpret_cast<gh8 *>(o.wt + ((size_t) (o.kp / 8 + b) * g.E + c) * 8) = lo;
            }
        }
        if (threadIdx.x == 0) { o.kw[blockIdx.x] = k; }
        return;
    }
    const int tb = (int) blockIdx.x - nw, t0 = tb * 8;
    constexpr int J = NEXP_MAX / 64;
    float v[2][J], s[2], om[2], dw[2];
    int e[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int t = t0 + wv + 4 * h;
        const bool in = t < g.n, pick = in && g.dw && lane < g.topk;
#pragma unroll
        for (int j = 0; j < J; ++j) { const int c = lane + 64 * j; v[h][j] = in && g.dz_in && c < ne ? g.dz_in[(size_t) t * ne + c] : 0.f; }
        e[h] = pick ? g.sel[(size_t) t * g.topk + lane] : -1;
        dw[h] = pick ? g.dw[(size_t) t * g.topk + lane] : 0.f;
        if ((unsigned) e[h] >= (unsigned) ne) { e[h] = -1; dw[h] = 0.f; }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float z = e[h] >= 0 ? g.logits[(size_t) (t0 + wv + 4 * h) * ne + e[h]] : -INFINITY;
        const float u = expf(-fabsf(z)), r = 1.f / (1.f + u);
        s[h] = z >= 0.f ? r : u * r; om[h] = z >= 0.f ? u * r : r;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int t = t0 + wv + 4 * h;
        float S = 0.f, D = 0.f;
#pragma unroll
        for (int k = 0; k < MAXK; ++k) { const float sk = rg_lane(s[h], k); S += sk; D += rg_lane(dw[h], k) * sk; }   // in pick order, as the forward pass adds; none: 0
        const float ds = S > RG_CLAMP ? g.scale / S * (dw[h] - D / S) : g.scale / RG_CLAMP * dw[h], gz = ds * (s[h] * om[h]);
#pragma unroll
        for (int k = 0; k < MAXK; ++k) {
            const int ek = (int) rdlane((uint32_t) e[h], k);
            const float gk = rg_lane(gz, k);
#pragma unroll
            for (int j = 0; j < J; ++j) { v[h][j] += ek == lane + 64 * j ? gk : 0.f; }
        }
        float m = 0.f;
        bool odd = false;
#pragma unroll
        for (int j = 0; j < J; ++j) { m = fmaxf(m, rg_mag(v[h][j])); odd = odd || !(fabsf(v[h][j]) < INFINITY); }
        m = rg_wave_max(m);
        const bool none = m == 0.f && __ballot(odd) == 0;
        const int k = none ? RG_NONE : rg_k(m);
        const float sc = none ? 1.f : rg_pow2(k);
        if (lane == 0) { s_on[wv + 4 * h] = none ? 0 : 1; if (g.dx) { o.kt[t] = (short) k; } }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int c = lane + 64 * j;
            if (t < g.n && c < ne && g.dz) { g.dz[(size_t) t * ne + c] = v[h][j]; }
            _Float16 a, l;
            rg_split(v[h][j] * sc, a, l);
            s_h[0][wv + 4 * h][c] = a; s_h[1][wv + 4 * h][c] = l;
            s_v[wv + 4 * h][c] = v[h][j];
        }
    }
    __syncthreads();
    if (g.dW) {   // 8 rows of expert threadIdx.x
        const int c = (int) threadIdx.x;
        if (c < o.ea) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) { m = fmaxf(m, rg_mag(s_v[i][c])); }
            const int k = m > 0.f ? rg_k<RG_ZNONE - 2>(m) : RG_ZNONE;
            gh8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; ++i) { _Float16 h, l; rg_split(ldexpf(s_v[i][c], k - RG_ZUP), h, l); hi[i] = h; lo[i] = l; }
            *reinterpret_cast<gh8 *>(o.zt + ((size_t) tb * 2 * o.ea + c) * 8) = hi;
            *reinterpret_cast<gh8 *>(o.zt + (((size_t) tb * 2 + 1) * o.ea + c) * 8) = lo;
            s_k[c] = (uint8_t) (k + RG_ZK);
        }
        __syncthreads();
        if (c < o.ea / 4) {
            uint2 w = { 0u, 0u };
#pragma unroll
            for (int i = 0; i < 4; ++i) { w.x |= (uint32_t) s_k[64 * (c >> 4) + 16 * i + (c & 15)] << (8 * i); }
#pragma unroll
            for (int i = 0; i < 8; ++i) { w.y |= (uint32_t) s_on[i] << i; }
            o.zk[(size_t) tb * (o.ea / 4) + c] = w;
        }
    }
    const int nc = o.kp / 8;
    for (int p = threadIdx.x; p < (g.dx ? 16 * nc : 0); p += 256) {    // 8 experts of a row
        const int i = p % 8, c = p / 8;
        const int h = c / nc, b = c % nc, t = t0 + i;
        *reinterpret_cast<gh8 *>(o.zs + ((((size_t) (t >> 4) * (nc / 4) + b / 4) * 2 + h) * 64 + (b % 4) * 16 + (t & 15)) * 8) = *reinterpret_cast<const gh8 *>(&s_h[h][i][8 * b]);
    }
}

constexpr int RG_W = 8, RG_T = 64 * RG_W, RG_COLS = ROUTE_COLS, RG_RT = 2;
static_assert(16 * RG_RT * RG_W == ROUTE_ROWS, "rows that a workgroup of dx takes at a time");

// dx: a workgroup keeps 128 columns of W, all experts, both halves, in LDS (at most 128 KB) and its waves take 32 rows at a time,
// whose dz comes straight from the caches, D - 1 steps of 32 experts ahead and into the wave's next tile; no barrier after the first.
// The product runs with the columns as rows of the matrix core's tile, so a lane stores 4 consecutive columns. dz's layout has each
// load's 64 lanes side by side: rows apart, with 64 bytes each, cost 8192 rows of 7168, 256 experts, 12 of their 112 us. 64 rows a
// wave need half the LDS reads but leave waves idle (both products, 1001 rows: 57 us instead of 48; 8192 rows: 203 instead of 205).
template <int D>
__device__ __forceinline__ void route_dx(const RouteGradArgs & g, const Ops & o, LK_LOCAL uint8_t * lds, int ct, int part, int parts) {
    constexpr int RT = RG_RT, AH = 1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), r = lane & 15, q = lane >> 4;
    const int j0 = ct * RG_COLS, nb = o.kp / 8, ns = o.kp / 32;
    const __amdgpu_buffer_rsrc_t rw = rg_rsrc(o.wt, (uint32_t) ((size_t) 2 * nb * g.E * 16));
    for (int i = wave; i < 2 * nb * 2; i += RG_W) {   // half and 8 experts i / 2, columns 64 (i % 2) ..
        rg_lds16(rw, lds + i * 1024, (uint32_t) (lane * 16), (uint32_t) ((size_t) (i >> 1) * g.E * 16 + (size_t) (j0 + 64 * (i & 1)) * 16));
    }
    const int kw[2] = { o.kw[j0 / 64], o.kw[j0 / 64 + 1] };
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __syncthreads();
    const uint32_t lo_off = (uint32_t) nb * 2048, lb = (uint32_t) (size_t) lds + (uint32_t) (q * 2048 + r * 16);
    const int tiles = (g.n + 16 * RT - 1) / (16 * RT), stride = parts * RG_W, tt0 = part * RG_W + wave, nsp = (ns + D - 1) / D * D;
    if (tt0 >= tiles) { return; }
    uint32_t vz[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) { vz[i] = (uint32_t) (i * ns * 2048 + lane * 16); }
    // the loads' place, D - 1 steps ahead of the products' and into the next tile (after the last one: it again, unread)
    auto rsrc = [&](int tt) { return rg_rsrc(o.zs + (size_t) tt * RT * ns * 1024, (uint32_t) (RT * ns * 2048)); };
    int lt = tt0, ls = 0;
    __amdgpu_buffer_rsrc_t rz = rsrc(lt);
    gh8 z[D][RT][2];
    auto load = [&](gh8 (&d)[RT][2]) {
        const uint32_t so = (uint32_t) (min(ls, ns - 1) * 2048);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            d[i][0] = __builtin_bit_cast(gh8, __builtin_amdgcn_raw_buffer_load_b128(rz, vz[i], so, 0));
            d[i][1] = __builtin_bit_cast(gh8, __builtin_amdgcn_raw_buffer_load_b128(rz, vz[i] + 1024u, so, 0));
        }
        if (++ls == nsp) { ls = 0; lt = lt + stride < tiles ? lt + stride : lt; rz = rsrc(lt); }
    };
#pragma unroll
    for (int k = 0; k < D - 1; ++k) { load(z[k]); }
    for (int tt = tt0; tt < tiles; tt += stride) {
        const int t0 = tt * 16 * RT;
        gf4 acc[8][RT];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
#pragma unroll
            for (int i = 0; i < RT; ++i) { acc[c][i] = (gf4) { 0.f, 0.f, 0.f, 0.f }; }
        }
        auto step = [&](int s, const gh8 (&d)[RT][2]) {
            const uint32_t a = lb + (uint32_t) s * 8192;   // 4 x 8 experts
            __builtin_amdgcn_sched_barrier(0);
            gh8 w[AH + 1][2];   // W's operands, AH column tiles ahead
            auto ld = [&](int c) { w[c % (AH + 1)][0] = *(const LK_LOCAL gh8 *) (size_t) (a + c * 256); w[c % (AH + 1)][1] = *(const LK_LOCAL gh8 *) (size_t) (a + lo_off + c * 256); };
#pragma unroll
            for (int c = 0; c < AH; ++c) { ld(c); }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (c + AH < 8) { ld(c + AH); }
                __builtin_amdgcn_sched_barrier(0);
                const gh8 wh = w[c % (AH + 1)][0], wl = w[c % (AH + 1)][1];
#pragma unroll
                for (int i = 0; i < RT; ++i) { acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, d[i][0], acc[c][i], 0, 0, 0); }
#pragma unroll
                for (int i = 0; i < RT; ++i) { acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, d[i][1], acc[c][i], 0, 0, 0); }
#pragma unroll
                for (int i = 0; i < RT; ++i) { acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl, d[i][0], acc[c][i], 0, 0, 0); }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        for (int s = 0; s < nsp; s += D) {
#pragma unroll
            for (int k = 0; k < D; ++k) {
                load(z[(k + D - 1) % D]);
                if (s + k < ns) { step(s + k, z[k]); }
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int t = t0 + 16 * i + r;
            if (t < g.n) {
                const int kt = (int) o.kt[t];
                float * row = g.dx + (size_t) t * g.E + j0 + 4 * q;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int k = kt == RG_NONE ? 0 : -kt - kw[c >> 2];
                    gf4 v;
#pragma unroll
                    for (int u = 0; u < 4; ++u) { v[u] = ldexpf(acc[c][i][u], k); }
                    __builtin_nontemporal_store(v, reinterpret_cast<gf4 *>(row + 16 * c));
                }
            }
        }
    }
}

// dW: a workgroup takes 128 columns of x, all experts (64 WR) and a run of 32-row steps. dz of a step is copied into LDS as it is
// stored; x is read once, each wave 16 columns x 32 rows of it into registers (8 consecutive rows a lane), scaled, split and
// written to LDS as 16-byte halves. Both are double-buffered: a step's barrier, the next step's copies and conversion, its products.
// Waves: WR along the experts (64 each), 8 / WR along the columns (16 WR each). x's conversion is spread between the products, one in
// three instructions, and dz's operands are read one row tile ahead. 8192 rows of 7168, 256 experts: both products 204 us at least in a
// kernel trace, the matrix cores busy 45 % of the cycles, other vector instructions 22 %, waves waiting for their turn to issue 44 %.
template <int WR>
__device__ __forceinline__ void route_dw(const RouteGradArgs & g, const Ops & o, LK_LOCAL uint8_t * lds, int ct, int run, int splits, float * part) {
    constexpr int EA = 64 * WR, AB = 4 * 2 * EA * 16, BB = 4 * 2 * RG_COLS * 16, BUF = AB + BB + RG_COLS * 4, JW = WR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), r = lane & 15, q = lane >> 4;
    const int j0 = ct * RG_COLS, we = wave % WR, wj = wave / WR;
    const int steps = o.np / 32, s0 = (int) ((int64_t) steps * run / splits), s1 = (int) ((int64_t) steps * (run + 1) / splits);
    struct Slab { float x[8]; uint2 k; };
    auto load_x = [&](int s, Slab & d) {   // rows 32 s + 8 q .. + 7, column j0 + 16 wave + r; rows past the batch's end read 0. Their dz's k
        const int t = 32 * min(s, s1 - 1), nt = min(32, g.n - t);
        const __amdgpu_buffer_rsrc_t rx = rg_rsrc(g.x + (size_t) t * g.E, (uint32_t) nt * (uint32_t) g.E * 4);
        const uint32_t v = ((uint32_t) (8 * q) * (uint32_t) g.E + (uint32_t) (j0 + 16 * wave + r)) * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) { d.x[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rx, v + (uint32_t) i * (uint32_t) g.E * 4, 0, 0)); }
        d.k = o.zk[(size_t) (t / 8 + q) * (EA / 4) + 16 * we + r];
    };
    auto copy_z = [&](int s, int b) {   // 4 x 8 rows' halves, as they are stored
        const int st = min(s, s1 - 1);
        const __amdgpu_buffer_rsrc_t rz = rg_rsrc(o.zt + (size_t) st * 4 * 2 * EA * 8, (uint32_t) AB);
#pragma unroll
        for (int i = 0; i < AB / 1024 / RG_W; ++i) { rg_lds16(rz, lds + b * BUF + (wave + i * RG_W) * 1024, (uint32_t) (lane * 16), (uint32_t) ((wave + i * RG_W) * 1024)); }
    };
    int kc = 200;   // the wave's columns' k (column r, the same in the four lane groups)
    uint32_t zk = 0;   // the k of the converted rows' dz
    int kr[4];         // the smallest k of experts 64 we + 16 i + r in the run's rows, + RG_ZK + RG_ZUP
    auto convert = [&](const Slab & sl, int b) {
        float y[8], m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { y[i] = sl.x[i] * (float) ((sl.k.y >> i) & 1u); m = fmaxf(m, fabsf(y[i])); }
        zk = sl.k.x;
        m = rg_max_rows(m);
        kc = min(kc, m > 0.f ? rg_k(m) : kc);   // (a column with an infinity is non-finite in every expert, whatever its k)
        const float sc = rg_pow2(kc);
        gh8 hi, lo;
#pragma unroll
        for (int i = 0; i < 8; ++i) { _Float16 h, l; rg_split(y[i] * sc, h, l); hi[i] = h; lo[i] = l; }
        LK_LOCAL uint8_t * d = lds + b * BUF + AB + (q * 2 * RG_COLS + 16 * wave + r) * 16;
        *(LK_LOCAL gh8 *) d = hi; *(LK_LOCAL gh8 *) (d + RG_COLS * 16) = lo;
        *(LK_LOCAL int *) (lds + b * BUF + AB + BB + (16 * wave + r) * 4) = kc;   // (the same from the four lane groups)
    };
    gf4 acc[4][JW];
    int cur[JW];
#pragma unroll
    for (int c = 0; c < JW; ++c) {
        cur[c] = 200;
#pragma unroll
        for (int i = 0; i < 4; ++i) { acc[i][c] = (gf4) { 0.f, 0.f, 0.f, 0.f }; }
    }
    Slab sl[3];   // three steps of x ahead: a step is about 0.6 us, memory answers in 1 to 2
    constexpr int LX = 9;   // loads of a slab
    auto step = [&](int s, Slab & next) {   // next: step s + 1's slab
            const int b = (s - s0) & 1;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0f70 | LX);   // all but the last slab's loads: this wave's copies of step s have landed
            __syncthreads();                           // and everyone's, with x's halves; the other buffer is free
            copy_z(s + 1, b ^ 1);
            __builtin_amdgcn_sched_barrier(0);
            const uint32_t lb = (uint32_t) (size_t) lds + (uint32_t) (b * BUF);
            int kn[JW];
            gh8 xh[JW], xl[JW], z[2][2];
            auto load_z = [&](int i) {
                const uint32_t a = lb + (uint32_t) ((q * 2 * EA + 64 * we + 16 * i + r) * 16);
                z[i & 1][0] = *(const LK_LOCAL gh8 *) (size_t) a; z[i & 1][1] = *(const LK_LOCAL gh8 *) (size_t) (a + EA * 16);
            };
#pragma unroll
            for (int c = 0; c < JW; ++c) { kn[c] = *(const LK_LOCAL int *) (size_t) (lb + AB + BB + (uint32_t) ((16 * JW * wj + 16 * c + r) * 4)); }
            load_z(0);
            _Float16 fz[4];   // of experts 64 we + 16 i + r, rows 8 q .. + 7: to the run's k (a row group far below it: 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) { fz[i] = (_Float16) ldexpf(1.f, kr[i] - (int) ((zk >> (8 * i)) & 255u)); }
#pragma unroll
            for (int c = 0; c < JW; ++c) {
                const uint32_t a = lb + AB + (uint32_t) ((q * 2 * RG_COLS + 16 * JW * wj + 16 * c + r) * 16);
                xh[c] = *(const LK_LOCAL gh8 *) (size_t) a; xl[c] = *(const LK_LOCAL gh8 *) (size_t) (a + RG_COLS * 16);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < JW; ++c) {   // columns whose k went down: what is summed so far follows
                if (__ballot(kn[c] != cur[c])) {
                    const float f = rg_pow2(kn[c] - cur[c]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) { acc[i][c] = acc[i][c] * f; }
                    cur[c] = kn[c];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i < 3) { load_z(i + 1); }
                const gh8 zh = z[i & 1][0] * fz[i], zl = z[i & 1][1] * fz[i];
#pragma unroll
                for (int c = 0; c < JW; ++c) { acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(zh, xh[c], acc[i][c], 0, 0, 0); }
#pragma unroll
                for (int c = 0; c < JW; ++c) { acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(zh, xl[c], acc[i][c], 0, 0, 0); }
#pragma unroll
                for (int c = 0; c < JW; ++c) { acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(zl, xh[c], acc[i][c], 0, 0, 0); }
            }
            convert(next, b ^ 1);
            load_x(s + 4, next);
#pragma unroll
            for (int i = 0; i < 12 * JW; ++i) {
                if (i % (3 * JW) == 0 && i < 9 * JW) { __builtin_amdgcn_sched_group_barrier(0x100, 2, 0); }
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
    };
    load_x(s0, sl[0]);
    copy_z(s0, 0);
    // kr: the waves that share the experts take the groups of 8 rows in turn, 8 loads at once; their minima meet in the second buffer,
    // which is free until the first step's barrier
    {
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 lo = { 255, 255 }, hi = lo;   // experts i = 0, 2 and 1, 3
        auto low = [&](uint32_t w) {
            lo = __builtin_elementwise_min(lo, __builtin_bit_cast(us2, w & 0x00FF00FFu));
            hi = __builtin_elementwise_min(hi, __builtin_bit_cast(us2, (w >> 8) & 0x00FF00FFu));
        };
        constexpr int G = 4 * RG_W / WR, AHEAD = 8;
        for (int t = 4 * s0 + 4 * wj + q; t < 4 * s1; t += G * AHEAD) {
            uint32_t w[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) { w[i] = o.zk[(size_t) min(t + G * i, 4 * s1 - 1) * (EA / 4) + 16 * we + r].x; }   // (past the run's end: its last again)
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) { low(w[i]); }
        }
        auto word = [&]() { return __builtin_bit_cast(uint32_t, lo) | (__builtin_bit_cast(uint32_t, hi) << 8); };
        low((uint32_t) __shfl_xor((int) word(), 16)); low((uint32_t) __shfl_xor((int) word(), 32));
        if (q == 0) { *(LK_LOCAL uint32_t *) (lds + BUF + 64 * wave + 4 * r) = word(); }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RG_W / WR; ++i) { low(*(const LK_LOCAL uint32_t *) (lds + BUF + 64 * (we + WR * i) + 4 * r)); }
        kr[0] = lo.x + RG_ZUP; kr[1] = hi.x + RG_ZUP; kr[2] = lo.y + RG_ZUP; kr[3] = hi.y + RG_ZUP;
    }
    convert(sl[0], 0);
    load_x(s0 + 1, sl[0]); load_x(s0 + 2, sl[1]); load_x(s0 + 3, sl[2]);
    for (int s = s0;;) {   // (past the run's end: its last rows again, unread)
        step(s, sl[0]);
        if (++s == s1) { break; }
        step(s, sl[1]);
        if (++s == s1) { break; }
        step(s, sl[2]);
        if (++s == s1) { break; }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);   // no copy into LDS outlives the workgroup
    float * out = splits > 1 ? part + (size_t) run * g.n_exp * g.E : g.dW;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = 64 * we + 16 * i + 4 * q + u, ke = __shfl(kr[i], 4 * q + u) - RG_ZUP - RG_ZK;
#pragma unroll
            for (int c = 0; c < JW; ++c) {
                const int k = cur[c] == 200 ? 0 : -cur[c] - ke;   // (200: nothing but zeros in the column)
                if (e < g.n_exp) {
                    float * d = out + (size_t) e * g.E + j0 + 16 * JW * wj + 16 * c + r;
                    const float v = ldexpf(acc[i][c][u], k);
                    *d = splits == 1 && g.accumulate ? *d + v : v;
                }
            }
        }
    }
}
// both products in one launch: the first E / 128 x splits workgroups dW, the others dx (E / 128 x parts)
template <int WR>
__global__ void __launch_bounds__(RG_T, 2) k_route_mm(RouteGradArgs g, Ops o, int splits, int parts, float * part) {
    extern __shared__ __attribute__((aligned(16))) uint8_t rg_dyn[];
    const int ct = g.E / RG_COLS, b = (int) blockIdx.x, dw = g.dW ? ct * splits : 0;
    if (b < dw) { route_dw<WR>(g, o, (LK_LOCAL uint8_t *) rg_dyn, b % ct, b / ct, splits, part); }
    else { route_dx<WR == 1 ? 2 : 4>(g, o, (LK_LOCAL uint8_t *) rg_dyn, (b - dw) % ct, (b - dw) / ct, parts); }
}
// the runs' sums, in order
__global__ void __launch_bounds__(256) k_route_join(const float * __restrict__ part, int splits, int64_t n4, int accumulate, float * __restrict__ dW) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) { return; }
    gf4 v = reinterpret_cast<const gf4 *>(part)[i];
    for (int s = 1; s < splits; ++s) { v = v + reinterpret_cast<const gf4 *>(part)[(int64_t) s * n4 + i]; }
    gf4 * d = reinterpret_cast<gf4 *>(dW) + i;
    *d = accumulate ? *d + v : v;
}

constexpr size_t up256(size_t v) { return (v + 255) / 256 * 256; }
struct Sizes { int kp, ea, np; size_t zs, zt, kt, zk, wt, kw, part, all; };
Sizes rg_sizes(int n, int ne, int E, bool dW, bool dx) {
    Sizes z{};
    z.kp = (ne + 31) / 32 * 32; z.ea = ne <= 64 ? 64 : ne <= 128 ? 128 : 256; z.np = (n + 31) / 32 * 32;
    z.zs = dx ? up256((size_t) z.np * 2 * z.kp * 2) : 0; z.zt = dW ? up256((size_t) z.np * 2 * z.ea * 2) : 0; z.kt = dx ? up256((size_t) z.np * 2) : 0;
    z.zk = dW ? up256((size_t) z.np / 8 * (z.ea / 4) * 8) : 0;
    z.wt = dx ? up256((size_t) 2 * z.kp * E * 2) : 0; z.kw = dx ? up256((size_t) (E / 64) * 4) : 0;
    const int sp = route_cut(n, E, dW, dx).splits;
    z.part = dW && sp > 1 ? (size_t) sp * ne * E * 4 : 0;
    z.all = std::max<size_t>(256, z.zs + z.zt + z.kt + z.zk + z.wt + z.kw + z.part);   // (256: a call for dlogits alone takes none of it)
    return z;
}
template <int WR> hipError_t go(const RouteGradArgs & a, const Ops & o, RouteCut cut, float * part, hipStream_t st) {
    constexpr int DW = 2 * (4 * 2 * 64 * WR * 16 + 4 * 2 * RG_COLS * 16 + RG_COLS * 4), DX = 2 * 64 * WR * RG_COLS * 2;
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_route_mm<WR>, std::max(DW, DX))) { return e; }
    const int ct = a.E / RG_COLS;
    k_route_mm<WR><<<(unsigned) (ct * ((a.dW ? cut.splits : 0) + (a.dx ? cut.parts : 0))), RG_T, std::max(a.dW ? DW : 0, a.dx ? 2 * o.kp * RG_COLS * 2 : 0), st>>>(a, o, cut.splits, cut.parts, part);
    return hipGetLastError();
}

}  // namespace

size_t route_grad_scratch(int n, int n_exp, int E, bool dW, bool dx) { return n > 0 ? rg_sizes(n, n_exp, E, dW, dx).all : 0; }

hipError_t launch_route_grad(const RouteGradArgs & a, void * scratch, hipStream_t st) {
    if (a.n < 0 || a.n_exp < 1 || a.n_exp > NEXP_MAX || a.E <= 0 || a.E % 1024 || a.topk < 1 || a.topk > MAXK || (a.n > 0 && !scratch)) { return hipErrorInvalidValue; }
    if (a.n == 0) { return hipSuccess; }
    const Sizes z = rg_sizes(a.n, a.n_exp, a.E, a.dW != nullptr, a.dx != nullptr);
    Ops o{};
    uint8_t * p = (uint8_t *) scratch;
    o.kp = z.kp; o.ea = z.ea; o.np = z.np;
    o.zs = (_Float16 *) p; p += z.zs; o.zt = (_Float16 *) p; p += z.zt; o.kt = (short *) p; p += z.kt; o.zk = (uint2 *) p; p += z.zk; o.wt = (_Float16 *) p; p += z.wt; o.kw = (int *) p; p += z.kw;
    float * part = (float *) p;
    const RouteCut cut = route_cut(a.n, a.E, a.dW != nullptr, a.dx != nullptr);
    const int nw = a.dx ? a.E / 64 : 0, sp = cut.splits;
    k_route_prep<<<nw + z.np / 8, 256, 0, st>>>(a, o, nw);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && (a.dW || a.dx)) { e = o.ea == 64 ? go<1>(a, o, cut, part, st) : o.ea == 128 ? go<2>(a, o, cut, part, st) : go<4>(a, o, cut, part, st); }
    if (e == hipSuccess && a.dW && sp > 1) {
        const int64_t n4 = (int64_t) a.n_exp * a.E / 4;
        k_route_join<<<(unsigned) ((n4 + 255) / 256), 256, 0, st>>>(part, sp, n4, a.accumulate, a.dW);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace lk
