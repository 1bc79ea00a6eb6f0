// q4k.hip -- products of Q4_K matrices (ggml's 4-bit blocks with 6-bit group scales and mins, read in place) with Q8_K
// rows. Q4_K is the format of the reference's attention and dense-layer matrices (tc_matvec<F_Q4K>,
// src/fused_layer.cu:71-101).
//
// A block is 256 weights in 144 bytes: fp16 d and dmin, 12 bytes of 6-bit scales s_j and mins m_j (8 sub-blocks of 32), 128
// bytes of quants; group jj = 0..3 of 32 quant bytes holds sub-block 2 jj in its low nibbles and 2 jj + 1 in its high ones.
// A weight is d s_j q - dmin m_j, so with a row's Q8_K integers x and their block scale d8
//   isum = sum_j s_j sum_i q_i x_i,   summ = sum_j m_j sum_i x_i           exact integers (|isum| < 2^25, |summ| < 2^21)
//   term = fma(-dmin, summ, d * isum),   y = fma(d8, term, y)              fp32, over the row's blocks in order, from 0
// with isum and summ rounded to fp32 once. Every kernel here forms the same integers and runs this same fp32 chain, so an
// output's bits depend on its matrix row and its activation row alone: not on n, R, or the kernel that a call gets.
#include "kquant_device.h"
#include "moe_kernels.h"

#include <algorithm>

namespace lk {

namespace {

constexpr int V_ROWS = 32;              // rows per workgroup tile at most
constexpr int V_LDS = 60 * 1024;        // its LDS at most
constexpr int V_NB = 256;               // blocks per row at most (K <= 65536)

// waves of a workgroup along K (8 blocks each per pass) and along its rows
constexpr int v_wk(int nb) { return nb > 24 ? 4 : nb > 16 ? 3 : nb > 8 ? 2 : 1; }
constexpr int v_wr(int nb) { return nb > 16 ? 1 : nb > 8 ? 2 : 4; }

// Mat-vecs: a workgroup takes one expert, a tile of rows and that expert's slots in token groups of up to TT, whose Q8_K
// columns it holds in registers. Lane = (block of 8, 32-weight slice of the block), so a wave reads 1152 consecutive bytes
// of a row per pass; the next row's bytes are in flight while one is computed. Each block's term goes to LDS, one lane
// per (row, token) then runs the chain.
template <int TT>
__global__ void __launch_bounds__(256) k_q4k_vec(KqArgs a) {
#pragma clang fp contract(off)
    constexpr int BS = 144;
    extern __shared__ float s_lds[];   // terms [rw][TT][nbp], then block scales [TT][nbp]
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int e, s_beg, s_end;
    if (a.act) {
        if ((int) blockIdx.y >= *a.nact) { return; }
        e = a.act[blockIdx.y]; s_beg = a.offsets[e]; s_end = a.offsets[e + 1];
    } else { e = 0; s_beg = 0; s_end = a.n; }
    const bool second = !a.act && blockIdx.y == 1;   // the second matrix (w2 -> out2)
    const int tr0 = (int) blockIdx.x * a.rw;
    if (tr0 >= a.R || s_beg >= s_end) { return; }
    const int nrow = min(a.rw, a.R - tr0), nb = a.K / QK, nbp = nb | 1, npass = (nb + 7) / 8;
    float * s_d = s_lds + a.rw * TT * nbp;
    const int wk = v_wk(nb), wr = v_wr(nb), kw = wv % wk, rg = wv / wk, c = lane & 7;
    const uint32_t rowb = (uint32_t) (nb * BS);
    // the tile's rows: reads past them give 0 (a lane past the row's last block reads the next row's bytes, unused)
    const uint8_t * W = (second ? a.w2 : a.w) + (size_t) e * a.estride + (size_t) tr0 * rowb;
    float * Out = second ? a.out2 : a.out;
    Src src;
    {
        const uint64_t p = (uint64_t) W;
        const uint32_t hi = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) (p >> 32));
        const uint32_t lo = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) p);
        src.rs = __builtin_amdgcn_make_buffer_rsrc((void *) (((uint64_t) hi << 32) | lo), (short) 0, (int) ((uint32_t) nrow * rowb), 0x00020000);
    }
    for (int sg = s_beg; sg < s_end; sg += TT) {
        const int nt = min(TT, s_end - sg);
        for (int p = kw; p < npass; p += wk) {
            const int b = 8 * p + (lane >> 3);
            const bool active = b < nb;
            XChunk xc[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                XChunk & x = xc[t];
                if (active && t < nt) {
                    load_x<KF_Q4K>(a.aq + (size_t) (sg + t) * a.K + 256 * b, c, x);
                    if (c == 0 && rg == 0) { s_d[t * nbp + b] = a.ad[(size_t) (sg + t) * nb + b]; }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) { x.x[i] = 0u; }
#pragma unroll
                    for (int i = 0; i < 4; ++i) { x.c0[i] = 0; x.bx[i] = 0; }
                }
            }
            auto row = [&](const Raw<KF_Q4K> & raw, int ri) {
                Chunk ck; decode<KF_Q4K>(raw, c, ck);
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    if (t < nt) {
                        int is, sm;
                        chunk_dot<KF_Q4K>(ck, xc[t], is, sm);
                        is = red8(is); sm = red8(sm);
                        if (c == 0 && active) { s_lds[(ri * TT + t) * nbp + b] = __builtin_fmaf(-ck.dmin, (float) sm, ck.d * (float) is); }
                    }
                }
            };
            const uint32_t step = (uint32_t) wr * rowb;
            Src sp = src; sp.vb = (uint32_t) (b * BS); sp.so = (uint32_t) rg * rowb;
            Raw<KF_Q4K> ra, rb;
            int ri = rg;
            if (ri < nrow) { load_raw<KF_Q4K>(sp, c, ra); }
            while (ri < nrow) {
                if (ri + wr < nrow) { Src sn = sp; sn.so += step; load_raw<KF_Q4K>(sn, c, rb); }
                row(ra, ri);
                ri += wr; sp.so += step;
                if (ri >= nrow) { break; }
                if (ri + wr < nrow) { Src sn = sp; sn.so += step; load_raw<KF_Q4K>(sn, c, ra); }
                row(rb, ri);
                ri += wr; sp.so += step;
            }
        }
        __syncthreads();
        for (int p = threadIdx.x; p < nrow * nt; p += blockDim.x) {   // blocks in order, one lane per (row, token)
            const int ri = p / nt, t = p % nt;
            const float * tp = s_lds + (ri * TT + t) * nbp, * dp = s_d + t * nbp;
            float acc = 0.f;
            for (int j = 0; j < nb; ++j) { acc = __builtin_fmaf(dp[j], tp[j], acc); }
            Out[(size_t) (sg + t) * a.ldo + tr0 + ri] = acc;
        }
        __syncthreads();
    }
}

template <int TT> hipError_t vec(KqArgs a, unsigned gy, hipStream_t st) {
    const int nb = a.K / QK, nbp = nb | 1;
    a.rw = std::max(1, std::min(a.rw, V_LDS / (int) (TT * nbp * sizeof(float)) - 1));
    const dim3 grid((unsigned) ((a.R + a.rw - 1) / a.rw), gy);
    k_q4k_vec<TT><<<grid, 64 * v_wk(nb) * v_wr(nb), (size_t) (a.rw + 1) * TT * nbp * sizeof(float), st>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_q4k(const KqArgs & args, int max_slots, int grid_experts, hipStream_t st) {
    KqArgs a = args;
    if (a.K <= 0 || a.K % QK || a.K > QK * V_NB || a.R <= 0 || max_slots <= 0 || grid_experts <= 0) { return hipErrorInvalidValue; }
    const unsigned gy = a.act ? (unsigned) grid_experts : (a.w2 ? 2u : 1u);
    const int tt = max_slots <= 1 ? 1 : max_slots <= 2 ? 2 : max_slots <= 4 ? 4 : 8;
    a.rw = (int) std::max<int64_t>(1, std::min<int64_t>(V_ROWS, (int64_t) a.R * gy / (tt >= 8 ? 512 : 1024)));
    return tt == 1 ? vec<1>(a, gy, st) : tt == 2 ? vec<2>(a, gy, st) : tt == 4 ? vec<4>(a, gy, st) : vec<8>(a, gy, st);
}

}  // namespace lk
