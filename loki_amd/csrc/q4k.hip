// q4k.hip -- products of Q4_K matrices (ggml's 4-bit blocks with 6-bit group scales and mins, read in place) with Q8_K
// rows. Q4_K is the format of the reference's attention and dense-layer matrices
// (src/fused_layer.cu:71-101).
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

// Mat-vec: a workgroup takes one expert and a tile of rows, that expert's slots one after the other, whose Q8_K columns it holds in
// registers. Lane = (block of 8, 32-weight slice of the block), so a wave reads 1152 consecutive bytes of a row per pass; the
// next row's bytes are in flight while one is computed. Each block's term goes to LDS, one lane per row then runs the chain.
// Bound by memory where the rows are many: one token through 131072 rows of 7168 94 us, 5.6 TB/s.
__global__ void __launch_bounds__(256) k_q4k_vec(KqArgs a) {
#pragma clang fp contract(off)
    constexpr int BS = 144;
    extern __shared__ float s_lds[];   // terms [rw][nbp], then block scales [nbp]
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
    float * s_d = s_lds + a.rw * nbp;
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
    for (int t = s_beg; t < s_end; ++t) {
        for (int p = kw; p < npass; p += wk) {
            const int b = 8 * p + (lane >> 3);
            const bool active = b < nb;
            XChunk x{};
            if (active) {
                load_x<KF_Q4K>(a.aq + (size_t) t * a.K + 256 * b, c, x);
                if (c == 0 && rg == 0) { s_d[b] = a.ad[(size_t) t * nb + b]; }
            }
            auto row = [&](const Raw<KF_Q4K> & raw, int ri) {
                Chunk ck; decode<KF_Q4K>(raw, c, ck);
                int is, sm;
                chunk_dot<KF_Q4K>(ck, x, is, sm);
                is = red8(is); sm = red8(sm);
                if (c == 0 && active) { s_lds[ri * nbp + b] = __builtin_fmaf(-ck.dmin, (float) sm, ck.d * (float) is); }
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
        for (int ri = threadIdx.x; ri < nrow; ri += blockDim.x) {   // blocks in order, one lane per row
            float acc = 0.f;
            for (int j = 0; j < nb; ++j) { acc = __builtin_fmaf(s_d[j], s_lds[ri * nbp + j], acc); }
            Out[(size_t) t * a.ldo + tr0 + ri] = acc;
        }
        __syncthreads();
    }
}

hipError_t vec(KqArgs a, unsigned gy, hipStream_t st) {
    const int nb = a.K / QK, nbp = nb | 1;
    a.rw = (int) std::max<int64_t>(1, std::min<int64_t>({ V_ROWS, (int64_t) a.R * gy / 1024, V_LDS / (int) (nbp * sizeof(float)) - 1 }));   // ~1024 workgroups
    const dim3 grid((unsigned) ((a.R + a.rw - 1) / a.rw), gy);
    k_q4k_vec<<<grid, 64 * v_wk(nb) * v_wr(nb), (size_t) (a.rw + 1) * nbp * sizeof(float), st>>>(a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- matrix cores
// Tiles of rows x tokens on v_mfma_i32_16x16x64_i8, the weights as two int8 digits: s_j = 8 h_j + l_j with both below 8, so
// h_j q and l_j q are at most 105 and isum = 8 sum (h q) x + sum (l q) x, both sums exact in int32. The digits are made in
// registers: a lane's 16 weights of one step share their sub-block, so a dword of 4 quants takes one 16-bit packed multiply per
// digit. summ comes from one v_mfma_f32_16x16x32_f16 per block: the min m_j against the sub-block's sum as 64 b + c (|64 b| <=
// 4096, 0 <= c < 64, all fp16 integers, k_q4k_sums), every partial sum an integer below 2^24, so exact in fp32.
//
// Lane (r, g) of a wave holds row r of each of its 16-row tiles and the quant bytes 64 p + 16 g .. + 15 (p = 0, 1) of a block;
// step (p, h) takes their nibbles h: sub-block 4 p + 2 (g / 2) + h, activations 128 p + 64 (g / 2) + 32 h + 16 (g % 2) .. + 15.
typedef int qi4 __attribute__((ext_vector_type(4)));
typedef float qf4 __attribute__((ext_vector_type(4)));
typedef _Float16 qh2 __attribute__((ext_vector_type(2)));
typedef _Float16 qh8 __attribute__((ext_vector_type(8)));
typedef unsigned short qu2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t q4_rsrc(const void * p, uint32_t bytes) {
    const uint64_t v = (uint64_t) p;
    const uint32_t hi = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) (v >> 32)), lo = (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) v);
    return __builtin_amdgcn_make_buffer_rsrc((void *) (((uint64_t) hi << 32) | lo), (short) 0, __builtin_amdgcn_readfirstlane((int) bytes), 0x00020000);
}
// BYTES (4 or 16) per lane from a buffer straight into LDS, lane L at dst + BYTES L; the builtin exists for the device pass only
template <int BYTES> __device__ __forceinline__ void q4_lds(__amdgpu_buffer_rsrc_t r, LK_LOCAL uint8_t * dst, uint32_t voff, uint32_t soff) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (BYTES == 16) { __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LK_LOCAL void *) dst, 16, voff, soff, 0, 0); }
    else { __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LK_LOCAL void *) dst, 4, voff, soff, 0, 0); }
#else
    (void) r; (void) dst; (void) voff; (void) soff;
#endif
}
// A barrier for what the waves wrote to LDS themselves: __syncthreads would also wait for the copies into LDS that are under way for
// later rounds (VM: loads that may stay out)
template <int VM> __device__ __forceinline__ void q4_barrier() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070 | (VM & 15) | ((VM >> 4) << 14));   // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    __asm__ volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t pk_mul(uint32_t a, uint32_t b) { return __builtin_bit_cast(uint32_t, (qu2) (__builtin_bit_cast(qu2, a) * __builtin_bit_cast(qu2, b))); }

// the sums of a row's sub-blocks as fp16 pairs: xs [row][block][64 b of sub-blocks 0 .. 7, c of sub-blocks 0 .. 7]
__global__ void __launch_bounds__(256) k_q4k_sums(const int8_t * __restrict__ q, int64_t nsub, _Float16 * __restrict__ xs) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;   // sub-block: 32 values
    if (i >= nsub) { return; }
    const uint4 a = gload16(q + 32 * i), b = gload16(q + 32 * i + 16);
    const uint32_t w[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
    int s = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) { s = __builtin_amdgcn_sdot4((int) w[k], 0x01010101, s, false); }
    _Float16 * o = xs + (i >> 3) * 16 + (i & 7);
    o[0] = (_Float16) (float) (s & ~63); o[8] = (_Float16) (float) (s & 63);
}

struct Q4Args {
    const uint8_t * w, * w2; const int8_t * aq; const float * ad; const _Float16 * xs;
    int K, R, n; float * out, * out2; int ldo;
    int rt, tt;   // row tiles and token tiles of the workgroups
};

// a workgroup's row tile and token tile: consecutive workgroups go to the 8 XCDs in turn, so each XCD gets a run of tiles,
// token tiles of one row tile next to each other (its L2 then serves the weights to all of them)
__device__ __forceinline__ void q4_tile(const Q4Args & a, int & rt, int & tt) {
    const int total = a.rt * a.tt, b = blockIdx.x, per = total / 8, rest = total % 8, x = b & 7, i = b >> 3;
    const int t = x * per + min(x, rest) + i;
    rt = t / a.tt; tt = t % a.tt;
}

// A lane's operands of one row tile's block from its header and quant words: digits (high and low) of the four steps
__device__ __forceinline__ void q4_digits(const u32x4 (&w)[3], uint32_t sel0, qi4 (&wl)[4], qi4 (&wh)[4]) {
    const uint32_t sc[2] = { w[0].y & 0x3F3F3F3Fu, (w[0].w & 0x0F0F0F0Fu) | ((w[0].y >> 2) & 0x30303030u) };
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const uint32_t lo = sc[p] & 0x07070707u, hi = (sc[p] >> 3) & 0x07070707u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t sl = __builtin_amdgcn_perm(0u, lo, sel0 + (h ? 0x00010001u : 0u)), sh = __builtin_amdgcn_perm(0u, hi, sel0 + (h ? 0x00010001u : 0u));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u = (w[1 + p][k] >> (4 * h)) & 0x0F0F0F0Fu;
                wl[2 * p + h][k] = (int) pk_mul(u, sl); wh[2 * p + h][k] = (int) pk_mul(u, sh);
            }
        }
    }
}
// the mins of a block's sub-blocks 0 .. 3 and 4 .. 7, one a byte
__device__ __forceinline__ void q4_mins(const u32x4 & hd, uint32_t (&mm)[2]) {
    mm[0] = hd.z & 0x3F3F3F3Fu; mm[1] = ((hd.w >> 4) & 0x0F0F0F0Fu) | ((hd.z >> 2) & 0x30303030u);
}

// Few tokens: a workgroup's 8 waves share its rows and tokens and split K, wave w taking blocks w, w + 8, ... of the rows. A round's 8
// blocks of a row are 1152 consecutive bytes: they are copied into LDS in whole, a round ahead (a wave's lanes fetching 16 rows'
// pieces of 64 bytes themselves make twice the cache accesses, 37 a load instead of 19: 16 tokens through 65536 rows of 7168 95 us instead
// of 86). A wave's activations come into registers straight from the caches, each round's loads issued as soon as the last round's
// products are done with the registers (a second set, filled a round earlier, holds every wave up at the round's start behind the
// others' loads: 37 tokens through 7168 rows of 16384 39 us instead of 33). Each round leaves the blocks' terms in LDS, and the
// workgroup's lanes run the chains over them, an output or two a lane. summ comes from a third product with the step's min in every
// byte (here the matrix cores have time to spare). 37 tokens through 7168 rows of 16384 take 31 us a call. Of 33, found by leaving out one part at a time: the copies and loads that
// the products wait for 7, products and digits 14, the barriers, LDS reads and terms of the 8 rounds 7, the launch and first fetch 4.
constexpr int KS_W = 8, KS_PITCH = 9 * KS_W + 1;   // 16-byte chunks from row to row in LDS: 16 rows start in 16 different quads of banks
// copy i of a wave (past the last one: an earlier one of its own again, the same bytes, so that every wave has as many out)
template <int ALLC> __device__ __forceinline__ int q4_copy(int wave, int i) { const int k = wave + KS_W * i; return k < ALLC ? k : wave; }
template <int RT, int NT> struct KsLds {
    static constexpr int ALLC = (16 * RT * KS_PITCH + 63) / 64, COPIES = (ALLC + KS_W - 1) / KS_W, WB = ALLC * 1024;   // copies of a round, a wave's, bytes
    static constexpr int TOK = 16 * NT, TT = 80 * 4 * NT;   // a wave's terms of a row tile: token t, row r at 80 (t / 4) + 16 (t % 4) + r
    static constexpr int T0 = 2 * WB, D0 = T0 + KS_W * RT * TT * 4, ALL = D0 + KS_W * TOK * 4;
};
template <int RT, int NT>
__global__ void __launch_bounds__(64 * KS_W, RT * NT == 1 ? 4 : 2) k_q4k_ks(KqArgs a) {
#pragma clang fp contract(off)
    using L = KsLds<RT, NT>;
    constexpr int BS = 144, TOK = L::TOK, TT = L::TT;
    extern __shared__ __attribute__((aligned(16))) uint8_t q4_dyn[];
    LK_LOCAL uint8_t * lds = (LK_LOCAL uint8_t *) q4_dyn;
    LK_LOCAL float * s_t = (LK_LOCAL float *) (lds + L::T0), * s_d = (LK_LOCAL float *) (lds + L::D0);   // [wave][row tile][TT], [wave][TOK]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), r = lane & 15, g = lane >> 4;
    int e, s_beg, s_end;
    if (a.act) {
        if ((int) blockIdx.y >= *a.nact) { return; }
        e = a.act[blockIdx.y]; s_beg = a.offsets[e]; s_end = a.offsets[e + 1];
    } else { e = 0; s_beg = (int) blockIdx.z * TOK; s_end = min(s_beg + TOK, a.n); }
    const bool second = !a.act && blockIdx.y == 1;
    const int row0 = (int) blockIdx.x * 16 * RT, nrow = min(16 * RT, a.R - row0), nb = a.K / QK;
    const uint32_t rowb = (uint32_t) (nb * BS);
    float * Out = second ? a.out2 : a.out;
    // rows past the matrix's end and tokens past the group's read 0, as does a lane offset of OUT: a descriptor spans less than
    // 2^31 bytes, and the scalar offset beside it stays inside the span
    constexpr uint32_t OUT = 0x80000000u;
    const __amdgpu_buffer_rsrc_t rw = q4_rsrc((second ? a.w2 : a.w) + (size_t) e * a.estride + (size_t) row0 * rowb, (uint32_t) nrow * rowb);
    uint32_t vw[L::COPIES], vx[NT];
    int cw[L::COPIES];   // the chunk of its row that the lane copies
#pragma unroll
    for (int i = 0; i < L::COPIES; ++i) {
        const int p = 64 * q4_copy<L::ALLC>(wave, i) + lane, row = p / KS_PITCH;
        cw[i] = p % KS_PITCH; vw[i] = (uint32_t) row * rowb + (uint32_t) (cw[i] * 16);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) { vx[t] = (uint32_t) (16 * t + r) * (uint32_t) a.K + (uint32_t) (64 * (g >> 1) + 16 * (g & 1)); }
    const uint32_t sel0 = 0x0c000c00u | (uint32_t) (2 * (g >> 1)) * 0x00010001u, selm = (uint32_t) (2 * (g >> 1)) * 0x01010101u;
    const uint32_t lw = (uint32_t) (size_t) lds + (uint32_t) (r * KS_PITCH * 16 + wave * BS);
    for (int sg = s_beg; sg < s_end; sg += TOK) {
        const int nt = min(TOK, s_end - sg);
        const __amdgpu_buffer_rsrc_t rx = q4_rsrc(a.aq + (size_t) sg * a.K, (uint32_t) nt * (uint32_t) a.K);
        const __amdgpu_buffer_rsrc_t rd = q4_rsrc(a.ad + (size_t) sg * nb, (uint32_t) nt * (uint32_t) nb * 4);
        auto copy = [&](int j, int s) {   // blocks j .. j + 7 of every row (past the row's end: nothing is fetched)
            const int nc = 9 * min(KS_W, nb - j);   // (none or fewer: every lane stays out)
#pragma unroll
            for (int i = 0; i < L::COPIES; ++i) {
                q4_lds<16>(rw, lds + s * L::WB + q4_copy<L::ALLC>(wave, i) * 1024, cw[i] < nc ? vw[i] : OUT, (uint32_t) (min(j, nb - 1) * BS));
            }
        };
        struct Act { qi4 x[NT][4]; uint32_t d; };
        auto load_x = [&](int b, Act & o) {   // (past the last block: nothing is fetched)
            const uint32_t out = b < nb ? 0u : OUT;
            b = min(b, nb - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {   // step (p, h) = (k / 2, k % 2): 128 p + 32 h further
                    o.x[t][k] = __builtin_bit_cast(qi4, __builtin_amdgcn_raw_buffer_load_b128(rx, (vx[t] | out) + (uint32_t) (128 * (k >> 1) + 32 * (k & 1)), (uint32_t) (b * QK), 0));
                }
            }
            o.d = __builtin_amdgcn_raw_buffer_load_b32(rd, (uint32_t) ((lane < TOK ? lane : 0) * nb * 4) | out, (uint32_t) (b * 4), 0);
        };
        float acc[(RT * TOK * 16 + 64 * KS_W - 1) / (64 * KS_W)];
        constexpr int NO = sizeof(acc) / sizeof(acc[0]);
#pragma unroll
        for (int i = 0; i < NO; ++i) { acc[i] = 0.f; }
        auto round = [&](Act & v, int j0, int s) {
            if (j0 + wave < nb) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const uint32_t at = lw + (uint32_t) (s * L::WB + 16 * i * KS_PITCH * 16);
                    u32x4 w[3];
                    w[0] = *(const LK_LOCAL u32x4 *) (size_t) at;
                    w[1] = *(const LK_LOCAL u32x4 *) (size_t) (at + 16u + 16u * g);
                    w[2] = *(const LK_LOCAL u32x4 *) (size_t) (at + 80u + 16u * g);
                    qi4 wl[4], wh[4];
                    uint32_t mm[2];
                    q4_digits(w, sel0, wl, wh);
                    q4_mins(w[0], mm);
                    const float dd = h2f((uint16_t) (w[0].x & 0xFFFFu)), dm = -h2f((uint16_t) (w[0].x >> 16));
                    qi4 mv[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int m = (int) __builtin_amdgcn_perm(0u, mm[k >> 1], selm + ((k & 1) ? 0x01010101u : 0u));
                        mv[k] = (qi4) { m, m, m, m };
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        qi4 hs = { 0, 0, 0, 0 }, ls = hs, ms = hs;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            hs = __builtin_amdgcn_mfma_i32_16x16x64_i8(v.x[t][k], wh[k], hs, 0, 0, 0);
                            ls = __builtin_amdgcn_mfma_i32_16x16x64_i8(v.x[t][k], wl[k], ls, 0, 0, 0);
                            ms = __builtin_amdgcn_mfma_i32_16x16x64_i8(v.x[t][k], mv[k], ms, 0, 0, 0);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {   // token 16 t + 4 g + k
                            const float fi = (float) (int) (((uint32_t) hs[k] << 3) + (uint32_t) ls[k]);
                            s_t[(wave * RT + i) * TT + 80 * (4 * t + g) + 16 * k + r] = __builtin_fmaf(dm, (float) ms[k], dd * fi);
                        }
                    }
                }
                if (lane < TOK) { s_d[wave * TOK + lane] = __builtin_bit_cast(float, v.d); }
            }
            load_x(j0 + KS_W + wave, v);   // the next round's, into the registers that the products are done with
            q4_barrier<63>();
            const int m = min(KS_W, nb - j0);
#pragma unroll
            for (int i = 0; i < NO; ++i) {
                const int p = threadIdx.x + 64 * KS_W * i, q = p >> 4, t = q % TOK, ri = q / TOK;   // row p % 16 of row tile ri, token t
                if (p < RT * TOK * 16) {
                    const LK_LOCAL float * tp = s_t + ri * TT + 80 * (t >> 2) + 16 * (t & 3) + (p & 15), * dp = s_d + t;
                    if (m == KS_W) {
#pragma unroll
                        for (int w = 0; w < KS_W; ++w) { acc[i] = __builtin_fmaf(dp[w * TOK], tp[w * RT * TT], acc[i]); }
                    } else {
                        for (int w = 0; w < m; ++w) { acc[i] = __builtin_fmaf(dp[w * TOK], tp[w * RT * TT], acc[i]); }
                    }
                }
            }
        };
        Act x;
        constexpr int XL = 4 * NT + 1;   // the next round's activations may still be out when a round starts
        copy(0, 0);
        load_x(wave, x);
        for (int j0 = 0;;) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                q4_barrier<XL>();   // the round's copies have landed, this wave's and so everyone's; the last round's buffer and the terms are free
                copy(j0 + KS_W, i ^ 1);
                __builtin_amdgcn_sched_barrier(0);
                round(x, j0, i);
                if ((j0 += KS_W) >= nb) { goto done; }
            }
        }
done:
#pragma unroll
        for (int i = 0; i < NO; ++i) {
            const int p = threadIdx.x + 64 * KS_W * i, q = p >> 4, t = q % TOK, row = 16 * (q / TOK) + (p & 15);
            if (p < RT * TOK * 16 && t < nt && row < nrow) { Out[(size_t) (sg + t) * a.ldo + row0 + row] = acc[i]; }
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);   // no copy into LDS is out (the last rounds' fetch nothing, but write)
        __syncthreads();                      // the buffers are free for the next group, or the next workgroup
    }
}
template <int RT, int NT> hipError_t ks(const KqArgs & a, unsigned gy, hipStream_t st) {
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_q4k_ks<RT, NT>, KsLds<RT, NT>::ALL)) { return e; }
    k_q4k_ks<RT, NT><<<dim3((unsigned) ((a.R + 16 * RT - 1) / (16 * RT)), gy, a.act ? 1u : (unsigned) ((a.n + 16 * NT - 1) / (16 * NT))), 64 * KS_W, KsLds<RT, NT>::ALL, st>>>(a);
    return hipGetLastError();
}

// Many tokens: W waves of RT 16-row tiles each, NT 16-token tiles; blocks run D - 1 ahead: weights in registers, activations in LDS
// (copied there by the loads themselves, 16-byte chunks swizzled so that a tile's reads meet no bank twice). Each weight is decoded
// once per workgroup and each activation read from LDS serves RT tiles, so the largest tile, 128 x 128, does the most work an
// instruction; smaller ones are for calls that it would leave CUs without a workgroup (launch_rules.h). 2048 tokens through 16384 rows of
// 7168 505 us, 953 TFLOP/s of the real product: the matrix cores are busy 55 % of the cycles and the vector units with digits and terms
// 50 %, at the 1.9 GHz that the card then holds. Where a CU gets one workgroup, one wave a SIMD does its products (40 % of the cycles) and
// its vector work (35 %) one after the other; 8 waves of one row tile then overlap the two, at twice the LDS reads: 501 tokens through
// 7000 rows of 7168 68 us instead of 75.
template <int RT, int NT, int W, int D>
__global__ void __launch_bounds__(64 * W, 2) k_q4k_mm(Q4Args a) {
#pragma clang fp contract(off)
    constexpr int BS = 144, TOK = 16 * NT, XB = TOK * 256, SB = TOK * 32, BUF = XB + SB + TOK * 4;
    constexpr int IX = TOK / 4 / W, IS = (TOK * 2 + 64 * W - 1) / (64 * W), ID = (TOK + 64 * W - 1) / (64 * W);   // copies a wave and block
    constexpr int NL = IX + IS + ID + 3 * RT, LEFT = (D - 2) * NL;
    static_assert(TOK / 4 % W == 0 && LEFT < 64, "x copies shared evenly; outstanding loads");
    extern __shared__ __attribute__((aligned(16))) uint8_t q4_dyn[];
    LK_LOCAL uint8_t * lds = (LK_LOCAL uint8_t *) q4_dyn;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = lane_id(), r = lane & 15, g = lane >> 4;
    int rt0, tt0;
    q4_tile(a, rt0, tt0);
    const bool second = blockIdx.y == 1;
    const int nb = a.K / QK, row0 = (rt0 * W + wave) * RT * 16, t0 = tt0 * TOK, nt = min(TOK, a.n - t0);
    const uint32_t rowb = (uint32_t) (nb * BS);
    // a wave's rows; one wholly past the matrix's end reads the first rows and stores nothing. Rows past the end read 0: scalar offsets stay
    // inside the descriptor's span, lane offsets pass it
    const int nrow = max(0, min(RT * 16, a.R - row0)), rrow = nrow > 0 ? row0 : 0;
    const __amdgpu_buffer_rsrc_t rw = q4_rsrc((second ? a.w2 : a.w) + (size_t) rrow * rowb, (uint32_t) min(RT * 16, a.R - rrow) * rowb);
    const __amdgpu_buffer_rsrc_t rx = q4_rsrc(a.aq + (size_t) t0 * a.K, (uint32_t) nt * (uint32_t) a.K);
    const __amdgpu_buffer_rsrc_t rs = q4_rsrc(a.xs + (size_t) t0 * nb * 16, (uint32_t) nt * (uint32_t) nb * 32);
    const __amdgpu_buffer_rsrc_t rd = q4_rsrc(a.ad + (size_t) t0 * nb, (uint32_t) nt * (uint32_t) nb * 4);
    // Copies into LDS. x: 4 rows a copy, 16-byte chunk c of token t at slot c ^ (t % 16); sums 32 a copy, block scales 64 (a wave
    // past their end copies the last ones again: the same bytes). Tokens past the batch's end repeat its last one.
    uint32_t vx[IX], vs[IS], vd[ID];
    const int ws = min(wave, (TOK * 2 - 1) / 64), wd = min(wave, (TOK - 1) / 64);
#pragma unroll
    for (int i = 0; i < IX; ++i) {
        const int t = 4 * (wave * IX + i) + (lane >> 4);
        vx[i] = (uint32_t) min(t, nt - 1) * (uint32_t) a.K + (uint32_t) (((lane & 15) ^ (t & 15)) << 4);
    }
#pragma unroll
    for (int i = 0; i < IS; ++i) { const int c = 64 * min(ws + i * W, (TOK * 2 - 1) / 64) + lane; vs[i] = (uint32_t) min(c >> 1, nt - 1) * (uint32_t) (nb * 32) + (uint32_t) ((c & 1) << 4); }
#pragma unroll
    for (int i = 0; i < ID; ++i) { const int t = 64 * min(wd + i * W, (TOK - 1) / 64) + lane; vd[i] = (uint32_t) min(t, nt - 1) * (uint32_t) (nb * 4); }
    uint32_t vw[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) { vw[i] = (uint32_t) (16 * i + r) * rowb + 16u * g; }
    const uint32_t vh = (uint32_t) 0 - 16u * g;   // from a lane's quants back to the block's header
    auto copy = [&](int j, int s) {   // (past the last block: it again, unread, so that every trip has the same loads)
        j = min(j, nb - 1);
        LK_LOCAL uint8_t * buf = lds + s * BUF;
#pragma unroll
        for (int i = 0; i < IX; ++i) { q4_lds<16>(rx, buf + 1024 * (wave * IX + i), vx[i], (uint32_t) j * QK); }
#pragma unroll
        for (int i = 0; i < IS; ++i) {   // (lanes past the sums' end stay out)
            const int k = min(ws + i * W, (TOK * 2 - 1) / 64);
            if (SB % 1024 == 0 || 1024 * k + 16 * lane < SB) { q4_lds<16>(rs, buf + XB + 1024 * k, vs[i], (uint32_t) j * 32); }
        }
#pragma unroll
        for (int i = 0; i < ID; ++i) {
            const int k = min(wd + i * W, (TOK - 1) / 64);
            if (TOK % 64 == 0 || 64 * k + lane < TOK) { q4_lds<4>(rd, buf + XB + SB + 256 * k, vd[i], (uint32_t) j * 4); }
        }
    };
    u32x4 raw[D - 1][RT][3];
    auto load = [&](int j, u32x4 (&w)[RT][3]) {
        const uint32_t so = (uint32_t) (min(j, nb - 1) * BS);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            w[i][0] = __builtin_amdgcn_raw_buffer_load_b128(rw, vw[i] + vh, so, 0);
            w[i][1] = __builtin_amdgcn_raw_buffer_load_b128(rw, vw[i] + 16u, so, 0);
            w[i][2] = __builtin_amdgcn_raw_buffer_load_b128(rw, vw[i] + 80u, so, 0);
        }
    };
    qf4 acc[RT][NT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
#pragma unroll
        for (int t = 0; t < NT; ++t) { acc[i][t] = (qf4) { 0.f, 0.f, 0.f, 0.f }; }
    }
    const uint32_t sel0 = 0x0c000c00u | (uint32_t) (2 * (g >> 1)) * 0x00010001u;       // the lane's byte of a scale word, for h = 0; + 1 for h = 1
    const _Float16 on = (_Float16) (g < 2 ? 1.f : 0.f), off = (_Float16) (g < 2 ? -1024.f : 0.f);   // lane groups 2 and 3 hold no sums
    const uint32_t c0 = (uint32_t) (4 * (g >> 1) + (g & 1));
    uint32_t ox[4];   // the lane's chunk of each step in a token row
#pragma unroll
    for (int k = 0; k < 4; ++k) { ox[k] = (uint32_t) (256 * r) + (((c0 + (uint32_t) (8 * (k >> 1) + 2 * (k & 1))) ^ (uint32_t) r) << 4); }
    const uint32_t os = (uint32_t) (XB + 32 * r + 16 * (g & 1)), od = (uint32_t) (XB + SB + 16 * g);
    auto block = [&](u32x4 (&w)[RT][3], int s, int jn) {
        qi4 wl[RT][4], wh[RT][4];
        qh8 mn[RT];
        float dd[RT], dm[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const u32x4 hd = w[i][0];
            dd[i] = h2f((uint16_t) (hd.x & 0xFFFFu)); dm[i] = -h2f((uint16_t) (hd.x >> 16));
            uint32_t mm[2];
            q4_mins(hd, mm);
            qh2 m2[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {   // mins 2 k, 2 k + 1 as fp16: 0x6400 | m = 1024 + m
                const qh2 v = __builtin_bit_cast(qh2, __builtin_amdgcn_perm(0x64646464u, mm[k >> 1], (k & 1) ? 0x04030402u : 0x04010400u));
                m2[k] = __builtin_elementwise_fma(v, (qh2) { on, on }, (qh2) { off, off });
            }
            mn[i] = (qh8) { m2[0][0], m2[0][1], m2[1][0], m2[1][1], m2[2][0], m2[2][1], m2[3][0], m2[3][1] };
            q4_digits(w[i], sel0, wl[i], wh[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);   // products before another wave's digits (1000 tokens through 7168 rows of 16384 258 us, without 273)
        load(jn, w);   // into the registers that the block is done with
        const uint32_t xb = (uint32_t) (size_t) lds + (uint32_t) (s * BUF);
        qi4 x[4]; qh8 sv; qf4 d8;
#pragma unroll
        for (int k = 0; k < 4; ++k) { x[k] = *(const LK_LOCAL qi4 *) (size_t) (xb + ox[k]); }
        sv = *(const LK_LOCAL qh8 *) (size_t) (xb + os);
        d8 = *(const LK_LOCAL qf4 *) (size_t) (xb + od);
#pragma unroll
        for (int t = 0; t < NT; ++t) {   // each operand's registers take the next tile's once it is used
            const uint32_t xn = xb + (uint32_t) ((t + 1) * 16 * 256);
            qi4 hs[RT], ls[RT]; qf4 ms[RT];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const qi4 z = { 0, 0, 0, 0 };
                    hs[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[k], wh[i][k], k == 0 ? z : hs[i], 0, 0, 0);
                    ls[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[k], wl[i][k], k == 0 ? z : ls[i], 0, 0, 0);
                }
                if (t + 1 < NT) { x[k] = *(const LK_LOCAL qi4 *) (size_t) (xn + ox[k]); }
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) { ms[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(sv, mn[i], (qf4) { 0.f, 0.f, 0.f, 0.f }, 0, 0, 0); }
            if (t + 1 < NT) { sv = *(const LK_LOCAL qh8 *) (size_t) (xb + os + (uint32_t) ((t + 1) * 16 * 32)); }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float fi = (float) (int) (((uint32_t) hs[i][k] << 3) + (uint32_t) ls[i][k]);
                    acc[i][t][k] = __builtin_fmaf(d8[k], __builtin_fmaf(dm[i], ms[i][k], dd[i] * fi), acc[i][t][k]);
                }
            }
            if (t + 1 < NT) { d8 = *(const LK_LOCAL qf4 *) (size_t) (xb + od + (uint32_t) ((t + 1) * 16 * 4)); }
        }
    };
#pragma unroll
    for (int s = 0; s < D - 1; ++s) { copy(s, s); load(s, raw[s]); }
    // D LDS buffers and D - 1 register sets: trips of D (D - 1) blocks have both fixed
    for (int j = 0;;) {
#pragma unroll
        for (int s = 0; s < D * (D - 1); ++s) {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0f70 | (LEFT & 15) | ((LEFT >> 4) << 14));   // block j: this wave's copies have landed
            __builtin_amdgcn_s_barrier();                                             // and everyone's; buffer (s + D - 1) % D is free
            copy(j + D - 1, (s + D - 1) % D);
            __builtin_amdgcn_sched_barrier(0);
            block(raw[s % (D - 1)], s % D, j + D - 1);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);   // (register moves of the next block's weights stay here: inside the block they would wait for them)
            if (++j == nb) { goto done; }   // (a jump, not a guard around each block: the compiler then knows which loads are out)
        }
    }
done:
    __builtin_amdgcn_s_waitcnt(0x0f70);   // no copy into LDS outlives the workgroup
    float * out = second ? a.out2 : a.out;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if (16 * i + r < nrow) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int tok = 16 * t + 4 * g + k;
                    if (tok < nt) { out[(size_t) (t0 + tok) * a.ldo + row0 + 16 * i + r] = acc[i][t][k]; }
                }
            }
        }
    }
}

template <int RT, int NT, int W, int D> hipError_t mm(const KqArgs & k, hipStream_t st) {
    constexpr int LDS = D * 16 * NT * (256 + 32 + 4);
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_q4k_mm<RT, NT, W, D>, LDS)) { return e; }
    Q4Args a{};
    a.w = k.w; a.w2 = k.w2; a.aq = k.aq; a.ad = k.ad; a.xs = (const _Float16 *) k.xs; a.K = k.K; a.R = k.R; a.n = k.n;
    a.out = k.out; a.out2 = k.out2; a.ldo = k.ldo;
    a.rt = (k.R + 16 * RT * W - 1) / (16 * RT * W); a.tt = (k.n + 16 * NT - 1) / (16 * NT);
    k_q4k_mm<RT, NT, W, D><<<dim3((unsigned) (a.rt * a.tt), k.w2 ? 2 : 1), 64 * W, LDS, st>>>(a);
    return hipGetLastError();
}

}  // namespace

size_t q4k_scratch_bytes(int n, int64_t R, int K) { return q4k_tiled(q4k_kernel(n, R, K, true)) ? (size_t) n * (K / QK) * 32 : 0; }

hipError_t launch_q4k(const KqArgs & a, int max_slots, int grid_experts, hipStream_t st) {
    if (a.K <= 0 || a.K % QK || a.K > QK * V_NB || a.R <= 0 || max_slots <= 0 || grid_experts <= 0) { return hipErrorInvalidValue; }
    const unsigned gy = a.act ? (unsigned) grid_experts : (a.w2 ? 2u : 1u);
    // (an expert's slots are known on the device alone: their expected number goes for the tokens)
    const int kernel = q4k_kernel(max_slots, (int64_t) a.R * gy, a.K, !a.act && a.xs);
    if (q4k_tiled(kernel)) {
        const int64_t nsub = (int64_t) a.n * (a.K / 32);
        k_q4k_sums<<<(unsigned) ((nsub + 255) / 256), 256, 0, st>>>(a.aq, nsub, (_Float16 *) a.xs);
        if (const hipError_t e = hipGetLastError()) { return e; }
    }
    switch (kernel) {
    case Q4_VEC: return vec(a, gy, st);
    case Q4_KS_16_16: return ks<1, 1>(a, gy, st);
    case Q4_KS_32_16: return ks<2, 1>(a, gy, st);
    case Q4_KS_32_32: return ks<2, 2>(a, gy, st);
    case Q4_KS_32_48: return ks<2, 3>(a, gy, st);
    case Q4_MM_64_32: return mm<1, 2, 4, 5>(a, st);
    case Q4_MM_64_64: return mm<1, 4, 4, 3>(a, st);
    case Q4_MM_128_64: return mm<1, 4, 8, 3>(a, st);
    case Q4_MM_256_64: return mm<2, 4, 8, 3>(a, st);
    case Q4_MM_128_128_8: return mm<1, 8, 8, 3>(a, st);
    default: return mm<2, 8, 4, 2>(a, st);
    }
}

}  // namespace lk
