// matmul.hip -- products of bfloat16 / float16 matrices, dense or grouped by expert, and their backward pass.
//
//   forward  y[s][r]     = sum_k x[row(s)][k] W[e][r][k], with an epilogue     s: expert e's slots
//   dx       dx[s][k]    = sum_r dz[s][r] W[e][r][k] (+ dz2 W2)
//   dW       dW[e][r][k] = sum over e's slots of dz[s][r] x[row(s)][k]
//
// All three are D[m][n] = sum_k A[m][k] B[n][k] with D's rows along n in memory. The matrix cores take B as their first operand, so that a
// lane's four results lie next to each other in a row of D.
//
// A workgroup takes tiles of BM x BN, BK = 32 of the sum's terms a step. A step's operands are copied straight into LDS, 16 bytes a lane, S
// steps ahead; what lies outside an operand is not read and arrives as 0 (the buffer's range), so that no row of another expert, infinite
// or not, takes part. While a step's products run, the next step's operands go from LDS into the other set of registers. One barrier a step.
//
// In LDS an operand whose terms are next to each other in memory ("row" operand) has 64 bytes a row, chunk c of 16 at c ^ f(row / 4 % 4), f
// = 0, 2, 3, 1: a ds_read_b128 is served in passes of 16 lanes (0-3, 12-15, 20-23, 24-27; 4-11, 16-19, 28-31; and 32 on), and so each pass
// has 16 different bank quads (with f the identity half of the cycles of the LDS were conflicts). One whose terms are rows of memory ("col" operand) has a row a
// term, segments of 32 bytes at segment ^ (term % 4 + term / 8 % 2 * 4), and is transposed by ds_read_b64_tr_b16: 16 lanes read 4 terms x 16
// columns and each gets its column's 4.
#include "matmul_device.h"

namespace lk {
namespace {

enum { FWD, DX, DW };
constexpr int BK = 32;
constexpr uint32_t FAR = 0xFFFF0000u, WINDOW = 0xFFFE0000u;   // an offset outside every buffer; the largest range of one

// one step's copy instruction: 16 bytes a lane to m0 + 16 * lane; nothing of it is known to the compiler, which would wait for all copies
// before each ds_read_b64_tr_b16: the waits below are counted by hand. m0 is set at least one instruction before.
__device__ __forceinline__ uint32_t copy_to(uint32_t lds, uint32_t off) {
    uint32_t m = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("s_add_u32 %0, %1, %2" : "={m0}"(m) : "s"(lds), "s"(off) : "scc");
#endif
    return m;
}
__device__ __forceinline__ void copy16(uint32_t m, uint32_t voff, u32x4 rsrc) {
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("buffer_load_dwordx4 %1, %2, 0 offen lds" :: "{m0}"(m), "v"(voff), "s"(rsrc) : "memory");
#endif
}
template <int N> __device__ __forceinline__ void wait_copies() {   // all but the last N, and all LDS reads
    __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
}
__device__ __forceinline__ void meet() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ u32x4 buffer(uint64_t base, uint32_t bytes) { return (u32x4) { (uint32_t) base, (uint32_t) (base >> 32) & 0xFFFFu, bytes, 0x00020000u }; }
__device__ __forceinline__ uint64_t uni64(const void * p) {
    const uint64_t v = (uint64_t) p;
    return ((uint64_t) (uint32_t) uni((int) (uint32_t) (v >> 32)) << 32) | (uint32_t) uni((int) (uint32_t) v);
}

// a row operand's lane: it copies chunk `chunk` of row `lane / 4` of 16, and reads row lane % 16, chunk lane / 16
struct RowLane {
    uint32_t chunk, read;
    __device__ __forceinline__ RowLane() {
        const int l = lane_id();
        chunk = (uint32_t) ((l & 3) ^ swz((l >> 4) & 3));
        read = (uint32_t) ((l & 15) * 64 + (((l >> 4) ^ swz((l >> 2) & 3)) * 16));
    }
    __device__ __forceinline__ static int swz(int b) { return (((b ^ (b >> 1)) & 1) << 1) | (b >> 1); }
};
// a col operand's: of an instruction's 1024 bytes = 512 / COLS terms
template <int COLS> struct ColLane {
    static constexpr int TERMS = 512 / COLS;   // terms an instruction copies
    __device__ __forceinline__ static int term(int j) { return j * TERMS + lane_id() / (COLS / 8); }
    __device__ __forceinline__ static int column(int j) {   // first of the 8 columns it copies
        const int k = term(j), p = lane_id() % (COLS / 8);
        return 8 * ((((p >> 1) ^ swz(k)) << 1) | (p & 1));
    }
    __device__ __forceinline__ static int swz(int k) { return (k & 3) | ((k >> 1) & 4); }
    // the address of columns 16 j .. 16 j + 15 (j = 0 .. 7, + 8 i: + 256 i bytes), terms 8 (lane / 16) .. + 3; + 4: + 4 rows
    __device__ __forceinline__ static uint32_t read(int j) {
        const int l = lane_id(), k = 8 * (l >> 4) + ((l >> 2) & 3);
        return (uint32_t) (k * COLS * 2 + ((j ^ swz(k)) & 7) * 32 + (l & 3) * 8);
    }
};
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <class T> __device__ __forceinline__ V8<T> lds_row(uint32_t a) { return *(const LK_LOCAL V8<T> *) (size_t) a; }
template <class T, int COLS> __device__ __forceinline__ V8<T> lds_col(uint32_t a) {
    union { s16x4 s[2]; V8<T> v; } u;
#if defined(__HIP_DEVICE_COMPILE__)
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LK_LOCAL s16x4 *) (size_t) a);
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LK_LOCAL s16x4 *) (size_t) (a + 4 * COLS * 2));
#else
    u.v = (V8<T>) {};
#endif
    return u.v;
}

// ---------------------------------------------------------------- the launch's tiles
struct Tiles { int first[NEXP_MAX + 1]; };   // m-tiles of the experts before e; [n_exp]: all of them
__device__ __forceinline__ void count_tiles(Tiles & t, const int * offsets, int n, int n_exp, int bm) {   // (all threads; ends with a barrier)
    if (threadIdx.x < 64) {
        const int l = threadIdx.x;
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
        for (int j = 0; j < 4; ++j) { t.first[4 * l + j] = at; at += c[j]; }
        if (l == 63) { t.first[NEXP_MAX] = at; }
    }
    __syncthreads();
}
// the expert of tile `i`, i < the sum: the last one whose tiles begin at or before it
__device__ __forceinline__ int expert_of(const Tiles & t, int i) {
    int e = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) { e += __popcll(__ballot(t.first[4 * lane_id() + j] <= i)); }
    return uni(e) - 1;
}
struct Spot { int e, slot, nm, n0; };   // expert, first slot, its slots in the tile, first column
// tile i of the launch, i < first[NEXP_MAX] * nt: an expert's tiles are next to each other, in bands of `band` m-tiles, m fastest
__device__ __forceinline__ Spot spot_of(const Tiles & t, const int * offsets, int n, int nt, int bm, int bn, int band, int i) {
    Spot s;
    s.e = expert_of(t, i / nt);   // (first[e] * nt <= i exactly when first[e] <= i / nt)
    const Span sp = span_of(offsets, n, s.e);
    const int mt = uni(t.first[s.e + 1]) - uni(t.first[s.e]), in = i - uni(t.first[s.e]) * nt, b = in / (band * nt), rows = min(band, mt - b * band), r = in - b * band * nt;
    s.slot = uni(sp.begin) + (b * band + r % rows) * bm;
    s.nm = min(bm, uni(sp.end) - s.slot);
    s.n0 = r / rows * bn;
    return s;
}

// ---------------------------------------------------------------- a tile's sums
// NW = WM * WN waves, a wave BM / WM x BN / WN. A: m side, B: n side; AC, BC: whether they are col operands
template <class T, bool AC, bool BC, int BM_, int BN_, int WM_, int WN_, int S_> struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_, NW = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
    static constexpr int AB = BM * BK * 2, BB = BN * BK * 2, STAGE = AB + BB, LDS = S * STAGE;
    static constexpr int IA = AB / 1024 < NW ? 1 : AB / 1024 / NW, IB = BB / 1024 < NW ? 1 : BB / 1024 / NW, NI = IA + IB;   // copies a wave and step
    static constexpr int threads = 64 * NW;
    typedef V8<T> F;
};
template <class H> struct Frags { typename H::F a[H::FM], b[H::FN]; };

// which of an operand's 1024-byte pieces copy i of wave w takes (fewer pieces than waves: some copy the same one)
template <int BYTES, int I> __device__ __forceinline__ int piece(int w, int i) { return (w * I + i) % (BYTES / 1024); }

// the loop over the sum's steps. begin(t) and then set(j, slot address) and copy(j), j = 0 .. NI - 1, copy step t's operands; they are called for
// t past the end too, and then copy nothing (zeros).
// A wave has its SIMD to itself, and its products (16 cycles each) follow each other without a gap only if no more than three other
// instructions go between two of them: the copies and reads are dealt out among the products in this order, and what the next step needs
// in scalars and addresses is made among the last ones. The barrier comes after the step's first products, whose operands are in registers.
template <class T, bool AC, bool BC, class H, class Begin, class Set, class Copy>
__device__ __forceinline__ void sums(f32x4 (&acc)[H::FM][H::FN], uint32_t lds, int steps, Begin begin, Set set, Copy copy) {
    const int wave = uni(threadIdx.x >> 6), wm = wave / H::WN, wn = wave % H::WN;
    const RowLane row;
    constexpr int RA = AC ? (H::FM < 8 ? H::FM : 8) : 1, RB = BC ? (H::FN < 8 ? H::FN : 8) : 1;
    static_assert(!AC || (H::FM & (H::FM - 1)) == 0, "addresses of a col operand"); static_assert(!BC || (H::FN & (H::FN - 1)) == 0, "addresses of a col operand");
    uint32_t ra[RA], rb[RB];   // a lane's addresses in a stage
    if constexpr (AC) {
#pragma unroll
        for (int j = 0; j < RA; ++j) { ra[j] = ColLane<H::BM>::read(wm * H::FM + j) + (uint32_t) (wm * H::FM + j) / 8 * 256 + lds; }
    } else { ra[0] = row.read + (uint32_t) (wm * H::FM * 1024) + lds; }
    if constexpr (BC) {
#pragma unroll
        for (int j = 0; j < RB; ++j) { rb[j] = ColLane<H::BN>::read(wn * H::FN + j) + (uint32_t) (wn * H::FN + j) / 8 * 256 + H::AB + lds; }
    } else { rb[0] = row.read + (uint32_t) (wn * H::FN * 1024) + H::AB + lds; }
    struct At { uint32_t a[RA], b[RB]; } at;
    auto at_slot = [&](uint32_t off) {
#pragma unroll
        for (int j = 0; j < RA; ++j) { at.a[j] = ra[j] + off; __asm__("" : "+v"(at.a[j])); }   // (one register each, the fragments by immediate offsets)
#pragma unroll
        for (int j = 0; j < RB; ++j) { at.b[j] = rb[j] + off; __asm__("" : "+v"(at.b[j])); }
    };
    auto read_a = [&](Frags<H> & f, int i) {
        if constexpr (AC) { f.a[i] = lds_col<T, H::BM>(at.a[i % RA] + (uint32_t) (i / RA * 256)); } else { f.a[i] = lds_row<T>(at.a[0] + (uint32_t) (i * 1024)); }
    };
    auto read_b = [&](Frags<H> & f, int i) {
        if constexpr (BC) { f.b[i] = lds_col<T, H::BN>(at.b[i % RB] + (uint32_t) (i / RB * 256)); } else { f.b[i] = lds_row<T>(at.b[0] + (uint32_t) (i * 1024)); }
    };
    // G groups of products; the first has none of the rest, then come RG groups with reads and copies, then those with the next step's set-up
    constexpr int MF = H::FM * H::FN, RD = H::FM + H::FN, G = MF, RG = G - G / 4 - 1;
    static_assert(RG > H::NI, "a group between two copies");
    int slot = 0;            // of step t
    uint32_t here = lds;     // its place
    auto step = [&](Frags<H> & cur, Frags<H> & nxt, int t) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g <= RG; ++g) {
#pragma unroll
            for (int j = g * MF / G; j < (g + 1) * MF / G; ++j) { acc[j / H::FN][j % H::FN] = mfma32(cur.b[j % H::FN], cur.a[j / H::FN], acc[j / H::FN][j % H::FN]); }
            __builtin_amdgcn_sched_barrier(0);
            if (g == 0) {
                wait_copies<(H::S - 2) * H::NI>();   // step t + 1 is there, and this wave has read step t
                meet();                              // and everyone's: step t's place is free
            } else {
#pragma unroll
                for (int j = (g - 1) * RD / RG; j < g * RD / RG; ++j) { if (j < H::FN) { read_b(nxt, j); } else { read_a(nxt, j - H::FN); } }
#pragma unroll
                for (int j = 0; j < H::NI; ++j) {   // copy j: its address, a group later the copy
                    if ((j + 1) * (RG - 1) / H::NI == g) { set(j, here); }
                    if ((j + 1) * (RG - 1) / H::NI == g - 1) { copy(j); }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        slot = slot + 1 == H::S ? 0 : slot + 1;
        here = lds + (uint32_t) (slot * H::STAGE);
        at_slot((uint32_t) ((slot + 1 == H::S ? 0 : slot + 1) * H::STAGE));
        begin(t + H::S + 1);
#pragma unroll
        for (int j = (RG + 1) * MF / G; j < MF; ++j) { acc[j / H::FN][j % H::FN] = mfma32(cur.b[j % H::FN], cur.a[j / H::FN], acc[j / H::FN][j % H::FN]); }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < H::FM; ++i) {
#pragma unroll
        for (int j = 0; j < H::FN; ++j) { acc[i][j] = (f32x4) { 0.f, 0.f, 0.f, 0.f }; }
    }
    for (int t = 0; t < H::S; ++t) {
        begin(t);
#pragma unroll
        for (int j = 0; j < H::NI; ++j) { set(j, lds + (uint32_t) (t * H::STAGE)); __asm__ volatile("s_nop 0"); copy(j); }
    }
    Frags<H> f0, f1;
    wait_copies<(H::S - 1) * H::NI>();
    meet();
    at_slot(0);
#pragma unroll
    for (int j = 0; j < H::FN; ++j) { read_b(f0, j); }
#pragma unroll
    for (int j = 0; j < H::FM; ++j) { read_a(f0, j); }
    at_slot(H::STAGE);
    begin(H::S);
    for (int t = 0; t < steps; t += 2) {   // (an odd number of steps: one more, of zeros)
        step(f0, f1, t);
        step(f1, f0, t + 1);
    }
    wait_copies<0>();   // nothing is written to LDS after the tile
    meet();
}

// 8 results next to each other in a row: lane (r, g) of fragments j and j + 1 gets row r, columns 16 (g % 2) + 8 (g / 2) .. + 7 of the 32
__device__ __forceinline__ void eight(f32x4 a, f32x4 b, float (&v)[8]) {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = a[i], o = b[i];   // (a bit cast of a vector's element would take the first)
        const auto q = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, p), __builtin_bit_cast(uint32_t, o), false, false);
        v[i] = __builtin_bit_cast(float, (uint32_t) q[0]); v[4 + i] = __builtin_bit_cast(float, (uint32_t) q[1]);
    }
#endif
}
template <class T> __device__ __forceinline__ void put8(T * p, const float (&v)[8]) {
    V8<T> u;
#pragma unroll
    for (int i = 0; i < 8; ++i) { u[i] = (T) v[i]; }
    *(LK_GLOBAL V8<T> *) p = u;
}
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

// the range [first, last) of tiles of this workgroup's XCD (workgroups go round the 8 XCDs), and where it begins in it
struct Share { int first, last, step; };
__device__ __forceinline__ Share share_of(int tiles) {
    const int x = blockIdx.x % 8, per = gridDim.x / 8;   // (the grid is a multiple of 8)
    return { (int) ((int64_t) tiles * x / 8) + (int) blockIdx.x / 8, (int) ((int64_t) tiles * (x + 1) / 8), per };
}

// ---------------------------------------------------------------- forward
// GATED: of a wave's columns of the tile the first half are W's rows, the second the same rows of W2
template <class T, int ACT, bool GATED, class H> __global__ void __launch_bounds__(H::threads) k_mm(MatmulArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    __shared__ Tiles tiles;
    constexpr int CN = GATED ? H::BN / 2 : H::BN, WC = CN / H::WN;   // result columns of a tile, of a wave
    const int nt = (a.R + CN - 1) / CN;
    count_tiles(tiles, a.offsets, a.n, a.n_exp, H::BM);
    const Share sh = share_of(uni(tiles.first[NEXP_MAX]) * nt);
    const uint32_t lds = lds_addr(dyn);
    const int wave = uni(threadIdx.x >> 6), lane = lane_id(), wm = wave / H::WN, wn = wave % H::WN;
    const RowLane row;
    for (int i = sh.first; i < sh.last; i += sh.step) {
        const Spot s = spot_of(tiles, a.offsets, a.n, nt, H::BM, CN, 4, i);
        uint32_t va[H::IA], vb[H::IB];
#pragma unroll
        for (int j = 0; j < H::IA; ++j) {
            const int m = piece<H::AB, H::IA>(wave, j) * 16 + (lane >> 2);
            uint32_t r = (uint32_t) m;
            bool ok = m < s.nm;
            if (a.perm && ok) { r = pair_row((uint32_t) a.perm[s.slot + m], a.magic); ok = r < (uint32_t) a.xrows; }
            va[j] = ok ? r * (uint32_t) a.K * 2 + row.chunk * 16 : FAR;
        }
#pragma unroll
        for (int j = 0; j < H::IB; ++j) {
            const int rr = piece<H::BB, H::IB>(wave, j) * 16 + (lane >> 2);
            const int c = GATED ? rr / (2 * WC) * WC + rr % WC : rr;
            vb[j] = s.n0 + c < a.R ? (uint32_t) c * (uint32_t) a.K * 2 + row.chunk * 16 : FAR;
        }
        const size_t w0 = ((size_t) s.e * a.R + s.n0) * a.K;
        const uint64_t pa = uni64((const T *) a.x + (a.perm ? 0 : (size_t) s.slot * a.K)), pb = uni64((const T *) a.W + w0), pb2 = GATED ? uni64((const T *) a.W2 + w0) : 0;
        f32x4 acc[H::FM][H::FN];
        u32x4 ba, bb, bb2;
        uint32_t dst, voff;
        bool in = true;   // the lane's chunk of the step is there (a branch for the last step costs registers, this one instruction a copy)
        sums<T, false, false, H>(acc, lds, (a.K + BK - 1) / BK, [&](int t) {
            const int left = a.K - t * BK;   // terms from this step on
            const uint32_t bytes = left > 0 ? WINDOW : 0;
            const uint64_t off = (uint64_t) (uint32_t) t * (BK * 2);
            ba = buffer(pa + off, bytes); bb = buffer(pb + off, bytes); bb2 = buffer(pb2 + off, bytes);
            in = left >= BK || (int) row.chunk * 8 < left;
        }, [&](int j, uint32_t at) {
            dst = copy_to(at, j < H::IA ? (uint32_t) (piece<H::AB, H::IA>(wave, j) * 1024) : (uint32_t) (H::AB + piece<H::BB, H::IB>(wave, j - H::IA) * 1024));
            voff = in ? j < H::IA ? va[j] : vb[j - H::IA] : FAR;
            __asm__ volatile("" : "+v"(voff));
        }, [&](int j) { copy16(dst, voff, j < H::IA ? ba : GATED && piece<H::BB, H::IB>(wave, j - H::IA) * 16 % (2 * WC) >= WC ? bb2 : bb); });
        constexpr int FC = GATED ? H::FN / 2 : H::FN;
#pragma unroll
        for (int m = 0; m < H::FM; ++m) {
            const int sr = (wm * H::FM + m) * 16 + (lane & 15);
#pragma unroll
            for (int j = 0; j < FC; j += 2) {
                const int c = s.n0 + wn * WC + 16 * (j + ((lane >> 4) & 1)) + 8 * (lane >> 5);
                float z[8], y[8], z2[8];
                eight(acc[m][j], acc[m][j + 1], z);
                if (GATED) { eight(acc[m][FC + j], acc[m][FC + j + 1], z2); }
                if (sr >= s.nm || c >= a.R) { continue; }
                const size_t at = (size_t) (s.slot + sr) * a.R + c;
                if (a.bias) { add8(a.bias + (size_t) s.e * a.R + c, z); }
#pragma unroll
                for (int u = 0; u < 8; ++u) { y[u] = act_fn<ACT>(z[u]); if (GATED) { y[u] *= z2[u]; } }
                if (a.residual) { add8((const T *) a.residual + at, y); }
                if (a.y_f32) { put8((float *) a.y + at, y); } else { put8((T *) a.y + at, y); }
                if (a.z) { put8((T *) a.z + at, z); }
                if (GATED && a.z2) { put8((T *) a.z2 + at, z2); }
            }
        }
    }
}

// ---------------------------------------------------------------- dx
template <class T, class H> __global__ void __launch_bounds__(H::threads) k_mm_dx(MatmulGradArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    __shared__ Tiles tiles;
    const int nt = (a.K + H::BN - 1) / H::BN;
    count_tiles(tiles, a.offsets, a.n, a.n_exp, H::BM);
    const Share sh = share_of(uni(tiles.first[NEXP_MAX]) * nt);
    const uint32_t lds = lds_addr(dyn);
    const int wave = uni(threadIdx.x >> 6), lane = lane_id(), wm = wave / H::WN, wn = wave % H::WN;
    const RowLane row;
    const int half = (a.R + BK - 1) / BK, steps = a.dz2 ? 2 * half : half;
    for (int i = sh.first; i < sh.last; i += sh.step) {
        const Spot s = spot_of(tiles, a.offsets, a.n, nt, H::BM, H::BN, 4, i);
        uint32_t va[H::IA], vb[H::IB];
#pragma unroll
        for (int j = 0; j < H::IA; ++j) {
            const int m = piece<H::AB, H::IA>(wave, j) * 16 + (lane >> 2);
            va[j] = m < s.nm ? (uint32_t) m * (uint32_t) a.R * 2 + row.chunk * 16 : FAR;
        }
#pragma unroll
        for (int j = 0; j < H::IB; ++j) {
            const int p = piece<H::BB, H::IB>(wave, j), c = ColLane<H::BN>::column(p);
            vb[j] = s.n0 + c < a.K ? (uint32_t) ColLane<H::BN>::term(p) * (uint32_t) a.K * 2 + (uint32_t) c * 2 : FAR;
        }
        const size_t a0 = (size_t) s.slot * a.R, w0 = (size_t) s.e * a.R * a.K + s.n0;
        const uint64_t pa = uni64((const T *) a.dz + a0), pb = uni64((const T *) a.W + w0);
        const uint64_t pa2 = a.dz2 ? uni64((const T *) a.dz2 + a0) : 0, pb2 = a.dz2 ? uni64((const T *) a.W2 + w0) : 0;
        f32x4 acc[H::FM][H::FN];
        u32x4 ba, bb;
        uint32_t dst, voff;
        bool in = true;
        sums<T, false, true, H>(acc, lds, steps, [&](int t) {
            const bool second = t >= half;   // (t < steps: the second pair's)
            const int u = second ? t - half : t, left = t < steps ? a.R - u * BK : 0;
            ba = buffer((second ? pa2 : pa) + (uint64_t) (uint32_t) u * (BK * 2), left > 0 ? WINDOW : 0);
            bb = buffer((second ? pb2 : pb) + (uint64_t) (uint32_t) u * ((uint64_t) (uint32_t) a.K * (BK * 2)),   // the range ends with the last term's row
                        left > 0 ? (uint32_t) min(left, BK) * (uint32_t) a.K * 2 - (uint32_t) s.n0 * 2 : 0);
            in = left >= BK || (int) row.chunk * 8 < left;
        }, [&](int j, uint32_t at) {
            dst = copy_to(at, j < H::IA ? (uint32_t) (piece<H::AB, H::IA>(wave, j) * 1024) : (uint32_t) (H::AB + piece<H::BB, H::IB>(wave, j - H::IA) * 1024));
            voff = j < H::IA ? in ? va[j] : FAR : vb[j - H::IA];
            __asm__ volatile("" : "+v"(voff));
        }, [&](int j) { copy16(dst, voff, j < H::IA ? ba : bb); });
#pragma unroll
        for (int m = 0; m < H::FM; ++m) {
            const int sr = (wm * H::FM + m) * 16 + (lane & 15);
#pragma unroll
            for (int j = 0; j < H::FN; j += 2) {
                const int c = s.n0 + (wn * H::FN + j + ((lane >> 4) & 1)) * 16 + 8 * (lane >> 5);
                float v[8];
                eight(acc[m][j], acc[m][j + 1], v);
                if (sr < s.nm && c < a.K) { put8((T *) a.dx + (size_t) (s.slot + sr) * a.K + c, v); }
            }
        }
    }
}

// ---------------------------------------------------------------- dW
// one workgroup a tile: [second][expert][m-tile band][n][m]
template <class T, bool F32, bool PERM, class H> __global__ void __launch_bounds__(H::threads) k_mm_dw(MatmulGradArgs a, int mt, int nt) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    const uint32_t lds = lds_addr(dyn);
    const int wave = uni(threadIdx.x >> 6), lane = lane_id(), wm = wave / H::WN, wn = wave % H::WN;
    const int all = (int) gridDim.x, b = (int) ((int64_t) all / 8 * (blockIdx.x % 8) + min((int) blockIdx.x % 8, all % 8)) + (int) blockIdx.x / 8;   // an XCD's share is a run
    const int per = mt * nt, which = b / per, e = which % a.n_exp, in = b % per;
    const bool second = which >= a.n_exp ? true : a.dW == nullptr;
    const Span sp = span_of(a.offsets, a.n, e);
    const int begin = uni(sp.begin), len = uni(sp.end) - begin, m0 = in % mt * H::BM, n0 = in / mt * H::BN;
    const T * dz = (const T *) (second ? a.dz2 : a.dz) + (size_t) begin * a.R + m0;
    uint32_t va[H::IA], vb[H::IB];
#pragma unroll
    for (int j = 0; j < H::IA; ++j) {
        const int p = piece<H::AB, H::IA>(wave, j), c = ColLane<H::BM>::column(p);
        va[j] = m0 + c < a.R ? (uint32_t) ColLane<H::BM>::term(p) * (uint32_t) a.R * 2 + (uint32_t) c * 2 : FAR;
    }
#pragma unroll
    for (int j = 0; j < H::IB; ++j) {
        const int p = piece<H::BB, H::IB>(wave, j), c = ColLane<H::BN>::column(p);
        vb[j] = n0 + c < a.K ? (PERM ? 0 : (uint32_t) ColLane<H::BN>::term(p) * (uint32_t) a.K * 2) + (uint32_t) c * 2 : FAR;
    }
    const uint64_t pa = uni64(dz), pb = uni64((const T *) a.x + (PERM ? 0 : (size_t) begin * a.K) + n0);
    f32x4 acc[H::FM][H::FN];
    u32x4 ba, bb;
    uint32_t dst, voff;
    constexpr int Q = ColLane<H::BN>::TERMS, NR = PERM ? H::IB * Q : 1;
    int pair[NR];        // PERM: the next step's pairs of this wave's copies, by scalar loads
    uint32_t off[NR];    // and the step's rows, as offsets
    auto load_pairs = [&](int t) {
#pragma unroll
        for (int j = 0; j < H::IB; ++j) {
#pragma unroll
            for (int q = 0; q < Q; ++q) {   // (past the end: its last one again, or any)
                const int i = min(t * BK + piece<H::BB, H::IB>(wave, j) * Q + q, len - 1);
                pair[j * Q + q] = ((const LK_CONST int *) a.perm)[uni(max(begin + i, 0))];
            }
        }
    };
    if constexpr (PERM) { load_pairs(0); }
    sums<T, true, true, H>(acc, lds, (len + BK - 1) / BK, [&](int t) {   // (what lies behind the last slot is outside the buffer)
        const int left = len - t * BK;
        ba = buffer(pa + (uint64_t) (uint32_t) t * ((uint64_t) (uint32_t) a.R * (BK * 2)), left > 0 ? (uint32_t) min(left, BK) * (uint32_t) a.R * 2 - (uint32_t) m0 * 2 : 0);
        if constexpr (PERM) {
            bb = buffer(pb, WINDOW);
#pragma unroll
            for (int j = 0; j < H::IB; ++j) {
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const uint32_t r = pair_row((uint32_t) pair[j * Q + q], a.magic);
                    off[j * Q + q] = piece<H::BB, H::IB>(wave, j) * Q + q < left && r < (uint32_t) a.xrows ? r * (uint32_t) a.K * 2 : WINDOW;   // (and a column: still outside)
                }
            }
            load_pairs(t + 1);
        } else {
            bb = buffer(pb + (uint64_t) (uint32_t) t * ((uint64_t) (uint32_t) a.K * (BK * 2)), left > 0 ? (uint32_t) min(left, BK) * (uint32_t) a.K * 2 - (uint32_t) n0 * 2 : 0);
        }
    }, [&](int j, uint32_t at) {
        dst = copy_to(at, j < H::IA ? (uint32_t) (piece<H::AB, H::IA>(wave, j) * 1024) : (uint32_t) (H::AB + piece<H::BB, H::IB>(wave, j - H::IA) * 1024));
        if (j < H::IA) { voff = va[j]; }
        else {
            const int i = j - H::IA;
            voff = vb[i];
            if constexpr (PERM) {
                const int q = lane / (64 / Q);
                uint32_t o = off[i * Q];
#pragma unroll
                for (int u = 1; u < Q; ++u) { o = q == u ? off[i * Q + u] : o; }
                voff = voff == FAR ? FAR : voff + o;
            }
        }
        __asm__ volatile("" : "+v"(voff));
    }, [&](int j) { copy16(dst, voff, j < H::IA ? ba : bb); });
#pragma unroll
    for (int m = 0; m < H::FM; ++m) {
        const int r = m0 + (wm * H::FM + m) * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < H::FN; j += 2) {
            const int c = n0 + (wn * H::FN + j + ((lane >> 4) & 1)) * 16 + 8 * (lane >> 5);
            float v[8];
            eight(acc[m][j], acc[m][j + 1], v);
            if (r >= a.R || c >= a.K) { continue; }
            const size_t at = ((size_t) e * a.R + r) * a.K + c;
            if (F32) { float * d = (float *) (second ? a.dW2 : a.dW) + at; if (a.accumulate) { add8(d, v); } put8(d, v); }
            else { T * d = (T *) (second ? a.dW2 : a.dW) + at; if (a.accumulate) { add8(d, v); } put8(d, v); }
        }
    }
}

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int CUS = 256;
// m-tiles of `bm` slots at most
int64_t most_tiles(int n, int n_exp, bool groups, int bm) { return ceil_div(n, bm) + (groups ? n_exp : 0); }
unsigned grid_of(int64_t tiles, int per_cu) { return (unsigned) std::min<int64_t>(CUS * per_cu, ceil_div(tiles, 8) * 8); }

template <class T, int ACT, bool GATED, class H> hipError_t fwd(const MatmulArgs & a, hipStream_t st, int per_cu) {
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_mm<T, ACT, GATED, H>, H::LDS)) { return e; }
    const int64_t tiles = most_tiles(a.n, a.n_exp, a.offsets, H::BM) * ceil_div(a.R, GATED ? H::BN / 2 : H::BN);
    k_mm<T, ACT, GATED, H><<<grid_of(tiles, per_cu), H::threads, H::LDS, st>>>(a);
    return hipGetLastError();
}
template <class T, int ACT, bool GATED> hipError_t fwd(const MatmulArgs & a, hipStream_t st) {
    const int per = a.n / a.n_exp;
    if (per > 96) { return fwd<T, ACT, GATED, Shape<T, false, false, 256, 256, 2, 2, 4>>(a, st, 1); }
    return fwd<T, ACT, GATED, Shape<T, false, false, 64, 128, 2, 2, 4>>(a, st, 3);
}
template <class T> hipError_t fwd(const MatmulArgs & a, hipStream_t st) {
    if (a.W2) { return a.act == ACT_SILU ? fwd<T, ACT_SILU, true>(a, st) : a.act == ACT_GELU ? fwd<T, ACT_GELU, true>(a, st) : fwd<T, ACT_NONE, true>(a, st); }
    return a.act == ACT_SILU ? fwd<T, ACT_SILU, false>(a, st) : a.act == ACT_GELU ? fwd<T, ACT_GELU, false>(a, st) : fwd<T, ACT_NONE, false>(a, st);
}
template <class T, class H> hipError_t dx(const MatmulGradArgs & a, hipStream_t st, int per_cu) {
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_mm_dx<T, H>, H::LDS)) { return e; }
    k_mm_dx<T, H><<<grid_of(most_tiles(a.n, a.n_exp, a.offsets, H::BM) * ceil_div(a.K, H::BN), per_cu), H::threads, H::LDS, st>>>(a);
    return hipGetLastError();
}
template <class T> hipError_t dx(const MatmulGradArgs & a, hipStream_t st) {
    if (a.n / a.n_exp > 96) { return dx<T, Shape<T, false, true, 256, 256, 2, 2, 4>>(a, st, 1); }
    return dx<T, Shape<T, false, true, 64, 128, 2, 2, 4>>(a, st, 3);
}
template <class T, bool F32, bool PERM, class H> hipError_t dw(const MatmulGradArgs & a, hipStream_t st) {
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_mm_dw<T, F32, PERM, H>, H::LDS)) { return e; }
    const int mt = (int) ceil_div(a.R, H::BM), nt = (int) ceil_div(a.K, H::BN);
    k_mm_dw<T, F32, PERM, H><<<(unsigned) (mt * nt * a.n_exp * ((a.dW ? 1 : 0) + (a.dW2 ? 1 : 0))), H::threads, H::LDS, st>>>(a, mt, nt);
    return hipGetLastError();
}
template <class T, bool F32, bool PERM> hipError_t dw(const MatmulGradArgs & a, hipStream_t st) {
    if ((int64_t) a.R * a.K * a.n_exp >= (int64_t) 192 * 256 * 256) { return dw<T, F32, PERM, Shape<T, true, true, 256, 256, 2, 2, 4>>(a, st); }
    return dw<T, F32, PERM, Shape<T, true, true, 128, 128, 2, 2, 4>>(a, st);
}
template <class T, bool F32> hipError_t dw(const MatmulGradArgs & a, hipStream_t st) { return a.perm && a.n > 0 ? dw<T, F32, true>(a, st) : dw<T, F32, false>(a, st); }

}  // namespace

hipError_t launch_matmul(const MatmulArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? fwd<__bf16>(a, st) : fwd<_Float16>(a, st); }
hipError_t launch_matmul_dx(const MatmulGradArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? dx<__bf16>(a, st) : dx<_Float16>(a, st); }
hipError_t launch_matmul_dw(const MatmulGradArgs & a, hipStream_t st) {
    if (a.dw_f32) { return a.type == TYPE_BF16 ? dw<__bf16, true>(a, st) : dw<_Float16, true>(a, st); }
    return a.type == TYPE_BF16 ? dw<__bf16, false>(a, st) : dw<_Float16, false>(a, st);
}

}  // namespace lk
