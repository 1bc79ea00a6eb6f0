// matmul.hip -- products of bfloat16 / float16 matrices, dense or grouped by expert, and their backward pass.
//
//   forward  y[s][r]     = sum_k x[row(s)][k] W[e][r][k], with an epilogue     s: expert e's slots
//   dx       dx[s][k]    = sum_r dz[s][r] W[e][r][k] (+ dz2 W2)
//   dW       dW[e][r][k] = sum over e's slots of dz[s][r] x[row(s)][k]
//
// All three are D[m][n] = sum_k A[m][k] B[n][k] with D's rows along n in memory. The matrix cores take B as their first operand, so that a
// lane's four results lie next to each other in a row of D.
//
// A workgroup takes tiles of BM x BN, BK = 64 of the sum's terms a round, in two halves of 32 (a product instruction's). A round's operands
// are copied straight into LDS, 16 bytes a lane, A into a ring of SA rounds and B into one of SB; what lies outside an operand is not
// read and arrives as 0 (the buffer's range), so that no row of another expert, infinite or not, takes part. While a half's products run,
// the next half's operands go from LDS into the other set of registers. One barrier a round.
//
// In LDS an operand whose terms are next to each other in memory ("row" operand) has 128 bytes a row, chunk c of 16 at c ^ (row / 2 % 8): a
// ds_read_b128 is served in passes of 16 lanes (0-3, 12-15, 20-23, 24-27; 4-11, 16-19, 28-31; and 32 on), and each pass has 16 different
// bank quads. (Rows of 64 bytes, 32 terms a round, ask the L2 for half lines: its requests were twice as many.) One whose terms are rows
// of memory ("col" operand) has a row a term, segments of 32 bytes at segment ^ (term % 4 + term / 8 % 2 * 4), and is transposed by
// ds_read_b64_tr_b16: 16 lanes read 4 terms x 16 columns and each gets its column's 4.
#include "matmul_device.h"

namespace lk {
namespace {

constexpr int BK = 64;
constexpr uint32_t FAR = 0xFFFF0000u, WINDOW = 0xFFFE0000u;   // an offset outside every buffer; the largest range of one

// one copy instruction: 16 bytes a lane to `to` + 16 * lane; nothing of it is known to the compiler, which would wait for all copies
// before each ds_read_b64_tr_b16: the waits below are counted by hand
struct Place { uint32_t base, off; };   // two scalars, added on the way into m0
__device__ __forceinline__ void copy16(Place to, uint32_t voff, u32x4 rsrc) {
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" :: "s"(to.base), "s"(to.off), "v"(voff), "s"(rsrc) : "memory", "scc");   // (m0 is reserved: the compiler keeps nothing in it)
#endif
}
template <int N> __device__ __forceinline__ void wait_copies() {   // all but the last N, and all LDS reads
    static_assert(N >= 0 && N < 64, "vmcnt");
    __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
}
__device__ __forceinline__ void meet() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}
__device__ __forceinline__ u32x4 buffer(uint64_t base, uint32_t bytes) { return (u32x4) { (uint32_t) base, (uint32_t) (base >> 32) & 0xFFFFu, bytes, 0x00020000u }; }
// a row operand's lane: of a piece of 8 rows it copies chunk(piece) of row lane / 8; it reads row lane % 16, chunk lane / 16 (second half: ^ 64)
struct RowLane {
    uint32_t read;
    __device__ __forceinline__ RowLane() {
        const int l = lane_id();
        read = (uint32_t) ((l & 15) * 128 + (((l >> 4) ^ ((l >> 1) & 7)) * 16));
    }
    __device__ __forceinline__ static uint32_t chunk(int piece) { return (uint32_t) ((lane_id() & 7) ^ ((4 * piece + (lane_id() >> 4)) & 7)); }
};
// a col operand's: of a piece of 1024 bytes = 512 / COLS terms
template <int COLS> struct ColLane {
    static constexpr int TERMS = 512 / COLS;   // terms a piece holds
    __device__ __forceinline__ static int term(int j) { return j * TERMS + lane_id() / (COLS / 8); }
    __device__ __forceinline__ static int column(int j) {   // first of the 8 columns it copies
        const int k = term(j), p = lane_id() % (COLS / 8);
        return 8 * ((((p >> 1) ^ swz(k)) << 1) | (p & 1));
    }
    __device__ __forceinline__ static int swz(int k) { return (k & 3) | ((k >> 1) & 4); }
    // the address of columns 16 j .. 16 j + 15 (j = 0 .. 7, + 8 i: + 256 i bytes), terms 8 (lane / 16) .. + 3; + 4 and + 32: so many rows
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
struct Spot { int e, slot, nm, n0; };   // expert, first slot, its slots in the tile, first column
// the sum's part of work item i: parts come one after the other, each with all tiles; rounds d0 .. d0 + rounds - 1
struct Part { int tile, part, d0, rounds; };
__device__ __forceinline__ Part part_of(int i, int tiles, int parts, int rounds) {
    const int p = parts > 1 ? uni(i / tiles) : 0, d0 = parts > 1 ? uni(rounds * p / parts) : 0;   // (at most 2^15 rounds, 16 parts)
    return { i - p * tiles, p, d0, (parts > 1 ? uni(rounds * (p + 1) / parts) : rounds) - d0 };
}
// tile i of the launch, i < all * nt: an expert's tiles are next to each other, in bands of `band` m-tiles, m fastest
__device__ __forceinline__ Spot spot_of(const Tiles & t, const int * offsets, int n, int nt, int bm, int bn, int band, int i) {
    Spot s;
    s.e = t.expert(i / nt);   // (before(e) * nt <= i exactly when before(e) <= i / nt)
    const Span sp = span_of(offsets, n, s.e);
    const int f = t.before(s.e), mt = t.before(s.e + 1) - f, in = i - f * nt, b = in / (band * nt), rows = min(band, mt - b * band), r = in - b * band * nt;
    s.slot = uni(sp.begin + (b * band + r % rows) * bm);
    s.nm = uni(min(bm, sp.end - s.slot));
    s.n0 = uni(r / rows * bn);
    return s;
}

// ---------------------------------------------------------------- a tile's sums
// 4 waves. A: m side, B: n side. PER_CU workgroups a CU
template <int BM_, int BN_, int SA_, int SB_, int PER_CU_> struct Shape {
    static constexpr int BM = BM_, BN = BN_, SA = SA_, SB = SB_, PER_CU = PER_CU_, NW = 4;
    static constexpr int AB = BM * BK * 2, BB = BN * BK * 2, LB = SA * AB, LDS = LB + SB * BB;   // a round's bytes; B's place
    static constexpr int CA = AB / 1024 < NW ? 1 : AB / 1024 / NW, CB = BB / 1024 < NW ? 1 : BB / 1024 / NW;   // copies a wave and round
    static constexpr int threads = 64 * NW;
};
// how the waves share a tile's first ROWS rows: WM x 4 / WM of them, FM x FN fragments of 16 x 16 each. A tile that is not full takes the one
// of as few rows as hold it (an expert's last tile: 256 experts of 256 slots on average leave a third of their rows empty)
template <class H, int ROWS_, int WM_> struct Waves {
    static constexpr int ROWS = ROWS_, WM = WM_, WN = H::NW / WM, FM = ROWS / WM / 16, FN = H::BN / WN / 16;
};
template <class T, class V> struct Frags { V8<T> a[V::FM], b[V::FN]; };

// which of an operand's 1024-byte pieces copy i of wave w takes (fewer pieces than waves: some copy the same one)
template <int BYTES, int I> __device__ __forceinline__ int piece(int w, int i) { return (w * I + i) % (BYTES / 1024); }

// The loop over the sum's rounds. `c` copies: c.begin_a(d) and then c.set_a(j, address), c.copy_a(j) for j = 0 .. CA - 1 copy A's round d, _b
// B's; they are called for rounds past the end too, and then copy nothing (zeros). start() comes before.
// A wave has its SIMD to itself, and its products (16 cycles each) follow each other without a gap only if no more than three other
// instructions go between two of them: the copies and reads are dealt out among the products in this order, and what comes next is
// prepared in scalars and addresses among the last ones. In a round's first half A of round d + SA - 1 is copied, in its second B of round
// d + SB, behind the barrier that comes after the half's first product: it says that round d + 1 is there and that round d's last half is
// in registers.
// a tile's first copies, before run(): A of rounds 0 .. SA - 2, B of 0 .. SB - 1
template <class H, class Copies> __device__ __forceinline__ void start(Copies & c, uint32_t lds) {
#pragma unroll
    for (int d = 0; d < (H::SA - 1 > H::SB ? H::SA - 1 : H::SB); ++d) {
        if (d < H::SA - 1) {
            c.begin_a(d);
#pragma unroll
            for (int j = 0; j < H::CA; ++j) { c.set_a(j, lds + (uint32_t) (d * H::AB)); c.copy_a(j); }
        }
        if (d < H::SB) {
            c.begin_b(d);
#pragma unroll
            for (int j = 0; j < H::CB; ++j) { c.set_b(j, lds + (uint32_t) (H::LB + d * H::BB)); c.copy_b(j); }
        }
    }
}
template <class T, bool AC, bool BC, class H, class V, class Copies> struct Sums {
    static constexpr int FM = V::FM, FN = V::FN, RA = AC ? (FM < 8 ? FM : 8) : 2, RB = BC ? (FN < 8 ? FN : 8) : 2;
    static_assert(!AC || (FM & (FM - 1)) == 0, "addresses of a col operand"); static_assert(!BC || (FN & (FN - 1)) == 0, "addresses of a col operand");
    typedef Frags<T, V> F;
    uint32_t lds, ra[RA], rb[RB];   // a lane's addresses in a round
    __device__ __forceinline__ Sums(uint32_t lds_) : lds(lds_) {
        const int wave = uni((int) threadIdx.x >> 6), wm = wave / V::WN, wn = wave % V::WN;
        const RowLane row;
#pragma unroll
        for (int j = 0; j < RA; ++j) {
            if constexpr (AC) { ra[j] = ColLane<H::BM>::read(wm * FM + j) + (uint32_t) ((wm * FM + j) / 8 * 256) + lds; }
            else { ra[j] = (row.read ^ (uint32_t) (64 * j)) + (uint32_t) (wm * FM * 2048) + lds; }
        }
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            if constexpr (BC) { rb[j] = ColLane<H::BN>::read(wn * FN + j) + (uint32_t) ((wn * FN + j) / 8 * 256) + lds + H::LB; }
            else { rb[j] = (row.read ^ (uint32_t) (64 * j)) + (uint32_t) (wn * FN * 2048) + lds + H::LB; }
        }
    }
    static __device__ __forceinline__ void pin_sum(f32x4 & v) {
#if defined(__HIP_DEVICE_COMPILE__)
        __asm__ volatile("" : "+a"(v));
#endif
    }
    static __device__ __forceinline__ void pin(uint32_t & v) { __asm__("" : "+v"(v)); }   // (a register of its own, the fragments by immediate offsets)
    struct At { uint32_t a[RA], b[RB]; };
    __device__ __forceinline__ void at_round(At & at, int sa, int sb) const {
#pragma unroll
        for (int j = 0; j < RA; ++j) { at.a[j] = ra[j] + (uint32_t) (sa * H::AB); pin(at.a[j]); }
#pragma unroll
        for (int j = 0; j < RB; ++j) { at.b[j] = rb[j] + (uint32_t) (sb * H::BB); pin(at.b[j]); }
    }
    // fragment j of half h
    static __device__ __forceinline__ void read(F & f, const At & at, int h, int j) {
        if (j < FN) {
            if constexpr (BC) { f.b[j] = lds_col<T, H::BN>(at.b[j % RB] + (uint32_t) (j / RB * 256 + h * 32 * H::BN * 2)); } else { f.b[j] = lds_row<T>(at.b[h] + (uint32_t) (j * 2048)); }
        } else {
            const int i = j - FN;
            if constexpr (AC) { f.a[i] = lds_col<T, H::BM>(at.a[i % RA] + (uint32_t) (i / RA * 256 + h * 32 * H::BM * 2)); } else { f.a[i] = lds_row<T>(at.a[h] + (uint32_t) (i * 2048)); }
        }
    }
    // the products of one round that is there, in the first places
    __device__ __forceinline__ void round(f32x4 (&acc)[FM][FN]) const {
        At at;
        at_round(at, 0, 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            F f;
#pragma unroll
            for (int j = 0; j < FM + FN; ++j) { read(f, at, h, j); }
#pragma unroll
            for (int j = 0; j < FM * FN; ++j) { acc[j / FN][j % FN] = mfma32(f.b[j % FN], f.a[j / FN], acc[j / FN][j % FN]); }
        }
    }
    __device__ __forceinline__ void run(f32x4 (&acc)[FM][FN], int rounds, Copies & c) const {
        constexpr int MF = FM * FN, RD = FM + FN, RG = MF - MF / 4 - 1;   // groups of one product: the first, RG with reads and copies, the rest
        constexpr int LATER = (H::SB - 1) * H::CA + (H::SB - 2) * H::CB < (H::SA - 2) * (H::CA + H::CB) ? (H::SB - 1) * H::CA + (H::SB - 2) * H::CB : (H::SA - 2) * (H::CA + H::CB);
        static_assert(RG > H::CA && RG > H::CB, "a group between two copies");
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j) { acc[i][j] = (f32x4) { 0.f, 0.f, 0.f, 0.f }; }
        }
        F f0, f1;
        At at;
        int sa = 0, sb = 0;                  // round d's places
        auto product = [&](const F & f, int j) __attribute__((always_inline)) { acc[j / FN][j % FN] = mfma32(f.b[j % FN], f.a[j / FN], acc[j / FN][j % FN]); };
        auto half = [&](auto second, const F & cur, F & nxt, uint32_t to) __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g <= RG; ++g) {
                product(cur, g);
                __builtin_amdgcn_sched_barrier(0);
                if (g == 0) {
                    if (second) { wait_copies<LATER>(); meet(); }
                } else {
#pragma unroll
                    for (int j = (g - 1) * RD / RG; j < g * RD / RG; ++j) { read(nxt, at, second ? 0 : 1, j); }
                    constexpr int CN = decltype(second)::value ? H::CB : H::CA;
#pragma unroll
                    for (int j = 0; j < CN; ++j) {   // copy j: its lane's offset, a group later the copy
                        const int when = second && RG > 2 * CN ? 1 + 2 * j : 1 + j * (RG - 1) / CN;   // (B has a round to arrive, A more: 2 % of dx and dW)
                        if (g == when) { if (second) { c.set_b(j, to); } else { c.set_a(j, to); } }
                        if (g == when + 1) { if (second) { c.copy_b(j); } else { c.copy_a(j); } }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto rest = [&](const F & cur) __attribute__((always_inline)) {
#pragma unroll
            for (int j = RG + 1; j < MF; ++j) { product(cur, j); }
            __builtin_amdgcn_sched_barrier(0);
        };
        wait_copies<LATER + H::CB>();   // (as in the loop, B's copies of one round more are out: round 0 is there)
        meet();
        at_round(at, 0, 0);
#pragma unroll
        for (int j = 0; j < RD; ++j) { read(f0, at, 0, j); }
        c.begin_a(H::SA - 1);
        for (int d = 0; d < rounds; ++d) {
            const int pa = sa == 0 ? H::SA - 1 : sa - 1;   // round d - 1's place of A is round d + SA - 1's
            half(std::false_type(), f0, f1, lds + (uint32_t) (pa * H::AB));
            const uint32_t to = lds + (uint32_t) (H::LB + sb * H::BB);
            sa = sa + 1 == H::SA ? 0 : sa + 1;
            sb = sb + 1 == H::SB ? 0 : sb + 1;
            at_round(at, sa, sb);
            c.begin_b(d + H::SB);
            rest(f0);
            half(std::true_type(), f1, f0, to);
            c.begin_a(d + H::SA);
            rest(f1);
        }
        wait_copies<0>();   // nothing is written to LDS after the tile
        meet();
        if constexpr (FM * FN == 64) {   // the sums fill one half of the registers: what follows must not move them inside the loop
#pragma unroll
            for (int i = 0; i < FM; ++i) {
#pragma unroll
                for (int j = 0; j < FN; ++j) { pin_sum(acc[i][j]); }
            }
        }
    }
};

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
// Whole lines: x and y are 16 bytes of row r, lane (r, g), a half line each; after it lane (r, g) has 16 of rows r % 8 (up) and r % 8 + 8
// (down), x's where r < 8, y's where not
template <class V> __device__ __forceinline__ void lines(V x, V y, V & up, V & down) {
    const bool low = (lane_id() & 8) == 0;
    const u32x4 p = __builtin_bit_cast(u32x4, x), q = __builtin_bit_cast(u32x4, y);
    u32x4 u, d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t other = (uint32_t) __builtin_amdgcn_update_dpp(0, (int) (low ? q[i] : p[i]), 0x128, 0xF, 0xF, false);   // (the lane 8 further in its 16)
        u[i] = low ? p[i] : other;
        d[i] = low ? other : q[i];
    }
    up = __builtin_bit_cast(V, u);
    down = __builtin_bit_cast(V, d);
}
// The workgroups (a multiple of 8) go round the 8 XCDs; an XCD's tiles are a run of the launch's, so that what runs at a time there shares
// panels in its L2. Tiles differ in cost, so after its first a workgroup takes the XCD's next one (queue[x]); the last to find none
// sets the two counters back to 0 for the next launch.
struct Queue {
    int * next, * gone; int first, last, per;
    __device__ __forceinline__ Queue(int * queue, int tiles) {
        const int x = (int) blockIdx.x % 8;
        per = (int) gridDim.x / 8;
        next = queue + x; gone = queue + 8 + x;
        first = (int) ((int64_t) tiles * x / 8); last = (int) ((int64_t) tiles * (x + 1) / 8);
    }
    __device__ __forceinline__ int begin() const { return first + (int) blockIdx.x / 8; }
    __device__ __forceinline__ int ask() const { return threadIdx.x == 0 ? atomicAdd(next, 1) : 0; }   // (called before a tile's sums, answered by then)
    // every thread: the answer, through LDS, which nothing else uses now
    __device__ __forceinline__ int told(int asked, uint32_t lds) const {
        if (threadIdx.x == 0) { *(LK_LOCAL int *) (size_t) lds = asked; }
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        meet();
        const int v = uni(*(const LK_LOCAL int *) (size_t) lds);
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        meet();
        return first + per + v;
    }
    __device__ __forceinline__ void leave() const {
        if (threadIdx.x == 0 && atomicAdd(gone, 1) == per - 1) { *next = 0; *gone = 0; }
    }
};

// ---------------------------------------------------------------- the operands' copies
// A row operand of `rows` rows of `ld` values from base on; row r of the tile is row at(r) of it (< 0: not there). Terms 0 .. K - 1
template <class H, int BYTES, int C> struct RowCopies {
    uint64_t base; uint32_t v[C], voff; Place dst; u32x4 buf; bool in[2];
    __device__ __forceinline__ void begin(int d, int K) {
        const int left = K - d * BK;   // terms from this round on
        buf = buffer(base + (uint64_t) (uint32_t) d * (BK * 2), left > 0 ? WINDOW : 0);
        in[0] = left >= BK || (int) RowLane::chunk(0) * 8 < left;   // the lane's chunk of the round is there, in even and odd pieces
        in[1] = left >= BK || (int) RowLane::chunk(1) * 8 < left;
    }
    __device__ __forceinline__ void set(int wave, int j, uint32_t to) {
        dst = { to, (uint32_t) (piece<BYTES, C>(wave, j) * 1024) };
        voff = in[C > 1 ? j & 1 : wave & 1] ? v[j] : FAR;
        __asm__ volatile("" : "+v"(voff));
    }
    __device__ __forceinline__ void copy() const { copy16(dst, voff, buf); }
};
// a col operand's: terms are rows of `ld` values, columns from the tile's first, which is `first` in its row
template <class H, int COLS, int BYTES, int C> struct ColCopies {
    uint64_t base; uint32_t v[C], voff; Place dst; u32x4 buf;
    __device__ __forceinline__ void init(const void * p, int ld, int first) {
        base = uni64(p);
        const int wave = uni((int) threadIdx.x >> 6);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int q = piece<BYTES, C>(wave, j), c = ColLane<COLS>::column(q);
            v[j] = first + c < ld ? (uint32_t) ColLane<COLS>::term(q) * (uint32_t) ld * 2 + (uint32_t) c * 2 : FAR;
        }
    }
    __device__ __forceinline__ void begin(int d, int K, int ld, int first) {   // the range ends with the last term's row
        const int left = K - d * BK;
        buf = buffer(base + (uint64_t) (uint32_t) d * ((uint64_t) (uint32_t) ld * (BK * 2)), left > 0 ? (uint32_t) min(left, BK) * (uint32_t) ld * 2 - (uint32_t) first * 2 : 0);
    }
    __device__ __forceinline__ void set(int wave, int j, uint32_t to) {
        dst = { to, (uint32_t) (piece<BYTES, C>(wave, j) * 1024) };
        voff = v[j];
    }
    __device__ __forceinline__ void copy() const { copy16(dst, voff, buf); }
};

// f on the sharing of a tile with nm rows
template <class H, class F> __device__ __forceinline__ void by_rows(int nm, F f) {
    if constexpr (H::BM == 256) { if (nm > 128) { f(Waves<H, 256, 2>()); return; } }
    if constexpr (H::BM >= 128 && H::BN == 256) { if (nm > 64) { f(Waves<H, 128, 1>()); return; } f(Waves<H, 64, 1>()); }
    else { static_assert(H::BM == 64, "the waves of another tile"); f(Waves<H, 64, 2>()); }
}

// ---------------------------------------------------------------- forward
// GATED: of a wave's columns of the tile the first half are W's rows, the second the same rows of W2
template <class T, bool GATED, class H> struct FwdCopies {
    static constexpr int CN = GATED ? H::BN / 2 : H::BN, WC = 32;   // result columns of a tile; GATED: W's and W2's rows take turns so many at a time
    RowCopies<H, H::AB, H::CA> a; RowCopies<H, H::BB, H::CB> b; uint64_t base2; u32x4 buf2; const int K, wave;   // K: the part's terms
    // GATED: a wave's first copies are of W's pieces, the others of W2's
    static __device__ __forceinline__ int piece_b(int w, int j) {
        if (!GATED) { return piece<H::BB, H::CB>(w, j); }
        static_assert(!GATED || (H::CB % 4 == 0 && WC % 16 == 0), "half a wave's copies, of even and odd pieces in turn");
        const int q = w * (H::CB / 2) + j % (H::CB / 2);
        return q / (WC / 8) * (WC / 4) + q % (WC / 8) + (j < H::CB / 2 ? 0 : WC / 8);
    }
    __device__ __forceinline__ FwdCopies(const MatmulArgs & g, const Spot & s, const Part & p) : K(min(g.K - p.d0 * BK, p.rounds * BK)), wave(uni((int) threadIdx.x >> 6)) {
        const int lane = lane_id();
#pragma unroll
        for (int j = 0; j < H::CA; ++j) {
            const int q = piece<H::AB, H::CA>(wave, j), m = q * 8 + (lane >> 3);
            uint32_t r = (uint32_t) m;
            bool ok = m < s.nm;
            if (g.perm && ok) { r = pair_row((uint32_t) g.perm[s.slot + m], g.magic); ok = r < (uint32_t) g.xrows; }
            a.v[j] = ok ? r * (uint32_t) g.K * 2 + RowLane::chunk(q) * 16 : FAR;
        }
#pragma unroll
        for (int j = 0; j < H::CB; ++j) {
            const int q = piece_b(wave, j), rr = q * 8 + (lane >> 3), c = GATED ? rr / (2 * WC) * WC + rr % WC : rr;
            b.v[j] = s.n0 + c < g.R ? (uint32_t) c * (uint32_t) g.K * 2 + RowLane::chunk(q) * 16 : FAR;
        }
        const size_t w0 = ((size_t) s.e * g.R + s.n0) * g.K + p.d0 * BK;
        a.base = uni64((const T *) g.x + (g.perm ? 0 : (size_t) s.slot * g.K) + p.d0 * BK);
        b.base = uni64((const T *) g.W + w0);
        base2 = GATED ? uni64((const T *) g.W2 + w0) : 0;
    }
    __device__ __forceinline__ void begin_a(int d) { a.begin(d, K); }
    __device__ __forceinline__ void begin_b(int d) { b.begin(d, K); if (GATED) { buf2 = buffer(base2 + (uint64_t) (uint32_t) d * (BK * 2), b.buf[2]); } }
    __device__ __forceinline__ void set_a(int j, uint32_t to) { a.set(wave, j, to); }
    __device__ __forceinline__ void set_b(int j, uint32_t to) { b.set(wave, j, to); b.dst.off = (uint32_t) (piece_b(wave, j) * 1024); }
    __device__ __forceinline__ void copy_a(int) const { a.copy(); }
    __device__ __forceinline__ void copy_b(int j) const { if (GATED && j >= H::CB / 2) { copy16(b.dst, b.voff, buf2); } else { b.copy(); } }
};
// the epilogue of a tile's results. Addresses are the tile's (scalars) and a lane's 32-bit offset: a tile's last row is below 2^28 values away
template <class T, bool GATED, class H, class V> __device__ __forceinline__ void fwd_results(const MatmulArgs & a, const Spot & s, int part, f32x4 (&acc)[V::FM][V::FN]) {
    constexpr int FC = GATED ? V::FN / 2 : V::FN;
    const int wave = uni((int) threadIdx.x >> 6), lane = lane_id(), wm = wave / V::WN, wn = wave % V::WN;
    const size_t t0 = (size_t) s.slot * a.R + s.n0, all = (size_t) a.n * a.R;
    const int c0 = wn * FC * 16 + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5);   // the lane's first column in the tile
    auto each = [&](auto column, auto ahead, auto f) __attribute__((always_inline)) {   // column(c), ahead(m, c) and f(m, offset, z, z2) on 8 results at a time
#pragma unroll
        for (int j = 0; j < FC; j += 2) {
            const int g = GATED ? 2 * j : j, c = c0 + 16 * j;   // (W's 2 fragments, W2's 2, and so on)
            column(c);
#pragma unroll
            for (int m = 0; m < V::FM; ++m) {
                const int sr = (wm * V::FM + m) * 16 + (lane & 15);
                float z[8], z2[8];
                ahead(m, c);
                eight(acc[m][g], acc[m][g + 1], z);
                if (GATED) { eight(acc[m][g + 2], acc[m][g + 3], z2); }
                if (sr < s.nm && s.n0 + c < a.R) { f(m, (uint32_t) sr * (uint32_t) a.R + (uint32_t) c, z, z2); }
            }
        }
    };
    auto none = [](int) {};
    auto none2 = [](int, int) {};
    if (a.parts > 1) {   // (k_mm_join does the rest)
        float * p = a.part + (size_t) part * all + t0, * p2 = p + (size_t) a.parts * all;
        each(none, none2, [&](int, uint32_t at, float (&z)[8], float (&z2)[8]) __attribute__((always_inline)) { put8(p + at, z); if (GATED) { put8(p2 + at, z2); } });
        return;
    }
    const float * bias = a.bias ? a.bias + (size_t) s.e * a.R + s.n0 : nullptr;
    const T * res = a.residual ? (const T *) a.residual + t0 : nullptr;
    T * y = (T *) a.y + (a.y_f32 ? 2 * t0 : t0), * pz = a.z ? (T *) a.z + t0 : nullptr, * pz2 = GATED && a.z2 ? (T *) a.z2 + t0 : nullptr;
    if (!GATED && !bias && !res && !pz && !a.act && !a.y_f32) {
        each(none, none2, [&](int, uint32_t at, float (&z)[8], float (&)[8]) __attribute__((always_inline)) { put8(y + at, z); });
        return;
    }
    float b8[8];
    constexpr int RA = V::FM < 4 ? V::FM : 4;
    V8<T> r8[RA];   // (the residuals of 4 row groups asked for together: 8192 rows, 2048 -> 7168 318 -> 290 us, 512 -> 16384 376 -> 315; without one, short sums lost 2 to 5 %: 2755 rows, 416 -> 12504 57 -> 60)
    each([&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 8; ++u) { b8[u] = 0.f; }
        if (bias && s.n0 + c < a.R) { add8(bias + c, b8); }
    }, [&](int m0, int c) __attribute__((always_inline)) {
        if (m0 % RA == 0 && res) {
#pragma unroll
            for (int m = 0; m < RA; ++m) {   // (where there is none, the tile's first)
                const int sr = (wm * V::FM + m0 + m) * 16 + (lane & 15);
                r8[m] = *(const LK_GLOBAL V8<T> *) (res + (sr < s.nm && s.n0 + c < a.R ? (uint32_t) sr * (uint32_t) a.R + (uint32_t) c : 0u));
            }
        }
    }, [&](int m, uint32_t at, float (&z)[8], float (&z2)[8]) __attribute__((always_inline)) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) { z[u] += b8[u]; }
        activate8(a.act, z, v);
        if (GATED) {
#pragma unroll
            for (int u = 0; u < 8; ++u) { v[u] *= z2[u]; }
        }
        if (res) {
#pragma unroll
            for (int u = 0; u < 8; ++u) { v[u] += (float) r8[m % RA][u]; }
        }
        if (a.y_f32) { put8((float *) y + at, v); } else { put8(y + at, v); }
        if (pz) { put8(pz + at, z); }
        if (pz2) { put8(pz2 + at, z2); }
    });
}
template <class T, bool GATED, class H> __global__ void __launch_bounds__(H::threads, H::PER_CU * H::NW / 4) k_mm(MatmulArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    typedef FwdCopies<T, GATED, H> C;
    const int nt = (a.R + C::CN - 1) / C::CN;
    const Tiles tiles(a.offsets, a.n, a.n_exp, H::BM);
    const Queue queue(a.queue, tiles.all * nt * a.parts);
    const uint32_t lds = lds_addr(dyn);
    const int rounds = (a.K + BK - 1) / BK;
    int i = queue.begin();
    auto part = [&](int t) __attribute__((always_inline)) { return part_of(t, tiles.all * nt, a.parts, rounds); };
    auto spot = [&](const Part & p) __attribute__((always_inline)) { return spot_of(tiles, a.offsets, a.n, nt, H::BM, C::CN, 4, p.tile); };
    auto first = [&](int t) __attribute__((always_inline)) {
        if (t < queue.last) { const Part p = part(t); C c(a, spot(p), p); start<H>(c, lds); }
    };
    for (first(i); i < queue.last;) {
        const int asked = queue.ask();
        const Part p = part(i);
        const Spot s = spot(p);
        by_rows<H>(s.nm, [&](auto v) __attribute__((always_inline)) {
            typedef decltype(v) V;
            const Sums<T, false, false, H, V, C> sums(lds);
            C c(a, s, p);
            f32x4 acc[V::FM][V::FN];
            sums.run(acc, p.rounds, c);
            i = queue.told(asked, lds);
            first(i);   // the next tile's first copies are out while this one's results are written
            fwd_results<T, GATED, H, V>(a, s, p.part, acc);
        });
    }
    queue.leave();
}

// ---------------------------------------------------------------- dx
// the sum goes over dz's columns and then, with a second pair, over dz2's: rounds 0 .. half - 1 and half .. 2 half - 1
template <class T, class H> struct DxCopies {
    RowCopies<H, H::AB, H::CA> a; ColCopies<H, H::BN, H::BB, H::CB> b; uint64_t a1, a2, b1, b2; const int R, K, wave, half, d0, end, n0;
    __device__ __forceinline__ DxCopies(const MatmulGradArgs & g, const Spot & s, const Part & p) : R(g.R), K(g.K), wave(uni((int) threadIdx.x >> 6)), half((g.R + BK - 1) / BK), d0(p.d0), end(p.d0 + p.rounds), n0(s.n0) {
        const int lane = lane_id();
#pragma unroll
        for (int j = 0; j < H::CA; ++j) {
            const int q = piece<H::AB, H::CA>(wave, j), m = q * 8 + (lane >> 3);
            a.v[j] = m < s.nm ? (uint32_t) m * (uint32_t) R * 2 + RowLane::chunk(q) * 16 : FAR;
        }
        const size_t a0 = (size_t) s.slot * R, w0 = (size_t) s.e * R * K + s.n0;
        b.init((const T *) g.W + w0, K, n0);
        a1 = uni64((const T *) g.dz + a0); b1 = b.base;
        a2 = g.dz2 ? uni64((const T *) g.dz2 + a0) : a1; b2 = g.dz2 ? uni64((const T *) g.W2 + w0) : b1;
    }
    __device__ __forceinline__ void begin_a(int d) { d += d0; a.base = d < half ? a1 : a2; a.begin(d < half ? d : d - half, d < end ? R : 0); }
    __device__ __forceinline__ void begin_b(int d) { d += d0; b.base = d < half ? b1 : b2; b.begin(d < half ? d : d - half, d < end ? R : 0, K, n0); }
    __device__ __forceinline__ void set_a(int j, uint32_t to) { a.set(wave, j, to); }
    __device__ __forceinline__ void set_b(int j, uint32_t to) { b.set(wave, j, to); }
    __device__ __forceinline__ void copy_a(int) const { a.copy(); }
    __device__ __forceinline__ void copy_b(int) const { b.copy(); }
};
template <class T, class H> __global__ void __launch_bounds__(H::threads, H::PER_CU * H::NW / 4) k_mm_dx(MatmulGradArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    typedef DxCopies<T, H> C;
    const int nt = (a.K + H::BN - 1) / H::BN;
    const Tiles tiles(a.offsets, a.n, a.n_exp, H::BM);
    const Queue queue(a.queue, tiles.all * nt * a.parts);
    const uint32_t lds = lds_addr(dyn);
    const int rounds = (a.R + BK - 1) / BK * (a.dz2 ? 2 : 1);
    int i = queue.begin();
    auto part = [&](int t) __attribute__((always_inline)) { return part_of(t, tiles.all * nt, a.parts, rounds); };
    auto spot = [&](const Part & p) __attribute__((always_inline)) { return spot_of(tiles, a.offsets, a.n, nt, H::BM, H::BN, 4, p.tile); };
    auto first = [&](int t) __attribute__((always_inline)) {
        if (t < queue.last) { const Part p = part(t); C c(a, spot(p), p); start<H>(c, lds); }
    };
    for (first(i); i < queue.last;) {
        const int asked = queue.ask();
        const Part p = part(i);
        const Spot s = spot(p);
        by_rows<H>(s.nm, [&](auto v) __attribute__((always_inline)) {
            typedef decltype(v) V;
            const Sums<T, false, true, H, V, C> sums(lds);
            C c(a, s, p);
            f32x4 acc[V::FM][V::FN];
            sums.run(acc, p.rounds, c);
            i = queue.told(asked, lds);
            first(i);
            MatmulArgs r{};   // the sums alone
            r.n = a.n; r.R = a.K; r.y = a.dx; r.parts = a.parts; r.part = a.part;
            fwd_results<T, false, H, V>(r, s, p.part, acc);
        });
    }
    queue.leave();
}

// ---------------------------------------------------------------- the parts of split sums, in order, and what follows the sum
template <class T> __global__ void __launch_bounds__(256) k_mm_join(MatmulArgs a) {
    int first = 0, last = a.n;
    if (a.offsets) { first = min(max(a.offsets[0], 0), a.n); last = min(max(a.offsets[a.n_exp], 0), a.n); }
    const int64_t all = (int64_t) a.n * a.R, end = (int64_t) last * (a.R / 8);
    for (int64_t i = (int64_t) first * (a.R / 8) + (int64_t) blockIdx.x * 256 + threadIdx.x; i < end; i += (int64_t) gridDim.x * 256) {
        float z[8] = {}, z2[8] = {}, y[8];
        for (int p = 0; p < a.parts; ++p) {
            add8(a.part + p * all + 8 * i, z);
            if (a.W2) { add8(a.part + (a.parts + p) * all + 8 * i, z2); }
        }
        if (a.bias) {
            const int slot = (int) (i / (a.R / 8)), col = (int) (i % (a.R / 8)) * 8;
            int e = 0;   // the last expert whose slots begin at or before this one
            if (a.offsets) { for (int b = NEXP_MAX / 2; b > 0; b >>= 1) { if (e + b < a.n_exp && a.offsets[e + b] <= slot) { e += b; } } }
            add8(a.bias + (size_t) e * a.R + col, z);
        }
        activate8(a.act, z, y);
        if (a.W2) {
#pragma unroll
            for (int u = 0; u < 8; ++u) { y[u] *= z2[u]; }
        }
        if (a.residual) { add8((const T *) a.residual + 8 * i, y); }
        if (a.y_f32) { put8((float *) a.y + 8 * i, y); } else { put8((T *) a.y + 8 * i, y); }
        if (a.z) { put8((T *) a.z + 8 * i, z); }
        if (a.z2) { put8((T *) a.z2 + 8 * i, z2); }
    }
}

// ---------------------------------------------------------------- dW
template <class T, bool PERM, class H> struct DwCopies {
    static constexpr int Q = ColLane<H::BN>::TERMS, NR = PERM ? H::CB * Q : 1;
    ColCopies<H, H::BM, H::AB, H::CA> a; ColCopies<H, H::BN, H::BB, H::CB> b;
    int pair[NR];        // PERM: the next round's pairs of this wave's copies, by scalar loads
    uint32_t off[NR];    // and the round's rows, as offsets
    const int * perm; uint32_t magic, xrows; int R, K, m0, n0, begin, len, wave;
    __device__ __forceinline__ void init(const MatmulGradArgs & g, const void * dz, int begin_, int len_, int m0_, int n0_) {
        perm = g.perm; magic = g.magic; xrows = (uint32_t) g.xrows; R = g.R; K = g.K; m0 = m0_; n0 = n0_; begin = begin_; len = len_; wave = uni((int) threadIdx.x >> 6);
        a.init((const T *) dz + (size_t) begin * R + m0, R, m0);
        b.init((const T *) g.x + (PERM ? 0 : (size_t) begin * K) + n0, K, n0);
        if constexpr (PERM) {
#pragma unroll
            for (int j = 0; j < H::CB; ++j) { b.v[j] = b.v[j] == FAR ? FAR : (uint32_t) ColLane<H::BN>::column(piece<H::BB, H::CB>(wave, j)) * 2; }
            load_pairs(0);
        }
    }
    __device__ __forceinline__ void load_pairs(int d) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {   // (past the end: its last one again, or any)
            const int at = min(d * BK + piece<H::BB, H::CB>(wave, i / Q) * Q + i % Q, len - 1);
            pair[i] = ((const LK_CONST int *) perm)[uni(max(begin + at, 0))];
        }
    }
    __device__ __forceinline__ void begin_a(int d) { a.begin(d, len, R, m0); }
    __device__ __forceinline__ void begin_b(int d) {
        if constexpr (PERM) {
            b.buf = buffer(b.base, WINDOW);
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const uint32_t r = pair_row((uint32_t) pair[i], magic);
                off[i] = d * BK + piece<H::BB, H::CB>(wave, i / Q) * Q + i % Q < len && r < xrows ? r * (uint32_t) K * 2 : WINDOW;   // (and a column: still outside)
            }
            load_pairs(d + 1);
        } else { b.begin(d, len, K, n0); }
    }
    __device__ __forceinline__ void set_a(int j, uint32_t to) { a.set(wave, j, to); }
    __device__ __forceinline__ void set_b(int j, uint32_t to) {
        b.set(wave, j, to);
        if constexpr (PERM) {
            const int q = lane_id() / (64 / Q);
            static_assert(Q == 2 || Q == 4, "tiles of 256 or 128 columns");
            uint32_t o = off[j * Q];
#pragma unroll
            for (int u = 1; u < Q; ++u) {
                uint32_t w = off[j * Q + u];
                __asm__("" : "+s"(w));   // (else the choice becomes an indexed load from scratch memory)
                o = q == u ? w : o;
            }
            b.voff = b.voff == FAR ? FAR : b.voff + o;
            __asm__ volatile("" : "+v"(b.voff));
        }
    }
    __device__ __forceinline__ void copy_a(int) const { a.copy(); }
    __device__ __forceinline__ void copy_b(int) const { b.copy(); }
};
// tile i of the launch: [matrix][expert][band of m-tiles][n][m of the band]; a part is a run of the expert's rounds
struct DwSpot { int e, begin, len, m0, n0, part; bool second; };
template <class H> __device__ __forceinline__ DwSpot dw_spot(const MatmulGradArgs & a, int i) {
    constexpr int BAND = 4;
    const int mt = (a.R + H::BM - 1) / H::BM, nt = (a.K + H::BN - 1) / H::BN, per = mt * nt, all = per * a.n_exp * ((a.dW ? 1 : 0) + (a.dW2 ? 1 : 0));
    DwSpot s;
    s.part = a.dw_parts > 1 ? uni(i / all) : 0;
    i -= s.part * all;
    const int which = uni(i / per), in = i - which * per, band = in / (BAND * nt), rows = min(BAND, mt - band * BAND), r = in - band * BAND * nt;
    s.e = uni(which % a.n_exp);
    s.second = which >= a.n_exp || !a.dW;
    const Span sp = span_of(a.offsets, a.n, s.e);
    s.begin = uni(sp.begin); s.len = uni(sp.end) - s.begin;
    if (a.dw_parts > 1) {
        const int rounds = (s.len + BK - 1) / BK, d0 = uni((int) ((int64_t) rounds * s.part / a.dw_parts)), d1 = uni((int) ((int64_t) rounds * (s.part + 1) / a.dw_parts));
        s.begin += d0 * BK; s.len = min(s.len - d0 * BK, (d1 - d0) * BK);
    }
    s.m0 = uni((band * BAND + r % rows) * H::BM); s.n0 = uni(r / rows * H::BN);
    return s;
}
// the results of a tile, past the caches that the operands live in and in whole lines (64 experts of 94 rows, 2 x 1024 x 2048, with dx 355 -> 325 us;
// half lines 336 us, but 256 of 128, 7168 x 2048, 4.3 -> 4.6 ms)
template <class T, bool F32, class V> __device__ __forceinline__ void dw_results(const MatmulGradArgs & a, const DwSpot & s, f32x4 (&acc)[V::FM][V::FN]) {
    const int wave = uni((int) threadIdx.x >> 6), lane = lane_id(), wm = wave / V::WN, wn = wave % V::WN;
    const size_t w = (size_t) a.R * a.K, t0 = (size_t) s.e * w + (size_t) s.m0 * a.K + s.n0;
    // f(offset, columns' 16 bytes) on whole lines: of float, or of T
    auto floats = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < V::FM; ++m) {
            const int row = (wm * V::FM + m) * 16 + (lane & 7);
#pragma unroll
            for (int j = 0; j < V::FN; j += 2) {
                const int col = (wn * V::FN + j + ((lane >> 3) & 1)) * 16 + 4 * (lane >> 4);
                f32x4 up, down;
                lines(acc[m][j], acc[m][j + 1], up, down);
                const uint32_t at = (uint32_t) row * (uint32_t) a.K + (uint32_t) col;
                if (s.n0 + col < a.K) {
                    if (s.m0 + row < a.R) { f(at, up); }
                    if (s.m0 + row + 8 < a.R) { f(at + 8 * (uint32_t) a.K, down); }
                }
            }
        }
    };
    auto halves = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < V::FM; ++m) {
            const int row = (wm * V::FM + m) * 16 + (lane & 7);
#pragma unroll
            for (int j = 0; j < V::FN; j += 4) {
                const int col = (wn * V::FN + j + ((lane >> 4) & 1) + ((lane >> 2) & 2)) * 16 + 8 * (lane >> 5);
                float v[8], w[8];
                eight(acc[m][j], acc[m][j + 1], v);
                eight(acc[m][j + 2], acc[m][j + 3], w);
                V8<T> up, down;
                lines(rounded<T>(v), rounded<T>(w), up, down);
                const uint32_t at = (uint32_t) row * (uint32_t) a.K + (uint32_t) col;
                if (s.n0 + col < a.K) {
                    if (s.m0 + row < a.R) { f(at, up); }
                    if (s.m0 + row + 8 < a.R) { f(at + 8 * (uint32_t) a.K, down); }
                }
            }
        }
    };
    if (a.dw_parts > 1) {
        float * p = a.dw_part + ((size_t) s.part * ((a.dW ? 1 : 0) + (a.dW2 ? 1 : 0)) + (a.dW && s.second ? 1 : 0)) * a.n_exp * w + t0;
        floats([&](uint32_t at, f32x4 v) __attribute__((always_inline)) { *(LK_GLOBAL f32x4 *) (p + at) = v; });
    } else if constexpr (F32) {
        float * d = (float *) (s.second ? a.dW2 : a.dW) + t0;
        if (a.accumulate) { floats([&](uint32_t at, f32x4 v) __attribute__((always_inline)) { LK_GLOBAL f32x4 * q = (LK_GLOBAL f32x4 *) (d + at); *q = *q + v; }); }
        else { floats([&](uint32_t at, f32x4 v) __attribute__((always_inline)) { __builtin_nontemporal_store(v, (LK_GLOBAL f32x4 *) (d + at)); }); }
    } else {
        T * d = (T *) (s.second ? a.dW2 : a.dW) + t0;
        if (!a.accumulate) { halves([&](uint32_t at, V8<T> v) __attribute__((always_inline)) { __builtin_nontemporal_store(v, (LK_GLOBAL V8<T> *) (d + at)); }); return; }
#pragma unroll
        for (int m = 0; m < V::FM; ++m) {   // the sum in fp32, rounded once
            const int row = (wm * V::FM + m) * 16 + (lane & 15);
#pragma unroll
            for (int j = 0; j < V::FN; j += 2) {
                const int col = (wn * V::FN + j + ((lane >> 4) & 1)) * 16 + 8 * (lane >> 5);
                float v[8];
                eight(acc[m][j], acc[m][j + 1], v);
                T * q = d + ((uint32_t) row * (uint32_t) a.K + (uint32_t) col);
                if (s.m0 + row < a.R && s.n0 + col < a.K) { add8(q, v); put8(q, v); }
            }
        }
    }
}
// one workgroup a tile, and an XCD's share a run of them: what a workgroup has written need not have arrived when the next one starts
__device__ __forceinline__ int dw_tile() {
    const int all = (int) gridDim.x, x = (int) blockIdx.x % 8;
    return all / 8 * x + min(x, all % 8) + (int) blockIdx.x / 8;
}
template <class T, bool F32, bool PERM, class H> __global__ void __launch_bounds__(H::threads, H::PER_CU * H::NW / 4) k_mm_dw(MatmulGradArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    typedef DwCopies<T, PERM, H> C;
    typedef Waves<H, H::BM, 2> V;
    const uint32_t lds = lds_addr(dyn);
    const DwSpot s = dw_spot<H>(a, dw_tile());
    const Sums<T, true, true, H, V, C> sums(lds);
    C c;
    c.init(a, s.second ? a.dz2 : a.dz, s.begin, s.len, s.m0, s.n0);
    start<H>(c, lds);
    f32x4 acc[V::FM][V::FN];
    sums.run(acc, (s.len + BK - 1) / BK, c);
    dw_results<T, F32, V>(a, s, acc);
}
// few rows an expert: the results' memory bounds it, and a tile has a round or two. Nothing is kept ahead; four workgroups a CU cover each
// other's waits (256 experts, 7168 x 2048: of 4 rows 1267 us, Middle 1931, Large 1777; of 128 rows 2335, 2455, 2350)
template <class T, bool F32, bool PERM, class H> __global__ void __launch_bounds__(H::threads, H::PER_CU * H::NW / 4) k_mm_dw_few(MatmulGradArgs a) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    typedef DwCopies<T, PERM, H> C;
    typedef Waves<H, H::BM, 2> V;
    const uint32_t lds = lds_addr(dyn);
    const DwSpot s = dw_spot<H>(a, dw_tile());
    const Sums<T, true, true, H, V, C> sums(lds);
    f32x4 acc[V::FM][V::FN];
#pragma unroll
    for (int i = 0; i < V::FM; ++i) {
#pragma unroll
        for (int j = 0; j < V::FN; ++j) { acc[i][j] = (f32x4) { 0.f, 0.f, 0.f, 0.f }; }
    }
    if (s.len > 0) {
        C c;
        c.init(a, s.second ? a.dz2 : a.dz, s.begin, s.len, s.m0, s.n0);
        for (int d = 0; d * BK < s.len; ++d) {
            c.begin_a(d);
#pragma unroll
            for (int j = 0; j < H::CA; ++j) { c.set_a(j, lds); c.copy_a(j); }
            c.begin_b(d);
#pragma unroll
            for (int j = 0; j < H::CB; ++j) { c.set_b(j, lds + H::LB); c.copy_b(j); }
            wait_copies<0>();
            meet();
            sums.round(acc);
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            meet();
        }
    }
    dw_results<T, F32, V>(a, s, acc);
}
// the parts of dW, in order
template <class T, bool F32> __global__ void __launch_bounds__(256) k_dw_join(MatmulGradArgs a, int64_t each) {
    const int mats = (a.dW ? 1 : 0) + (a.dW2 ? 1 : 0);
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < each / 8 * mats; i += (int64_t) gridDim.x * 256) {
        float v[8] = {};
        for (int p = 0; p < a.dw_parts; ++p) { add8(a.dw_part + p * each * mats + 8 * i, v); }
        const bool second = i >= each / 8 || !a.dW;
        const int64_t at = 8 * i - (second && a.dW ? each : 0);
        if (F32) { float * d = (float *) (second ? a.dW2 : a.dW) + at; if (a.accumulate) { add8(d, v); } put8(d, v); }
        else { T * d = (T *) (second ? a.dW2 : a.dW) + at; if (a.accumulate) { add8(d, v); } put8(d, v); }
    }
}

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int CUS = 256;
// m-tiles of `bm` slots at most
int64_t most_tiles(int n, int n_exp, bool groups, int bm) { return ceil_div(n, bm) + (groups ? n_exp : 0); }
unsigned grid_of(int64_t tiles, int per_cu) { return (unsigned) std::min<int64_t>(CUS * per_cu, ceil_div(tiles, 8) * 8); }

template <class T> hipError_t join(const MatmulArgs & a, hipStream_t st) {
    k_mm_join<T><<<(unsigned) std::min<int64_t>(4096, ceil_div((int64_t) a.n * a.R, 2048)), 256, 0, st>>>(a);
    return hipGetLastError();
}
template <class T, bool GATED, class H> hipError_t fwd(const MatmulArgs & a, hipStream_t st) {
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_mm<T, GATED, H>, H::LDS)) { return e; }
    const int64_t tiles = most_tiles(a.n, a.n_exp, a.offsets, H::BM) * ceil_div(a.R, GATED ? H::BN / 2 : H::BN) * a.parts;
    k_mm<T, GATED, H><<<grid_of(tiles, H::PER_CU), H::threads, H::LDS, st>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.parts > 1) { e = join<T>(a, st); }
    return e;
}
// (B, often weights straight from memory, a round further ahead where LDS holds it: 501 rows, gated, 7168 -> 2 x 7000, weights not in any cache,
// 124 -> 110 us; A a round less and B one more 138)
// (Large's sums take half of the registers: k_mm spills 16 of the others, k_mm_dx 25 and k_mm_dw 1 or 2, all outside the loop over the rounds, once a tile)
typedef Shape<256, 256, 3, 2, 1> Large;
typedef Shape<128, 256, 3, 3, 1> Wide;
typedef Shape<64, 128, 3, 3, 2> Small;
typedef Shape<128, 128, 3, 2, 2> Middle;   // (dW)
template <class T, bool GATED> hipError_t fwd(const MatmulArgs & a, hipStream_t st) {
    switch (a.shape) {
        case MM_LARGE: return fwd<T, GATED, Large>(a, st);
        case MM_WIDE: return fwd<T, GATED, Wide>(a, st);
        default: return fwd<T, GATED, Small>(a, st);
    }
}
template <class T> hipError_t fwd(const MatmulArgs & a, hipStream_t st) { return a.W2 ? fwd<T, true>(a, st) : fwd<T, false>(a, st); }
template <class T, class H> hipError_t dx(const MatmulGradArgs & a, hipStream_t st) {
    static LdsLimit limit;
    if (const hipError_t e = limit((const void *) k_mm_dx<T, H>, H::LDS)) { return e; }
    k_mm_dx<T, H><<<grid_of(most_tiles(a.n, a.n_exp, a.offsets, H::BM) * ceil_div(a.K, H::BN) * a.parts, H::PER_CU), H::threads, H::LDS, st>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.parts > 1) {
        MatmulArgs j{};   // the sums alone
        j.n = a.n; j.R = a.K; j.n_exp = a.n_exp; j.offsets = a.offsets; j.y = a.dx; j.parts = a.parts; j.part = a.part;
        e = join<T>(j, st);
    }
    return e;
}
template <class T> hipError_t dx(const MatmulGradArgs & a, hipStream_t st) {
    switch (a.shape) {
        case MM_LARGE: return dx<T, Large>(a, st);
        case MM_WIDE: return dx<T, Wide>(a, st);
        default: return dx<T, Small>(a, st);
    }
}
template <class T, bool F32, bool PERM, class H, bool FEW> hipError_t dw(const MatmulGradArgs & a, hipStream_t st) {
    static LdsLimit limit;
    const int mats = (a.dW ? 1 : 0) + (a.dW2 ? 1 : 0);
    const int64_t all = ceil_div(a.R, H::BM) * ceil_div(a.K, H::BN) * a.n_exp * mats * a.dw_parts, each = (int64_t) a.n_exp * a.R * a.K;
    if constexpr (FEW) {
        if (const hipError_t e = limit((const void *) k_mm_dw_few<T, F32, PERM, H>, H::LDS)) { return e; }
        k_mm_dw_few<T, F32, PERM, H><<<(unsigned) all, H::threads, H::LDS, st>>>(a);
    } else {
        if (const hipError_t e = limit((const void *) k_mm_dw<T, F32, PERM, H>, H::LDS)) { return e; }
        k_mm_dw<T, F32, PERM, H><<<(unsigned) all, H::threads, H::LDS, st>>>(a);
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.dw_parts > 1) {
        k_dw_join<T, F32><<<(unsigned) std::min<int64_t>(4096, ceil_div(each * mats, 2048)), 256, 0, st>>>(a, each);
        e = hipGetLastError();
    }
    return e;
}
template <class T, bool F32, bool PERM> hipError_t dw(const MatmulGradArgs & a, hipStream_t st) {
    if (a.dw_shape == MM_FEW) { return dw<T, F32, PERM, Shape<128, 128, 1, 1, 4>, true>(a, st); }
    return a.dw_shape == MM_LARGE ? dw<T, F32, PERM, Large, false>(a, st) : dw<T, F32, PERM, Middle, false>(a, st);
}
template <class T, bool F32> hipError_t dw(const MatmulGradArgs & a, hipStream_t st) { return a.perm && a.n > 0 ? dw<T, F32, true>(a, st) : dw<T, F32, false>(a, st); }

}  // namespace

hipError_t launch_matmul(const MatmulArgs & a, hipStream_t st) {
    if (a.shape == MM_FEW) { return launch_matmul_few(a, st); }
    return a.type == TYPE_BF16 ? fwd<__bf16>(a, st) : fwd<_Float16>(a, st);
}
hipError_t launch_matmul_dx(const MatmulGradArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? dx<__bf16>(a, st) : dx<_Float16>(a, st); }
hipError_t launch_matmul_dw(const MatmulGradArgs & a, hipStream_t st) {
    if (a.dw_f32) { return a.type == TYPE_BF16 ? dw<__bf16, true>(a, st) : dw<_Float16, true>(a, st); }
    return a.type == TYPE_BF16 ? dw<__bf16, false>(a, st) : dw<_Float16, false>(a, st);
}

}  // namespace lk
