// matmul_few.hip -- the 16-bit products' forward pass for few rows: decode, and experts with a row or two.
//
// Bound by the weights' memory. A workgroup takes 16 rows of W (gated: and the same 16 of W2) and up to 16 slots of one expert; its waves share
// the sum's terms, 64 at a time in turn, straight from memory into registers: lane (r, g) = 16 g + r reads 32 bytes of row r, so that the
// four lanes of a row ask for a whole line, and the order of the terms in a product instruction is the same for both operands. What lies
// outside an operand is outside its buffer's range and arrives as 0. The waves' sums meet in LDS, in order. Against the split tiles of matmul.hip,
// which need a second launch: 1 row, 2048 -> 7168 9.7 us, those 13; 7168 -> 7168 19 and 23 (5.3 TB/s)
#include "matmul_device.h"

namespace lk {
namespace {

constexpr uint32_t FAR = 0xFFFF0000u, WINDOW = 0xFFFE0000u;   // an offset outside every buffer; the largest range of one
constexpr int NW = 8, U = 4;   // waves; pieces of 64 terms a wave has under way
typedef __amdgpu_buffer_rsrc_t Buf;
__device__ __forceinline__ Buf buf_of(const void * p) { return __builtin_amdgcn_make_buffer_rsrc((void *) uni64(p), (short) 0, WINDOW, 0x00020000); }
template <class T> __device__ __forceinline__ V8<T> get8(Buf b, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(V8<T>, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
#else
    (void) b; (void) off; return (V8<T>) {};
#endif
}
template <class T> __device__ __forceinline__ void put4(T * p, const float (&v)[4]) { *(LK_GLOBAL V4<T> *) p = (V4<T>) { (T) v[0], (T) v[1], (T) v[2], (T) v[3] }; }
__device__ __forceinline__ void put4(float * p, const float (&v)[4]) { *(LK_GLOBAL f32x4 *) p = (f32x4) { v[0], v[1], v[2], v[3] }; }

template <class T, bool GATED> __global__ void __launch_bounds__(64 * NW) k_mm_few(MatmulArgs a) {
    __shared__ f32x4 sums[GATED ? 2 : 1][NW][64];
    const Tiles tiles(a.offsets, a.n, a.n_exp, 16);
    const int t = (int) blockIdx.y;
    if (t >= tiles.all) { return; }
    const int e = tiles.expert(t), n0 = (int) blockIdx.x * 16, wave = uni((int) threadIdx.x >> 6), lane = lane_id(), r = lane & 15, g = lane >> 4;
    const Span sp = span_of(a.offsets, a.n, e);
    const int slot = uni(sp.begin + (t - tiles.before(e)) * 16), nm = uni(min(16, sp.end - slot));
    uint32_t xo = FAR;
    if (r < nm) {
        if (!a.perm) { xo = (uint32_t) r * (uint32_t) a.K * 2; }
        else { const uint32_t row = pair_row((uint32_t) a.perm[slot + r], a.magic); if (row < (uint32_t) a.xrows) { xo = row * (uint32_t) a.K * 2; } }
    }
    const uint32_t wo = n0 + r < a.R ? (uint32_t) r * (uint32_t) a.K * 2 : FAR;
    const size_t w0 = ((size_t) e * a.R + n0) * a.K;
    const Buf bx = buf_of((const T *) a.x + (a.perm ? 0 : (size_t) slot * a.K)), bw = buf_of((const T *) a.W + w0), bw2 = buf_of((const T *) (GATED ? a.W2 : a.W) + w0);
    f32x4 acc = (f32x4) {}, acc2 = (f32x4) {};
    auto some = [&](int c, auto count) __attribute__((always_inline)) {   // pieces c, c + NW, ...
        constexpr int N = decltype(count)::value;
        V8<T> x[N][2], w[N][2], v[N][2];
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = (c + i * NW) * 64 + 16 * g + 8 * h;
                const bool in = k < a.K;
                w[i][h] = get8<T>(bw, in && wo != FAR ? wo + 2 * (uint32_t) k : FAR);
                if (GATED) { v[i][h] = get8<T>(bw2, in && wo != FAR ? wo + 2 * (uint32_t) k : FAR); }
                x[i][h] = get8<T>(bx, in && xo != FAR ? xo + 2 * (uint32_t) k : FAR);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                acc = mfma32(w[i][h], x[i][h], acc);
                if (GATED) { acc2 = mfma32(v[i][h], x[i][h], acc2); }
            }
        }
    };
    const int pieces = (a.K + 63) / 64;
    int c = wave;
    for (; c + (U - 1) * NW < pieces; c += U * NW) { some(c, std::integral_constant<int, U>()); }
    for (; c < pieces; c += NW) { some(c, std::integral_constant<int, 1>()); }
    sums[0][wave][lane] = acc;
    if (GATED) { sums[GATED ? 1 : 0][wave][lane] = acc2; }
    __syncthreads();
    if (wave > 0) { return; }
#pragma unroll
    for (int w = 1; w < NW; ++w) { acc = acc + sums[0][w][lane]; if (GATED) { acc2 = acc2 + sums[GATED ? 1 : 0][w][lane]; } }
    const int col = n0 + 4 * g;   // lane (r, g): slot r, columns 4 g .. + 3
    if (r >= nm || col >= a.R) { return; }
    const size_t at = (size_t) (slot + r) * a.R + col;
    float z[8] = {}, y[8], z2[4];   // (4 of the 8)
#pragma unroll
    for (int u = 0; u < 4; ++u) { z[u] = acc[u] + (a.bias ? a.bias[(size_t) e * a.R + col + u] : 0.f); z2[u] = acc2[u]; }
    activate8(a.act, z, y);
    float o[4], q[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        o[u] = GATED ? y[u] * z2[u] : y[u];
        q[u] = z[u];
        if (a.residual) { o[u] += (float) ((const T *) a.residual)[at + u]; }
    }
    if (a.y_f32) { put4((float *) a.y + at, o); } else { put4((T *) a.y + at, o); }
    if (a.z) { put4((T *) a.z + at, q); }
    if (GATED && a.z2) { put4((T *) a.z2 + at, z2); }
}

template <class T> hipError_t go(const MatmulArgs & a, hipStream_t st) {
    // an expert has a tile for 16 slots; with few slots no more experts than slots have any
    const int64_t tiles = a.offsets ? std::min<int64_t>(a.n, (a.n + 15) / 16 + a.n_exp) : (a.n + 15) / 16;
    const dim3 grid((unsigned) ((a.R + 15) / 16), (unsigned) tiles);
    if (a.W2) { k_mm_few<T, true><<<grid, 64 * NW, 0, st>>>(a); } else { k_mm_few<T, false><<<grid, 64 * NW, 0, st>>>(a); }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_matmul_few(const MatmulArgs & a, hipStream_t st) { return a.type == TYPE_BF16 ? go<__bf16>(a, st) : go<_Float16>(a, st); }

}  // namespace lk
