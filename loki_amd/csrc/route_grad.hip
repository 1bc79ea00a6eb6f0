// route_grad.hip -- the router's backward pass: from the gradients of the routing weights (and of the logits themselves) to
// the logits, the router weight and the rows.
//
// z = x W^T, s = sigmoid(z), S = sum_j s_j over the row's picks, w_k = scale s_k / max(S, 2^-14) (router.hip), so
//   S > 2^-14:  ds_k = scale / S (dw_k - sum_j dw_j s_j / S),  else  ds_k = scale / 2^-14 dw_k
//   dz = dz_in + sum over the picks of ds_k s_k (1 - s_k),   dW = dz^T x,   dx = dz W
// The bias only takes part in the selection and has no gradient.
#include "moe_device.h"
#include "moe_kernels.h"

namespace lk {

namespace {

constexpr float RG_CLAMP = 0x1p-14f;   // select_token_p's
typedef float gf4 __attribute__((ext_vector_type(4)));

// one wave per row: lane k < topk holds pick k; the columns e = lane + 64 j of the row
__global__ void __launch_bounds__(256) k_route_dz(RouteGradArgs g) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = lane_id();
    if (t >= g.n) { return; }
    const int ne = g.n_exp;
    int e = -1; float gz = 0.f;
    if (g.dw) {
        float s = 0.f, om = 0.f, dw = 0.f;
        if (lane < g.topk) {
            e = g.sel[(size_t) t * g.topk + lane];
            if ((unsigned) e < (unsigned) ne) {
                const float z = g.logits[(size_t) t * ne + e], u = expf(-fabsf(z)), r = 1.f / (1.f + u);
                s = z >= 0.f ? r : u * r; om = z >= 0.f ? u * r : r;
                dw = g.dw[(size_t) t * g.topk + lane];
            } else { e = -1; }
        }
        float S = 0.f, D = 0.f;
        for (int k = 0; k < g.topk; ++k) {   // in pick order, as the forward pass adds
            const float sk = __builtin_bit_cast(float, rdlane(__builtin_bit_cast(uint32_t, s), k));
            S += sk; D += __builtin_bit_cast(float, rdlane(__builtin_bit_cast(uint32_t, dw), k)) * sk;
        }
        const float ds = S > RG_CLAMP ? g.scale / S * (dw - D / S) : g.scale / RG_CLAMP * dw;
        gz = ds * (s * om);
    }
#pragma unroll
    for (int j = 0; j < NEXP_MAX / 64; ++j) {
        const int c = lane + 64 * j;
        float v = g.dz_in && c < ne ? g.dz_in[(size_t) t * ne + c] : 0.f;
        if (g.dw) {
            for (int k = 0; k < g.topk; ++k) {
                const int ek = (int) rdlane((uint32_t) e, k);
                const float gk = __builtin_bit_cast(float, rdlane(__builtin_bit_cast(uint32_t, gz), k));
                v += ek == c ? gk : 0.f;
            }
        }
        if (c < ne) { g.dz[(size_t) t * ne + c] = v; }
    }
}

// C [M][N] = (or +=) sum_k A(m, k) B[k][N], A(m, k) = a[m sm + k sk]: a wave takes 16 rows x 64 columns on the fp32 matrix
// cores (v_mfma_f32_16x16x4_f32: lane (r, g) holds row / column r at k = g), operands straight from memory
__global__ void __launch_bounds__(64) k_route_mm(const float * __restrict__ a, int64_t sm, int64_t sk, const float * __restrict__ b, int M, int N, int K,
                                                 float * __restrict__ c, int accumulate) {
    const int lane = lane_id(), r = lane & 15, g = lane >> 4, m0 = blockIdx.y * 16, n0 = blockIdx.x * 64;
    gf4 acc[4] = {};
    const float * ap = a + (int64_t) min(m0 + r, M - 1) * sm;
    for (int k = 0; k < K; k += 4) {
        const bool in = k + g < K;
        const float av = in ? ap[(int64_t) (k + g) * sk] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float bv = in ? b[(int64_t) (k + g) * N + n0 + 16 * i + r] : 0.f;
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(av, bv, acc[i], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int m = m0 + 4 * g + q;
            if (m < M) {
                float * o = c + (int64_t) m * N + n0 + 16 * i + r;
                *o = accumulate ? *o + acc[i][q] : acc[i][q];
            }
        }
    }
}

}  // namespace

hipError_t launch_route_grad(const RouteGradArgs & a, hipStream_t st) {
    if (a.n < 0 || a.n_exp < 1 || a.n_exp > NEXP_MAX || a.E <= 0 || a.E % 64 || a.topk < 1 || a.topk > MAXK || !a.dz) { return hipErrorInvalidValue; }
    if (a.n > 0) { k_route_dz<<<(a.n + 3) / 4, 256, 0, st>>>(a); }
    if (a.dW) { k_route_mm<<<dim3(a.E / 64, (a.n_exp + 15) / 16), 64, 0, st>>>(a.dz, 1, a.n_exp, a.x, a.n_exp, a.E, a.n, a.dW, a.accumulate); }
    if (a.dx && a.n > 0) { k_route_mm<<<dim3(a.E / 64, (a.n + 15) / 16), 64, 0, st>>>(a.dz, a.n_exp, 1, a.W, a.n, a.E, a.n_exp, a.dx, 0); }
    return hipGetLastError();
}

}  // namespace lk
