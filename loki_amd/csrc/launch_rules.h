// launch_rules.h -- which kernel a call's sizes get: plain functions of the sizes, without HIP, so that a CPU test can hold
// them against each other (tests/test_launch_rules.py, test_q4k_rules.py, test_route_rules.py).
#pragma once
#include <stdint.h>

namespace lk {

// ---------------------------------------------------------------- router (router.hip)
// The matrix-core router works on tiles of 32 tokens x 32 experts and splits a tile's 256 chunks over `parts` workgroups, so
// that the launch fills the 256 CUs: the fewer tiles, the more parts. It depends on the tiles, not on the tokens alone: 400
// tokens are 104 tiles with 256 experts (2 parts: 60 us) but 26 with 64 (2 parts 59 us, 8 parts 25).
// 0: not split (or another kernel): below RM_MIN tokens one workgroup per expert (k_router_wg: 20.6 us at 16 tokens and 0.5 a
// token more, against 22.6 here at 17, 23.2 at 24 with 256 experts, 23.3 and 23.5 with 64); above RM_TILES tiles the
// unsplit kernel, which keeps the parts' scratch (parts x tokens x experts doubles) at 8 MiB.
constexpr int RM_MIN = 21, RM_TILES = 512;
constexpr int router_tiles(int n, int n_exp) { return ((n + 31) / 32) * ((n_exp + 31) / 32); }
constexpr int router_parts(int n, int n_exp, int K) {
    return K != 7168 || n < RM_MIN || router_tiles(n, n_exp) > RM_TILES ? 0
         : router_tiles(n, n_exp) <= 32 ? 8 : router_tiles(n, n_exp) <= 64 ? 4 : 2;
}

// ---------------------------------------------------------------- grouped GEMM columns (moe_prefill.hip, kq_gemm.hip)
// Slots of a column at most: the IQ2_XXS GEMMs' table, the two classes of a split table (narrow, few), the K-quant GEMMs'.
constexpr int PF_TOK = 112, SPLIT_TOK = 32, FEW_TOK = 8, KQ_TOK = 64;
// The IQ2_XXS table of n shared and P routed slots of n_exp experts. A split table (columns of at most 8 and of 9 .. 32 slots, one
// launch) streams a column's weights at about the memory's rate and pays for every column; the other one (columns of up to
// 112) does more work per byte and needs its three launches filled. So the line depends on the slots per expert, and on the
// slots alone where the experts are few. Split against not split, us a layer: 256 experts of 8 picks 400 tokens 932 / 956, 450
// 989 / 974; of 2 picks 1600 tokens 1214 / 1291, 2000 1369 / 1376; of 4 picks 800 tokens 994 / 1045, 1300 1481 / 1353; 128
// experts 256 tokens 574 / 629, 350 695 / 690; 64 experts 200 tokens 393 / 474, 330 562 / 523; 32 experts 200 tokens 358 / 385,
// 256 418 / 394; 16 experts 160 tokens 293 / 303, 350 489 / 484. Prompts that share a few experts: 16 hot of 256, 400 tokens
// 844 / 926; identical tokens (8 experts) 128 of them 221 / 220, 160 246 / 254, 200 311 / 303, 300 457 / 413 (the counts that
// would tell them are on the device). The shared expert alone (its pass over a prompt's rows): 256 rows 359 / 461, 512 648 /
// 746, 1000 1245 / 1245.
constexpr bool pf_split(int n, int P, int n_exp) { return P > 0 ? P <= 1280 + 8 * n_exp : n <= 768; }
// A split table takes narrow columns where they replace at least so many columns of 8 for each round of 16 narrow ones: a narrow
// column is 16 gate/up items, a round of them about 37 us more than the few columns beside it, a column of 8 about 2.2. At 17
// against always 8, and against 10 and 22: 84 rows of 2 picks, where the shared expert alone would be narrow, 286 / 286 us, 298
// at 10; 24 rows on 32 experts 139 / 139, 158 at 10; 64 rows of 8 picks 399 / 408, 404 at 22; 76 rows 435 / 461, 446 at 22.
constexpr int SPLIT_GAIN = 17;
// the shared expert's columns in a split table; alone (no routed slots) it takes smaller ones, to occupy the CUs: 65 rows 141
// us in columns of 8, 146 of 16, 157 of 32; 190 rows 315, 292, 292; 300 rows of 16 444, of 32 417
constexpr int split_shared_tok(int n, int P) { return P > 0 ? SPLIT_TOK : n <= 80 ? FEW_TOK : n <= 256 ? 16 : SPLIT_TOK; }
// the K-quant shared expert's columns: enough (column, 128 rows) items of its gate and up for the 256 CUs (at 201 tokens
// 64-slot columns are 128 items in two launches, 32-slot ones 224 in one)
constexpr int kq_shared_tok(int n) { return n <= 128 ? 16 : n <= 256 ? 32 : KQ_TOK; }

// ---------------------------------------------------------------- Q4_K products (q4k.hip)
// Every kernel gives the same bits; a call gets the one that should take least time. All but the mat-vec cut the output into workgroups
// of rows x tokens, G of them, and with nb blocks a row a launch takes about
//   max(s0 + s1 nb, ceil(G / 256) (p0 + p1 nb)) us:
// what one workgroup needs from start to end, or the rounds of workgroups a CU goes through at its steady rate. The constants are
// fitted to 247 sizes (512 .. 65536 rows, 4 .. 64 blocks, 1 .. 2000 tokens, weights from memory): 5 to 13 % rms a kernel, and the pick
// is within 1 % of the best kernel on average, 16 % at worst from 3 tokens on. Examples, us: 16 tokens through 16384 -> 7168 19 (K split, 32 rows
// x 16 tokens) against 24 (16 x 16); 37 through it 33 (K split, 32 x 48) against 43 (32 x 16) and 46 (64 x 32 tiles); 64 through 7168 ->
// 65536 85 (256 x 64) against 99 (128 x 64); 501 through 7168 -> 7000, which leaves each CU one workgroup, 68 (128 x 128 on 8 waves) against
// 75 (on 4); 2048 through 7168 -> 16384 502 (128 x 128 on 4 waves, two workgroups a CU) against 569 (8 waves) and 668 (128 x 64).
struct Q4Kernel { int rows, toks; float s0, s1, p0, p1; };
enum { Q4_KS_16_16, Q4_KS_32_16, Q4_KS_32_32, Q4_KS_32_48, Q4_MM_64_32, Q4_MM_64_64, Q4_MM_128_64, Q4_MM_256_64, Q4_MM_128_128_8, Q4_MM_128_128, Q4_KERNELS, Q4_VEC = Q4_KERNELS };
constexpr Q4Kernel Q4_KERNEL[Q4_KERNELS] = {
    { 16, 16, 4.0f, 0.113f, 1.1f, 0.138f }, { 32, 16, 3.8f, 0.194f, 2.3f, 0.226f }, { 32, 32, 4.2f, 0.325f, 2.9f, 0.344f }, { 32, 48, 5.2f, 0.311f, 3.4f, 0.471f },
    { 64, 32, 5.4f, 0.639f, 1.9f, 0.573f }, { 64, 64, 5.2f, 0.91f, 2.1f, 0.749f }, { 128, 64, 5.4f, 1.27f, 4.6f, 1.29f }, { 256, 64, 7.2f, 2.25f, 7.2f, 2.25f },
    { 128, 128, 6.3f, 2.06f, 6.3f, 2.06f }, { 128, 128, 6.3f, 2.33f, 5.1f, 1.93f } };
constexpr float q4k_us(const Q4Kernel & k, int n, int64_t R, int K) {
    const int64_t g = (R + k.rows - 1) / k.rows * ((n + k.toks - 1) / k.toks), q = (g + 255) / 256;
    const float nb = (float) (K / 256), one = k.s0 + k.s1 * nb, all = (float) q * (k.p0 + k.p1 * nb);
    return one > all ? one : all;
}
// R: rows of all matrices of the call; tiles: the tiled kernels may be taken (their scratch is there). One token: the mat-vec for very many
// rows (65536 of 7168: 53 us against 63, 65536 of 1024: 15 against 25), the K-split kernels below (16384 of 7168: 18 against 21, 2048 of 2048:
// 3.7 against 6.1).
constexpr int q4k_kernel(int n, int64_t R, int K, bool tiles) {
    if (n <= 1 && R > 24576) { return Q4_VEC; }
    int best = Q4_KS_16_16;
    for (int k = 1; k < (tiles && n > 16 ? (int) Q4_KERNELS : (int) Q4_MM_64_32); ++k) {   // (the tiled ones' times are of more than 16 tokens)
        if (q4k_us(Q4_KERNEL[k], n, R, K) < q4k_us(Q4_KERNEL[best], n, R, K)) { best = k; }
    }
    return best;
}
constexpr bool q4k_tiled(int kernel) { return kernel >= Q4_MM_64_32 && kernel < Q4_KERNELS; }

// ---------------------------------------------------------------- the router's backward products (route_grad.hip)
// Runs of rows that a tile of ROUTE_COLS columns of dW is split into, and parts of dx (ROUTE_ROWS rows at a time). One of the two products
// alone: one workgroup a CU. Both: one a CU together, three fifths of them dW's, whose rows cost more (5000 rows of 4096, 256 experts, 5 + 3
// 85 us, 8 + 8 89; 3000 rows of 6144, 160 experts, 3 + 2 67, 5 + 5 83); where that leaves more than a tenth of the CUs idle and x is large,
// several rounds of workgroups pay instead, dx's in small pieces (8192 rows of 7168: 4 + 18 207 us, 2 + 2 229; 700 rows: 39 and 37). Over
// 141 sizes (200 .. 16000 rows of 1024 .. 16384, 64 .. 256 experts) the pick is within 3 % of the best measured on average. (Times of these
// cuts side by side; dW's scale per expert has added up to 3 % to all of them since.)
constexpr int ROUTE_COLS = 128, ROUTE_ROWS = 256;
struct RouteCut { int splits, parts; };
constexpr RouteCut route_cut(int n, int E, bool dW, bool dx) {
    const int ct = E / ROUTE_COLS, one = 256 / ct;   // workgroups a column tile, one a CU
    int splits = one, parts = one;
    if (dW && dx) {
        const int both = one > 2 ? one : 2;
        if (one * ct < 230 && (int64_t) n * E >= 25000000) { parts = 1024 / ct; }
        else { splits = (3 * both + 2) / 5; parts = both - splits; }
    }
    const int ms = n / 128, mp = (n + ROUTE_ROWS - 1) / ROUTE_ROWS;   // a run of at least 128 rows, a part that has rows
    splits = splits < ms ? splits : ms; parts = parts < mp ? parts : mp;
    return { splits > 1 ? splits : 1, parts > 1 ? parts : 1 };
}

}  // namespace lk
