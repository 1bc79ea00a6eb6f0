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

// ---------------------------------------------------------------- 16-bit products (matmul.hip)
// Tiles of bm x bn, `slots` of them at a time on the chip. A tile takes fixed + rounds * (a round of 64 terms) us, a round `one` where
// few CUs have work and `full` where all have (the clock falls with the power, and Small's two workgroups share a CU). A sum can be split into
// parts, whose results a second launch adds up. The constants were fitted to 112 sizes (16 .. 2048 rows, 512 .. 16384 columns and terms, weights from
// memory) when the kernels copied B two rounds ahead; with the present ones the choice is 2.8 % above the best on average there, 20 % at most.
// Examples, us, Small / Wide / Large, then the best split: 64 rows, 7168 terms -> 2048 columns 35 / 55 / -, 16 (Small, 6 parts); 501, 7168 -> 2048
// 36 / 72 / 132, 30 (Small, 2); 501, 2048 -> 7168 25 / 28 / 49; 1024, 7168 -> 7168 133 / 88 / 137; 2048, 7168 -> 7168 288 / 184 / 159; 2048,
// 2048 -> 2048 28 / 29 / 49; 512 rows, columns and terms 7.5 / 13 / 21.
enum { MM_SMALL, MM_WIDE, MM_LARGE, MM_FEW };
struct MmPlan { int shape, parts; };
struct MmCost { int bm, bn, slots; float fixed, one, full, stream; };
constexpr MmCost MM_COST[3] = { { 64, 128, 512, 3.7f, 0.40f, 0.69f, 1.f }, { 128, 256, 256, 5.4f, 0.55f, 0.86f, 1.06f }, { 256, 256, 256, 10.0f, 1.07f, 1.33f, 1.08f } };
// experts with rows, about: n_exp (1 - e^-x) for x rows an expert
constexpr float mm_used(int n, int n_exp) {
    const float x = (float) n / (float) n_exp;
    return n_exp == 1 || x > 3.f ? (float) n_exp : (float) n_exp * x / (1.f + 0.5f * x + 0.0833f * x * x);
}
constexpr float mm_time(int shape, int parts, int n, int n_exp, int cols, int terms) {
    const MmCost k = MM_COST[shape];
    const float per = (float) n / (float) n_exp;
    // m-tiles: an expert's last one is half full on average (and costs less: the waves share as many rows as it has)
    const float mt = n_exp == 1 ? (float) ((n + k.bm - 1) / k.bm) : (float) n / (float) k.bm + 0.5f * (float) (n < n_exp ? n : n_exp);
    const float fill = per / ((float) n_exp >= 2.f ? mt * (float) k.bm / (float) n_exp : per);
    const float items = mt * (float) ((cols + k.bn - 1) / k.bn) * (float) parts;
    const int rounds = (terms + 63) / 64, r = (rounds + parts - 1) / parts;
    float waves = items / (float) k.slots;
    const float busy = waves >= 1.f ? 1.f : shape == MM_SMALL ? (waves > 0.5f ? 1.f : 0.f) : waves;
    if (n_exp == 1 || waves < 1.f) { const int w = (int) waves; waves = (float) w < waves ? (float) (w + 1) : (float) w; }
    const float cost = (k.one + (k.full - k.one) * busy) * (shape == MM_LARGE && n_exp > 1 ? 0.62f + 0.38f * fill : 1.f);
    const float sums = waves * (k.fixed + (float) r * cost);
    const float memory = ((float) cols * (float) terms * mm_used(n, n_exp) * 3.1e-7f + (float) n * (float) cols * 4e-7f) * (shape == MM_SMALL && busy == 0.f ? 1.3f : k.stream);   // the weights and the results
    const float join = parts > 1 ? 4.f + 0.15f * (float) parts + (float) parts * (float) n * (float) cols * 1.2e-6f : 0.f;
    return 2.5f + (sums > memory ? sums + 0.15f * memory : memory + 0.15f * sums) + join;
}
// Few rows (matmul_few.hip; up to 16 of an expert with one reading of its matrix): 16 columns a workgroup, whose 8 waves take 64 terms each in turn.
// Us against the best of the above: 1 row of 2048 terms -> 7168 columns 9.7 / 13, 7168 -> 7168 19 / 23, 7168 -> 131072 357 / 309; 8 rows 11 / 14,
// 24 / 23, 463 / 310; 16 rows 12 / 14, 28 / 23; one token's 8 experts of 256, 7168 -> 2 x 2048, 90 / 84, two tokens' 170 / 151; 6 of 64, 2048 ->
// 2 x 1024, 12 / 19, 48 51 / 51, 192 98 / 92.
constexpr float mm_few_time(int n, int n_exp, int cols, int terms) {
    const float used = mm_used(n, n_exp), rows = (float) n / used;
    const float tiles = n_exp == 1 ? (float) ((n + 15) / 16) : rows < 8.f ? used : used * (0.5f + rows / 16.f), groups = tiles * (float) cols / 16.f;
    const float memory = (float) cols * (float) terms * tiles * 2.9e-7f * (1.f + 0.036f * (rows < 16.f ? rows : 16.f)), waves = 0.53f * (float) ((terms + 511) / 512);
    return 4.f + (memory > waves ? memory : waves) + (groups > 1024.f ? 0.01f * (groups - 1024.f) : 0.f);
}
// n rows of n_exp experts, `cols` results a row (gated: of both matrices), sums of `terms`
constexpr MmPlan mm_plan(int n, int n_exp, int cols, int terms, bool forward) {
    const int split[8] = { 1, 2, 3, 4, 6, 8, 12, 16 };
    MmPlan best{ MM_SMALL, 1 };
    float least = mm_time(MM_SMALL, 1, n, n_exp, cols, terms);
    for (int s = 0; s < 3; ++s) {
        for (int i = 0; i < 8; ++i) {
            if (split[i] > 1 && split[i] * 128 > terms) { break; }   // two rounds a part at least
            const float t = mm_time(s, split[i], n, n_exp, cols, terms);
            if (t < least) { least = t; best = { s, split[i] }; }
        }
    }
    if (forward && n <= 1 << 15 && mm_few_time(n, n_exp, cols, terms) < least) { return { MM_FEW, 1 }; }
    return best;
}

// dW of `mats` matrices [n_exp][R][K] from n rows: tiles of 256 x 256 (MM_LARGE), of 128 x 128 with two workgroups a CU (MM_SMALL) or four
// that keep nothing ahead (MM_FEW); the rows can be split into parts. Fitted to 25 sizes before the results went past the caches; with the present
// kernels 2.0 % above the best there, 20 % at most. Us, MM_SMALL / MM_LARGE / MM_FEW: 16 rows, 7168 x 7168 31 / 37 / 23; 501 65 / 69 / 62; 8192
// 910 / 676 / 1048; 8192 rows, 2048 x 2048 66 / 142 / 129, 512 x 512 57 and 19 in 8 parts; 256 experts of 4, 128 and 256 rows, 7168 x 2048,
// 1931 / 1777 / 1267, 2455 / 2350 / 2335, 3205 / 2840 / 3009.
constexpr float dw_time(int shape, int parts, int n, int n_exp, int R, int K, int mats) {
    const int b = shape == MM_LARGE ? 256 : 128, slots = shape == MM_LARGE ? 256 : shape == MM_FEW ? 1024 : 512;
    const float fixed = shape == MM_LARGE ? 10.f : shape == MM_FEW ? 5.4f : 5.f, one = shape == MM_LARGE ? 0.92f : shape == MM_FEW ? 1.05f : 0.5f,
                full = shape == MM_LARGE ? 1.28f : shape == MM_FEW ? 1.75f : 0.88f;
    const float all = (float) ((R + b - 1) / b) * (float) ((K + b - 1) / b) * (float) n_exp * (float) mats * (float) parts;
    const float rounds = n_exp == 1 ? (float) ((n + 63) / 64) : (float) n / (float) n_exp / 64.f + 0.5f;
    const float r = parts == 1 ? rounds : (float) (int) (rounds / (float) parts + 0.999f);
    float waves = all / (float) slots;
    const float busy = waves >= 1.f ? 1.f : shape == MM_SMALL ? (waves > 0.5f ? 1.f : 0.f) : waves;
    if (waves < 8.f) { const int w = (int) waves; waves = (float) w < waves ? (float) (w + 1) : (float) w; }
    const float values = (float) R * (float) K * (float) n_exp * (float) mats, sums = waves * (fixed + r * (one + (full - one) * busy)), memory = values * 3.7e-7f;
    return 2.5f + (sums > memory ? sums + 0.15f * memory : memory + 0.15f * sums) + (parts > 1 ? 4.f + 0.15f * (float) parts + (float) parts * values * 1.2e-6f : 0.f);
}
constexpr MmPlan dw_plan(int n, int n_exp, int R, int K, int mats) {
    const int split[8] = { 1, 2, 4, 8, 16, 1, 1, 1 }, shapes[3] = { MM_SMALL, MM_LARGE, MM_FEW };
    MmPlan best{ MM_SMALL, 1 };
    float least = dw_time(MM_SMALL, 1, n, n_exp, R, K, mats);
    for (int s = 0; s < 3; ++s) {
        for (int i = 0; i < 5; ++i) {
            if (split[i] > 1 && (long long) split[i] * 128 * n_exp > n) { break; }   // two rounds a part at least
            const float t = dw_time(shapes[s], split[i], n, n_exp, R, K, mats);
            if (t < least) { least = t; best = { shapes[s], split[i] }; }
        }
    }
    return best;
}

}  // namespace lk
