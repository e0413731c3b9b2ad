// Which tile a product takes and into how many K parts it is split: a function of sizes alone, so that the workspace query
// and the launch agree.
#pragma once
#include "gfl_internal.hpp"

#include <algorithm>

namespace gfl {

struct GmPlan
{
    int tm, tn;          // output rows and columns of a tile (tn: of each of the two matrices of a gate|up product)
    int deep;            // 128-row tiles: 8 waves and 5 steps of loads, one workgroup a CU (else 4 waves, 2 steps, two a CU)
    int parts;           // K parts
    int first;           // columns of a first launch of whole rounds (the rest is planned by itself), 0: all in one
    double time;         // estimated, us
    int64_t ldp;         // elements between the rows of a part
    size_t part_bytes;
};

// Estimated time of each tile and number of K parts, the least of which is taken. A workgroup's K step of 128 bytes a row
// costs nearly the same whether its CU's other places are filled or not (it waits for its loads), so what counts is how many
// rounds of workgroups there are and how full they are, with the first loads and last stores of each; and the bytes of B, read
// at 4.8 TB/s, are a floor. Measured, 16-bit types, us a step, in a round that fills half the places and in a fuller one: 128 x
// 128 0.83 and 1.03, deep 0.62, 64 x 128 0.5, 256 x 256 1.05 and 1.5; a round's ends 14 for 256 x 256, 4 for 128 x 128, 2 for the others; 3 for
// the launch; a join 2.5 and the parts' bytes written and read at 4 TB/s. nz: products of one launch (the gradients of gate and
// up), which fill rounds together.
// Against the other choice, us of a backward call for the gradients of gate's and up's weights, dh's product with them: 333 tokens
// of 5504 x 2048 128 x 128 69, 256 x 256 108; 1024 tokens of 11008 x 4096 256 x 256 343, 128 x 128 406; 2048 tokens of 5504 x 2048,
// where the estimates are 2% apart, 190 by either.
inline GmPlan gm_plan_one(int form, int ep, int dual, int aligned, int M, int N, int K, int segs, int nz = 1)
{
    GmPlan best = {};
    const int d = dual ? 2 : 1;
    if (M <= 16 && form == GM_NT)   // the kernels for few tokens
    {
        best.tm = 16, best.tn = 16 / d, best.parts = 1;
        return best;
    }
    const int steps = (int)((((int64_t)K * (ep == EP_I8 ? 1 : 2) + 127) / 128) * segs);
    const int64_t ldp = ((int64_t)N + 3) / 4 * 4;
    struct Tile { int tm, tn, deep, places; double alone, beside, ends; };
    const Tile tiles[] = { { 16, 128, 0, 512, 0.45, 0.45, 2 },  { 64, 128, 0, 512, 0.5, 0.5, 2 },
                           { 128, 128, 1, 256, 0.62, 0.62, 2 }, { 128, 128, 0, 512, 0.83, 1.03, 4 },
                           { 256, 256, 0, 256, 1.05, 1.5, 14 } };
    const double floor = (double)d * nz * N * K * (ep == EP_I8 ? 1 : 2) * segs / 4.8e6;
    for (const Tile& t : tiles)
    {
        if ((t.tm == 16) != (M <= 16 && form == GM_NN)) continue;
        if (t.tm == 64 && (M > 64 || !aligned || form == GM_TN)) continue;
        if (t.tm > 128 && !aligned) continue;
        if (t.deep && (!aligned || form == GM_TN)) continue;
        const int64_t wg = (int64_t)((M + t.tm - 1) / t.tm) * ((N + t.tn / d - 1) / (t.tn / d));
        const int most = form == GM_TN || t.tm == 256 ? 1 : std::max(1, std::min(steps / 4, 32));
        for (int p = 1; p <= most; ++p)
        {
            if (p > 1 && wg * (p - 1) >= t.places) break;
            const int64_t whole = nz * wg * p / t.places, left = nz * wg * p % t.places;
            double r = whole * t.beside + (left > t.places / 2 ? t.beside : left ? t.alone : 0), ends = whole + (left > 0);
            if (whole >= 3)   // many rounds overlap at their ends
            {
                ends = (double)(nz * wg * p) / t.places + 0.25;
                r = ends * t.beside;
            }
            const double time = std::max(r * ((steps + p - 1) / p) + ends * t.ends, floor) + 3 +
                                (p > 1 ? 2.5 + (double)p * d * M * ldp * 8 / 4e6 : 0);
            if (best.parts == 0 || time < best.time)
            {
                best.time = time;
                best.tm = t.tm, best.tn = t.tn / d, best.deep = t.deep, best.parts = p;
            }
        }
    }
    best.ldp = ldp;
    best.part_bytes = best.parts > 1 ? (size_t)best.parts * d * M * ldp * 4 : 0;
    return best;
}

// The 256 x 256 tiles of a product in whole rounds, and the columns left in a launch of their own where a smaller tile spreads
// them better than a last round that leaves most CUs idle: 4096 x 5120 x 12288 (320 tiles) 463 us, 572 in
// one launch.
inline GmPlan gm_plan(int form, int ep, int dual, int aligned, int M, int N, int K, int segs, int nz = 1)
{
    GmPlan p = gm_plan_one(form, ep, dual, aligned, M, N, K, segs, nz);
    if (p.tm != 256) return p;
    const int rows = (M + 255) / 256 * nz, cols = (N + p.tn - 1) / p.tn, first = (int)((int64_t)rows * cols / 256 * 256 / rows);
    if (first == 0 || first == cols) return p;
    const GmPlan a = gm_plan_one(form, ep, dual, aligned, M, first * p.tn, K, segs, nz);
    const GmPlan b = gm_plan(form, ep, dual, aligned, M, N - first * p.tn, K, segs, nz);
    if (a.tm != 256 || a.time + b.time >= p.time) return p;
    p.first = first * p.tn;
    p.time = a.time + b.time;
    p.part_bytes = b.part_bytes;
    return p;
}

// A product with a 4-bit weight whose weights are unpacked in its own launch: the kernel for few tokens, or tiles of 16 tt tokens and
// 128 nt channels over `parts` of the inputs.
struct Q4Plan
{
    int few, tt, nt, parts;
    int64_t ldp;
    size_t part_bytes;
};

constexpr int Q4_TOKENS = 144 << 10;   // bytes of LDS for the tokens of the kernel for few

inline Q4Plan q4_plan(int M, int N, int K)
{
    Q4Plan p = {};
    const int blocks = (K + 127) / 128;
    p.few = K < 8 || (M <= 16 && (int64_t)M * (blocks * 256 + 16) <= Q4_TOKENS);
    p.parts = 1;
    if (p.few) return p;
    p.tt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    const int64_t tall = (M + 16 * p.tt - 1) / (16 * p.tt);
    p.nt = tall * ((N + 255) / 256) * (blocks / 4) < 256 ? 1 : 2;
    const int64_t wg = tall * ((N + 128 * p.nt - 1) / (128 * p.nt));
    // parts of two steps of 256 inputs or more, or of one where that makes up to four: us with and without those of one, 1024 -> 1024 128
    // tokens 9.3 and 13.0, 64 9.1 and 10.8; in 8 parts of one 2048 -> 2048 128 tokens 13.9, in 4 of two 12.8
    const int most = std::max(blocks / 4, std::min((blocks + 1) / 2, 4));
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(most, 16), 256 / wg));
    p.ldp = ((int64_t)N + 3) / 4 * 4;
    p.part_bytes = p.parts > 1 ? (size_t)p.parts * M * p.ldp * 4 : 0;
    return p;
}

// Whether the weights are unpacked in the product's own launch, where they enter exactly, or to 16 bits first for the tile GEMM, where
// (v - z) s is rounded to x's type: up to 2^-8 of a weight in bf16 (2.2e-3 of the result instead of 1.7e-3, which is the result's own
// rounding), chosen because the exact tiles take 682 us of 4096 tokens 5120 -> 12288 where the GEMM takes 416 (2048 tokens 339 and 245). By
// estimated time. A round of 256 tiles of 64 x 256 takes 2.8 us a step of 256 inputs, 3.0 with groups of 64, 3.6 of 32, the launch and
// the join 5 to 10; unpacking moves 2.5 bytes a weight at 4.2 TB/s. Measured, us, here and there: 5120 -> 12288 groups of 128 128
// tokens 38 and 72, 256 58 and 84, 512 115 and 116, 1024 185 and 155, groups of 32 256 tokens 73 and 93, 512 147 and 125; 2048 -> 2048
// 1024 tokens 25 and 32.
inline bool q4_exact(int M, int N, int K, int group)
{
    if (M <= 64 || K < 8) return true;
    const Q4Plan p = q4_plan(M, N, K);
    const int64_t wg = (int64_t)((M + 63) / 64) * ((N + 128 * p.nt - 1) / (128 * p.nt)) * p.parts, steps = ((K + 127) / 128 / p.parts + 1) / 2;
    const double own = 5 + (p.parts > 1 ? 5 : 0) + (double)((wg + 255) / 256) * steps * (group == 128 ? 2.8 : group == 64 ? 3.0 : 3.6);
    return own <= 3 + 2.5 * N * K / 4.2e6 + gm_plan(GM_NT, EP_OUT, 0, 1, M, N, K, 1).time;
}

// Its gradient with respect to the input: straight from the packed weights, by tiles of 16 tt tokens and 128 columns over `parts` of the
// weight's rows, or (direct 0) from weights unpacked to 16 bits first, by the tile GEMM. By estimated time: a step of 256 rows takes a
// tile 0.8, 1.1 or 1.6 us, the launch 5, a join 5 and the parts' bytes written and read at 4 TB/s; unpacking moves 2.5 bytes a weight at
// 4.2 TB/s. Measured, us, direct and otherwise, 11008 -> 4096: 1 token 14 and 45, 24 17 and 45, 64 22 and 47, 100 28 and 49, 300 62 and 65,
// 1001 142 and 147; 5120 -> 12288, 4096 tokens 758 and 471. 256 workgroups, not 512: 8 tokens 14 and 18.
struct Q4DxPlan
{
    int direct, tt, parts;
    int64_t ldp;
    size_t part_bytes;
};

inline Q4DxPlan q4_dx_plan(int M, int N, int K)
{
    Q4DxPlan p = {};
    if (N < 8 || M == 0) return p;   // (a lane loads 8 neighbouring rows)
    const int blocks = (K + 127) / 128, steps = (N + 31) / 32;
    p.tt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    const int64_t wg = (int64_t)((M + 16 * p.tt - 1) / (16 * p.tt)) * blocks;
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(steps / 16, 16), 256 / wg));
    p.ldp = ((int64_t)K + 3) / 4 * 4;
    p.part_bytes = p.parts > 1 ? (size_t)p.parts * M * p.ldp * 4 : 0;
    // (parts of at least two steps a wave: with one, 64 tokens take 13.1 us and not 11.5 at 1024 -> 1024, 14.1 and not 13.8 at 2048 -> 2048)
    const int64_t each = ((steps + p.parts - 1) / p.parts + 7) / 8;   // a wave's
    const double own = 5 + (double)((wg * p.parts + 255) / 256) * each * (p.tt == 1 ? 0.8 : p.tt == 2 ? 1.1 : 1.6) +
                       (p.parts > 1 ? 5 + (double)p.part_bytes * 2 / 4e6 : 0);
    p.direct = wg * p.parts < 1 << 22 && own <= 3 + 2.5 * N * K / 4.2e6 + gm_plan(GM_NN, EP_OUT, 0, 1, M, K, N, 1).time;
    return p;
}

}  // namespace gfl
