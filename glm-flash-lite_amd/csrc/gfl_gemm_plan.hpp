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

}  // namespace gfl
