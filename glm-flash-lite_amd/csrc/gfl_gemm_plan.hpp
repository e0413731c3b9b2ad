// Which tile a product takes and into how many K parts it is split: a function of sizes alone, so that the workspace query
// and the launch agree.
#pragma once
#include "gfl_internal.hpp"

#include <algorithm>

namespace gfl {

struct GmPlan
{
    int tm, tn;          // output rows and columns of a tile (tn: of each of the two matrices of a gate|up product)
    int deep;            // 128-row tiles: 8 waves and 4 steps of loads, one workgroup a CU (else 4 waves, 2 steps, two a CU)
    int parts;           // K parts
    int64_t ldp;         // elements between the rows of a part
    size_t part_bytes;
};

// Estimated time of each tile and number of K parts, the least of which is taken. A workgroup's K step of 128 bytes a row
// costs nearly the same whether its CU's other places are filled or not (it waits for its loads), so what counts is how many
// rounds of workgroups there are and how full they are; and the bytes of B, read at 4.8 TB/s, are a floor. Measured, bf16, us a
// step, in a round that fills half the places and in a fuller one: 128 x 128 0.83 and 1.03, deep 0.62 (1.0 with B [K][N]), 64 x
// 128 0.5, 256 x 256 1.05 and 1.5; 3 for the launch with its first loads and last stores; a join 2.5 and the parts' bytes written and read at 4 TB/s.
// Against measured launches it is within 15%: 333 x 2048 x 11008 in 10 parts 37 (33 measured), in 1 part 146 (167); 101 x 2 x
// 12288 x 5120 deep 56 (53), 128 x 128 69 (72); 4096 x 12288 x 5120 of 256 x 256 393 (370), 4096 x 5120 x 12288 493 (486).
inline GmPlan gm_plan(int form, int ep, int dual, int aligned, int M, int N, int K, int segs)
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
    struct Tile { int tm, tn, deep, places; double alone, beside; };
    const double deep = form == GM_NN ? 1.0 : 0.62;
    const Tile tiles[] = { { 16, 128, 0, 512, 0.45, 0.45 },  { 64, 128, 0, 512, 0.5, 0.5 },   { 128, 128, 1, 256, deep, deep },
                           { 128, 128, 0, 512, 0.83, 1.03 }, { 256, 256, 0, 256, 1.05, 1.5 } };
    const double floor = (double)d * N * K * (ep == EP_I8 ? 1 : 2) * segs / 4.8e6;
    double least = 0;
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
            const int64_t whole = wg * p / t.places, left = wg * p % t.places;
            double r = whole * t.beside + (left > t.places / 2 ? t.beside : left ? t.alone : 0);
            if (whole >= 3) r = ((double)(wg * p) / t.places + 0.25) * t.beside;   // many rounds overlap at their ends
            const double time = std::max(r * ((steps + p - 1) / p), floor) + 3 +
                                (p > 1 ? 2.5 + (double)p * d * M * ldp * 8 / 4e6 : 0);
            if (best.parts == 0 || time < least)
            {
                least = time;
                best.tm = t.tm, best.tn = t.tn / d, best.deep = t.deep, best.parts = p;
            }
        }
    }
    best.ldp = ldp;
    best.part_bytes = best.parts > 1 ? (size_t)best.parts * d * M * ldp * 4 : 0;
    return best;
}

}  // namespace gfl
