// Which tile a product takes and into how many K parts it is split: a function of sizes alone, so that the workspace query
// and the launch agree.
#pragma once
#include "gfl_internal.hpp"

#include <algorithm>

namespace gfl {

struct GmPlan
{
    int tm, tn;          // output rows and columns of a tile (tn: of each of the two matrices of a gate|up product)
    int parts;           // K parts
    int64_t ldp;         // elements between the rows of a part
    size_t part_bytes;
};

inline GmPlan gm_plan(int form, int ep, int dual, int aligned, int M, int N, int K, int segs)
{
    GmPlan p;
    const int64_t cu = 256;
    auto tiles = [&](int64_t tm, int64_t tn) { return ((M + tm - 1) / tm) * ((N + tn - 1) / tn); };
    const int d = dual ? 2 : 1;
    if (M <= 16 && form == GM_NT)   // the kernels for few tokens
    {
        p.tm = 16, p.tn = 16 / d, p.parts = 1, p.ldp = 0, p.part_bytes = 0;
        return p;
    }
    if (M <= 16 && form == GM_NN) p.tm = 16, p.tn = 128 / d;
    else if (!aligned) p.tm = 128, p.tn = 128 / d;
    else if (M <= 64) p.tm = 64, p.tn = 128 / d;
    else if (tiles(256, 256 / d) >= cu * 3 / 4) p.tm = 256, p.tn = 256 / d;
    else p.tm = 128, p.tn = 128 / d;
    p.parts = 1;
    const int64_t steps = ((int64_t)K * (ep == EP_I8 ? 1 : 2) + 127) / 128;
    if (form != GM_TN && ep != EP_DACT && segs == 1 && p.tm <= 128)
    {
        const int64_t t = tiles(p.tm, p.tn), want = 2 * cu;
        if (t < want * 3 / 4) p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({ want / t, steps / 4, 32 }));
    }
    p.ldp = (N + 3) / 4 * 4;
    p.part_bytes = p.parts > 1 ? (size_t)p.parts * d * M * p.ldp * 4 : 0;
    return p;
}

}  // namespace gfl
