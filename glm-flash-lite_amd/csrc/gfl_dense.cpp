// C-ABI host layer of the dense operators (include/gfl_moe.h): argument checks, workspace layout, launches.
#include "gfl_moe.h"
#include "gfl_gemm_plan.hpp"
#include "gfl_internal.hpp"

#include <algorithm>
#include <cmath>

namespace {

using gfl::api_fail;

constexpr size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

// rows of whole 4-byte words, which the direct tile loads need
bool words(const void* p, int64_t ld_bytes)
{
    // at least a chunk long: what a chunk reads past its row then lies in the next one
    return reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld_bytes % 4 == 0 && ld_bytes >= 16;
}

// rows of a matrix in memory: n of them, `bytes` long, ld (elements of `size` bytes) apart
struct Span
{
    uintptr_t at;
    int64_t n, bytes, step;
    Span(const void* p, int64_t rows, int64_t cols, int64_t ld, int size)
        : at(reinterpret_cast<uintptr_t>(p)), n(rows), bytes(cols * size), step(ld * size)
    {
    }
    uintptr_t row(int64_t i) const { return at + i * step; }
    uintptr_t end() const { return row(n - 1) + bytes; }
};

// Whether two matrices (of one row or more, whose own rows do not overlap) share a byte. Matrices beside each other in rows of one buffer
// do not.
bool overlap(const Span& a, const Span& b)
{
    if (a.end() <= b.at || b.end() <= a.at) return false;
    if (a.step == b.step && a.step > 0)
    {
        const int64_t d = (int64_t)(b.at - a.at), r = (d % a.step + a.step) % a.step;
        if (r >= a.bytes && r + b.bytes <= a.step) return false;
    }
    for (int64_t i = 0, j = 0; i < a.n && j < b.n;)
    {
        if (a.row(i) + a.bytes <= b.row(j)) ++i;
        else if (b.row(j) + b.bytes <= a.row(i)) ++j;
        else return true;
    }
    return false;
}

int size_of(int dtype) { return dtype == GFL_F32 ? 4 : 2; }

int check_launch(const char* what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GFL_OK : gfl::api_hip_fail(e, what);
}

// one product of 16-bit matrices; nz = outputs side by side (grid z)
int gemm16(const char* what, int dtype, int form, int ep, int dual, int aligned, gfl::GmArgs& a, void* ws, size_t ws_bytes,
           int nz, hipStream_t st)
{
    const int r = (dtype == GFL_BF16 ? gfl::launch_gemm_bf16 : gfl::launch_gemm_f16)(form, ep, dual, aligned, a, ws, ws_bytes,
                                                                                      nz, st);
    if (r) return api_fail(GFL_EINVAL, what);
    return check_launch(what);
}

// layout of the blocks' workspaces: h (and dg, du) [M][I], then the K parts of one product at a time
struct FfnSizes
{
    int64_t ldh = 0;
    size_t h = 0, part = 0;
    size_t forward() const { return h + part; }
};

FfnSizes ffn_sizes(int M, int H, int I, bool backward)
{
    FfnSizes z;
    z.ldh = ((int64_t)I + 7) / 8 * 8;
    z.h = up256((size_t)M * z.ldh * 2);
    // aligned and other operands may be split differently: room for both
    for (int al = 0; al < 2; ++al)
    {
        if (backward)
        {
            z.part = std::max(z.part, gfl::gm_plan(gfl::GM_NN, gfl::EP_DACT, 0, al, M, I, H, 1).part_bytes);
            z.part = std::max(z.part, gfl::gm_plan(gfl::GM_NN, gfl::EP_OUT, 0, al, M, H, I, 2).part_bytes);
        }
        else
        {
            z.part = std::max(z.part, gfl::gm_plan(gfl::GM_NT, gfl::EP_GATE, 1, al, M, I, H, 1).part_bytes);
            z.part = std::max(z.part, gfl::gm_plan(gfl::GM_NT, gfl::EP_OUT, 0, al, M, H, I, 1).part_bytes);
        }
    }
    z.part = up256(z.part);
    return z;
}

int ffn_check(const char* what, int dtype, int M, int H, int I)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16) return api_fail(GFL_EINVAL, "gfl_ffn: dtype must be GFL_F16 or GFL_BF16");
    if (M < 0 || M >= GFL_MAX_ROWS || H < 1 || I < 1 || H >= GFL_MAX_LD || I >= GFL_MAX_LD)
        return api_fail(GFL_EINVAL, "gfl_ffn: need M >= 0, M < GFL_MAX_ROWS and 1 <= H, I < GFL_MAX_LD");
    (void)what;
    return GFL_OK;
}

}  // namespace

extern "C" {

int gfl_ffn_workspace(int dtype, int M, int H, int I, size_t* forward, size_t* backward)
{
    if (int rc = ffn_check("gfl_ffn_workspace", dtype, M, H, I)) return rc;
    if (forward) *forward = M ? ffn_sizes(M, H, I, false).forward() : 0;
    if (backward) *backward = M ? 3 * ffn_sizes(M, H, I, true).h + ffn_sizes(M, H, I, true).part : 0;
    return GFL_OK;
}

int gfl_ffn_forward(const void* x, int64_t ldx, const void* wg, const void* wu, const void* wd, int dtype, int M, int H,
                    int I, float act_limit, float* g, float* u, void* out, int64_t ldo, int out_dtype, int accumulate,
                    void* ws, size_t ws_bytes, gfl_stream stream)
{
    if (int rc = ffn_check("gfl_ffn_forward", dtype, M, H, I)) return rc;
    if (!(act_limit >= 0.0f)) return api_fail(GFL_EINVAL, "gfl_ffn_forward: act_limit must be 0 (off) or positive");
    if (out_dtype != dtype && out_dtype != GFL_F32)
        return api_fail(GFL_EINVAL, "gfl_ffn_forward: out_dtype must be dtype or GFL_F32");
    if (accumulate && out_dtype != GFL_F32)
        return api_fail(GFL_EINVAL, "gfl_ffn_forward: accumulate needs an out of GFL_F32");
    if (M == 0) return GFL_OK;
    if (!x || !wg || !wu || !wd || !out) return api_fail(GFL_EINVAL, "gfl_ffn_forward: NULL argument");
    if (!g != !u) return api_fail(GFL_EINVAL, "gfl_ffn_forward: g and u are given together");
    if (ldx < H || ldo < H || ldx >= GFL_MAX_LD || ldo >= GFL_MAX_LD)
        return api_fail(GFL_EINVAL, "gfl_ffn_forward: row strides must be in [H, GFL_MAX_LD)");
    const FfnSizes z = ffn_sizes(M, H, I, false);
    if (!ws || ws_bytes < z.forward() || reinterpret_cast<uintptr_t>(ws) % 16)
        return api_fail(GFL_EINVAL, "gfl_ffn_forward: workspace missing, too small or not 16-byte aligned");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    char* h = static_cast<char*>(ws);
    void* part = h + z.h;

    gfl::GmArgs a;
    a.A[0] = a.A[1] = static_cast<const char*>(x);
    a.B[0] = static_cast<const char*>(wg);
    a.B[1] = static_cast<const char*>(wu);
    a.lda = ldx * 2;
    a.ldb = (int64_t)H * 2;
    a.M = M; a.N = I; a.K = H;
    a.out[0] = h;
    a.ldo = z.ldh;
    a.limit = act_limit;
    a.g = g; a.u = u; a.ldg = I;
    int al = words(x, a.lda) && words(wg, a.ldb) && words(wu, a.ldb);
    a.ragged = H % 8 != 0;
    if (int rc = gemm16("gfl_ffn_forward: gate and up product", dtype, gfl::GM_NT, gfl::EP_GATE, 1, al, a, part, z.part, 1, st))
        return rc;

    gfl::GmArgs b;
    b.A[0] = b.A[1] = h;
    b.B[0] = b.B[1] = static_cast<const char*>(wd);
    b.lda = z.ldh * 2;
    b.ldb = (int64_t)I * 2;
    b.M = M; b.N = H; b.K = I;
    b.out[0] = out;
    b.ldo = ldo;
    b.odt = out_dtype;
    b.accumulate = accumulate;
    al = words(wd, b.ldb);
    b.ragged = I % 8 != 0;
    return gemm16("gfl_ffn_forward: down product", dtype, gfl::GM_NT, gfl::EP_OUT, 0, al, b, part, z.part, 1, st);
}

int gfl_ffn_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* g, const float* u,
                     const void* wg, const void* wu, const void* wd, int dtype, int M, int H, int I, float act_limit,
                     void* dx, int64_t lddx, void* dwg, void* dwu, void* dwd, void* ws, size_t ws_bytes, gfl_stream stream)
{
    if (int rc = ffn_check("gfl_ffn_backward", dtype, M, H, I)) return rc;
    if (!(act_limit >= 0.0f)) return api_fail(GFL_EINVAL, "gfl_ffn_backward: act_limit must be 0 (off) or positive");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (!dx && !dwg && !dwu && !dwd) return GFL_OK;
    const FfnSizes z = ffn_sizes(std::max(M, 1), H, I, true);
    char *dg = static_cast<char*>(ws), *du = dg + z.h, *h = du + z.h, *part = h + z.h;
    if (M > 0)
    {
        if (!dy || !x || !g || !u || !wg || !wu || !wd) return api_fail(GFL_EINVAL, "gfl_ffn_backward: NULL argument");
        if (lddy < H || ldx < H || (dx && lddx < H) || lddy >= GFL_MAX_LD || ldx >= GFL_MAX_LD || (dx && lddx >= GFL_MAX_LD))
            return api_fail(GFL_EINVAL, "gfl_ffn_backward: row strides must be in [H, GFL_MAX_LD)");
        if (!ws || ws_bytes < 3 * z.h + z.part || reinterpret_cast<uintptr_t>(ws) % 16)
            return api_fail(GFL_EINVAL, "gfl_ffn_backward: workspace missing, too small or not 16-byte aligned");
        gfl::GmArgs a;   // dh = dy Wd, through the activation
        a.A[0] = a.A[1] = static_cast<const char*>(dy);
        a.B[0] = a.B[1] = static_cast<const char*>(wd);
        a.lda = lddy * 2;
        a.ldb = (int64_t)I * 2;
        a.M = M; a.N = I; a.K = H;
        a.out[0] = h;
        a.dg = dg; a.du = du;
        a.ldo = z.ldh;
        a.limit = act_limit;
        a.g = const_cast<float*>(g); a.u = const_cast<float*>(u); a.ldg = I;
        const int al = words(dy, a.lda) && words(wd, a.ldb);
        a.ragged = H % 8 != 0 || I % 8 != 0;
        if (int rc = gemm16("gfl_ffn_backward: dh", dtype, gfl::GM_NN, gfl::EP_DACT, 0, al, a, part, z.part, 1, st)) return rc;
        if (dx)
        {
            gfl::GmArgs b;   // dx = dg Wg + du Wu
            b.A[0] = dg; b.A[1] = du;
            b.B[0] = static_cast<const char*>(wg); b.B[1] = static_cast<const char*>(wu);
            b.lda = z.ldh * 2;
            b.ldb = (int64_t)H * 2;
            b.M = M; b.N = H; b.K = I;
            b.segs = 2;
            b.out[0] = dx;
            b.ldo = lddx;
            b.odt = dtype;
            const int bl = words(wg, b.ldb) && words(wu, b.ldb);
            b.ragged = H % 8 != 0 || I % 8 != 0;
            if (int rc = gemm16("gfl_ffn_backward: dx", dtype, gfl::GM_NN, gfl::EP_OUT, 0, bl, b, part, z.part, 1, st)) return rc;
        }
    }
    // the weights' gradients: [dg | du]^T x and dy^T h (zeros at M = 0: no K step)
    const int ragged = H % 8 != 0 || I % 8 != 0;
    if (dwg || dwu)
    {
        gfl::GmArgs b;
        const int both = dwg && dwu;
        b.A[0] = dwg ? dg : du; b.A[1] = du;
        b.B[0] = b.B[1] = static_cast<const char*>(x);
        b.lda = z.ldh * 2;
        b.ldb = ldx * 2;
        b.M = I; b.N = H; b.K = M;
        b.out[0] = dwg ? dwg : dwu; b.out[1] = dwu;
        b.ldo = H;
        b.odt = dtype;
        b.ragged = ragged;
        const int al = M == 0 || words(x, b.ldb);
        if (int rc = gemm16("gfl_ffn_backward: dWg, dWu", dtype, gfl::GM_TN, gfl::EP_OUT, 0, al, b, nullptr, 0, both ? 2 : 1, st))
            return rc;
    }
    if (dwd)
    {
        gfl::GmArgs b;
        b.A[0] = b.A[1] = static_cast<const char*>(dy);
        b.B[0] = b.B[1] = h;
        b.lda = lddy * 2;
        b.ldb = z.ldh * 2;
        b.M = H; b.N = I; b.K = M;
        b.out[0] = dwd;
        b.ldo = I;
        b.odt = dtype;
        b.ragged = ragged;
        const int al = M == 0 || words(dy, b.lda);
        if (int rc = gemm16("gfl_ffn_backward: dWd", dtype, gfl::GM_TN, gfl::EP_OUT, 0, al, b, nullptr, 0, 1, st)) return rc;
    }
    return GFL_OK;
}

static int i8_check(int M, int N, int K)
{
    // N: a launch of 64 threads a channel has fewer than 2^32; M likewise, 256 a row
    if (M < 0 || M >= GFL_MAX_ROWS || N < 1 || K < 1 || K > 131071 || N >= GFL_MAX_N)
        return api_fail(GFL_EINVAL, "gfl_i8: need 0 <= M < GFL_MAX_ROWS (M >= 0), 1 <= N < GFL_MAX_N and 1 <= K <= 131071 (the "
                                    "int32 sum is then exact)");
    return GFL_OK;
}

static size_t i8_part(int M, int N, int K)
{
    return up256(std::max(gfl::gm_plan(gfl::GM_NT, gfl::EP_I8, 0, 0, M, N, K, 1).part_bytes,
                          gfl::gm_plan(gfl::GM_NT, gfl::EP_I8, 0, 1, M, N, K, 1).part_bytes));
}
static int64_t i8_ldq(int K) { return ((int64_t)K + 15) / 16 * 16; }

int gfl_i8_workspace(int M, int N, int K, size_t* gemm, size_t* linear)
{
    if (int rc = i8_check(M, N, K)) return rc;
    const size_t part = M ? i8_part(M, N, K) : 0;
    if (gemm) *gemm = part;
    if (linear) *linear = part + up256((size_t)M * i8_ldq(K)) + up256((size_t)M * 4);
    return GFL_OK;
}

int gfl_quant_i8(const void* x, int64_t ldx, int dtype, int M, int K, int8_t* q, float* scale, gfl_stream stream)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16) return api_fail(GFL_EINVAL, "gfl_quant_i8: dtype must be GFL_F16 or GFL_BF16");
    if (M < 0 || M >= GFL_MAX_ROWS || K < 1 || K >= GFL_MAX_LD)
        return api_fail(GFL_EINVAL, "gfl_quant_i8: need 0 <= M < GFL_MAX_ROWS and 1 <= K < GFL_MAX_LD");
    if (M == 0) return GFL_OK;
    if (!x || !q || !scale) return api_fail(GFL_EINVAL, "gfl_quant_i8: NULL argument");
    if (ldx < K || ldx >= GFL_MAX_LD) return api_fail(GFL_EINVAL, "gfl_quant_i8: the row stride must be in [K, GFL_MAX_LD)");
    gfl::launch_quant_i8(x, ldx, dtype == GFL_BF16, M, K, q, K, scale, reinterpret_cast<hipStream_t>(stream));
    return check_launch("gfl_quant_i8");
}

static int i8_product(const char* what, const int8_t* a, int64_t lda, const float* sa, const int8_t* b, int64_t ldb,
                      const float* sb, int M, int N, int K, void* out, int64_t ldo, int out_dtype, void* part,
                      size_t part_bytes, hipStream_t st)
{
    gfl::GmArgs g;
    g.A[0] = g.A[1] = reinterpret_cast<const char*>(a);
    g.B[0] = g.B[1] = reinterpret_cast<const char*>(b);
    g.lda = lda;
    g.ldb = ldb;
    g.M = M; g.N = N; g.K = K;
    g.out[0] = out;
    g.ldo = ldo;
    g.odt = out_dtype;
    g.sa = sa; g.sb = sb;
    g.ragged = K % 16 != 0;
    const int al = words(a, lda) && words(b, ldb);
    if (gfl::launch_gemm_i8(gfl::GM_NT, gfl::EP_I8, 0, al, g, part, part_bytes, 1, st)) return api_fail(GFL_EINVAL, what);
    return check_launch(what);
}

static int i8_out_check(int N, int K, int64_t ldb, const void* out, int64_t ldo, int out_dtype)
{
    if (out_dtype != GFL_F16 && out_dtype != GFL_BF16 && out_dtype != GFL_F32)
        return api_fail(GFL_EINVAL, "gfl_i8: out_dtype must be GFL_F16, GFL_BF16 or GFL_F32");
    if (!out) return api_fail(GFL_EINVAL, "gfl_i8: NULL argument");
    if (ldb < K || ldb >= GFL_MAX_LD || ldo < N || ldo >= (1 << 30))
        return api_fail(GFL_EINVAL, "gfl_i8: row strides must be at least the width (inputs below GFL_MAX_LD, out below 2^30)");
    return GFL_OK;
}

int gfl_gemm_i8(const int8_t* a, int64_t lda, const float* sa, const int8_t* b, int64_t ldb, const float* sb, int M, int N,
                int K, void* out, int64_t ldo, int out_dtype, void* ws, size_t ws_bytes, gfl_stream stream)
{
    if (int rc = i8_check(M, N, K)) return rc;
    if (M == 0) return GFL_OK;
    if (!a || !sa || !b || !sb) return api_fail(GFL_EINVAL, "gfl_gemm_i8: NULL argument");
    if (int rc = i8_out_check(N, K, ldb, out, ldo, out_dtype)) return rc;
    if (lda < K || lda >= GFL_MAX_LD) return api_fail(GFL_EINVAL, "gfl_gemm_i8: the row stride of a must be in [K, GFL_MAX_LD)");
    const size_t part = i8_part(M, N, K);
    if (part && (!ws || ws_bytes < part || reinterpret_cast<uintptr_t>(ws) % 16))
        return api_fail(GFL_EINVAL, "gfl_gemm_i8: workspace missing, too small or not 16-byte aligned");
    return i8_product("gfl_gemm_i8", a, lda, sa, b, ldb, sb, M, N, K, out, ldo, out_dtype, ws, part,
                      reinterpret_cast<hipStream_t>(stream));
}

int gfl_linear_i8(const void* x, int64_t ldx, int dtype, const int8_t* b, int64_t ldb, const float* sb, int M, int N, int K,
                  void* out, int64_t ldo, int out_dtype, void* ws, size_t ws_bytes, gfl_stream stream)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16) return api_fail(GFL_EINVAL, "gfl_linear_i8: dtype must be GFL_F16 or GFL_BF16");
    if (int rc = i8_check(M, N, K)) return rc;
    if (M == 0) return GFL_OK;
    if (!x || !b || !sb) return api_fail(GFL_EINVAL, "gfl_linear_i8: NULL argument");
    if (int rc = i8_out_check(N, K, ldb, out, ldo, out_dtype)) return rc;
    if (ldx < K || ldx >= GFL_MAX_LD) return api_fail(GFL_EINVAL, "gfl_linear_i8: the row stride of x must be in [K, GFL_MAX_LD)");
    size_t need = 0;
    gfl_i8_workspace(M, N, K, nullptr, &need);
    if (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16)
        return api_fail(GFL_EINVAL, "gfl_linear_i8: workspace missing, too small or not 16-byte aligned");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (M <= 2 && K % 8 == 0 && K >= 1024 && K <= gfl::LQ_K && reinterpret_cast<uintptr_t>(x) % 16 == 0 && (M == 1 || ldx % 8 == 0))
    {
        gfl::GmArgs g;
        g.A[0] = static_cast<const char*>(x);
        g.B[0] = reinterpret_cast<const char*>(b);
        g.lda = ldx * 2;
        g.ldb = ldb;
        g.M = M; g.N = N; g.K = K;
        g.out[0] = out;
        g.ldo = ldo;
        g.odt = out_dtype;
        g.sb = sb;
        gfl::launch_linear_row_i8(g, dtype == GFL_BF16, st);
        return check_launch("gfl_linear_i8");
    }
    const size_t part = i8_part(M, N, K);
    const int64_t ldq = i8_ldq(K);
    int8_t* q = static_cast<int8_t*>(ws) + part;
    float* sa = reinterpret_cast<float*>(q + up256((size_t)M * ldq));
    gfl::launch_quant_i8(x, ldx, dtype == GFL_BF16, M, K, q, ldq, sa, st);
    if (int rc = check_launch("gfl_linear_i8: rows to 8 bits")) return rc;
    return i8_product("gfl_linear_i8", q, ldq, sa, b, ldb, sb, M, N, K, out, ldo, out_dtype, ws, part, st);
}

int gfl_sample_workspace(int B, int V, size_t* bytes)
{
    if (B < 0 || V < 1 || V > gfl::MAX_VOCAB) return api_fail(GFL_EINVAL, "gfl_sample: need B >= 0 and 1 <= V <= 2^20");
    if (bytes) *bytes = gfl::sample_ws_bytes(B, V);
    return GFL_OK;
}

int gfl_sample(const void* logits, int64_t ld, int dtype, int B, int V, const float* temperature, const int32_t* top_k,
               const float* top_p, const float* min_p, const float* u, int64_t* token, float* prob, void* ws,
               size_t ws_bytes, gfl_stream stream)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16 && dtype != GFL_F32)
        return api_fail(GFL_EINVAL, "gfl_sample: dtype must be GFL_F16, GFL_BF16 or GFL_F32");
    size_t need = 0;
    if (int rc = gfl_sample_workspace(B, V, &need)) return rc;
    if (B == 0) return GFL_OK;
    if (!logits || !u || !token) return api_fail(GFL_EINVAL, "gfl_sample: NULL argument");
    if (ld < V) return api_fail(GFL_EINVAL, "gfl_sample: the row stride must be at least V");
    if (need && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16))
        return api_fail(GFL_EINVAL, "gfl_sample: workspace missing, too small or not 16-byte aligned");
    gfl::SampleArgs a;
    a.logits = logits; a.ld = ld; a.dtype = dtype; a.B = B; a.V = V;
    a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.u = u;
    a.token = token; a.prob = prob; a.ws = ws;
    gfl::launch_sample(a, reinterpret_cast<hipStream_t>(stream));
    return check_launch("gfl_sample");
}

// ---- 4-bit weights ----

static int i4_check(int64_t M, int N, int K, int group)
{
    if (M < 0 || M >= GFL_MAX_ROWS || N < 1 || N >= GFL_MAX_LD || K < 1 || K >= GFL_MAX_LD)
        return api_fail(GFL_EINVAL, "gfl_i4: need 0 <= M < GFL_MAX_ROWS (M >= 0) and 1 <= N, K < GFL_MAX_LD");
    if (((int64_t)K + 127) / 128 * 128 * N > (int64_t)1 << 32)   // 32-bit byte offsets in the products: 2^31 bytes of values, 2^28 of scales
        return api_fail(GFL_EINVAL, "gfl_i4: N * K (K up to a multiple of 128) must be at most 2^32");
    if (group != 32 && group != 64 && group != 128) return api_fail(GFL_EINVAL, "gfl_i4: group must be 32, 64 or 128");
    return GFL_OK;
}

// (a result of more bits than the weights rounded to x's type have is formed from the exact ones)
static bool i4_exact(int M, int N, int K, int group, int dtype, int out_dtype)
{
    return out_dtype != dtype || gfl::q4_exact(M, N, K, group);
}
static int64_t i4_ldw(int K) { return ((int64_t)K + 7) / 8 * 8; }

static size_t i4_part(int form, int M, int N, int K)
{
    return up256(std::max(gfl::gm_plan(form, gfl::EP_OUT, 0, 0, M, N, K, 1).part_bytes,
                          gfl::gm_plan(form, gfl::EP_OUT, 0, 1, M, N, K, 1).part_bytes));
}

int gfl_i4_workspace(int dtype, int out_dtype, int M, int N, int K, int group, size_t* forward, size_t* backward)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16) return api_fail(GFL_EINVAL, "gfl_i4: dtype must be GFL_F16 or GFL_BF16");
    if (int rc = i4_check(M, N, K, group)) return rc;
    const size_t w = up256((size_t)N * i4_ldw(K) * 2);
    if (forward) *forward = i4_exact(M, N, K, group, dtype, out_dtype) ? up256(gfl::q4_plan(M, N, K).part_bytes) : w + i4_part(gfl::GM_NT, M, N, K);
    if (backward)
    {
        const gfl::Q4DxPlan p = gfl::q4_dx_plan(M, N, K);
        *backward = M == 0 ? 0 : p.direct ? up256(p.part_bytes) : w + i4_part(gfl::GM_NN, M, K, N);
    }
    return GFL_OK;
}

int gfl_quant_i4(const void* w, int64_t ldw, int dtype, int N, int K, int group, uint8_t* q, void* scale, uint8_t* zero,
                 gfl_stream stream)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16) return api_fail(GFL_EINVAL, "gfl_quant_i4: dtype must be GFL_F16 or GFL_BF16");
    if (int rc = i4_check(0, N, K, group)) return rc;
    if (!w || !q || !scale) return api_fail(GFL_EINVAL, "gfl_quant_i4: NULL argument");
    if (ldw < K || ldw >= GFL_MAX_LD) return api_fail(GFL_EINVAL, "gfl_quant_i4: the row stride must be in [K, GFL_MAX_LD)");
    if (reinterpret_cast<uintptr_t>(q) % 16) return api_fail(GFL_EINVAL, "gfl_quant_i4: q must be 16-byte aligned");
    gfl::launch_quant_i4(w, ldw, dtype == GFL_BF16, N, K, group, q, scale, zero, reinterpret_cast<hipStream_t>(stream));
    return check_launch("gfl_quant_i4");
}

int gfl_pack_i4(const uint8_t* v, int64_t ldv, int N, int K, uint8_t* q, gfl_stream stream)
{
    if (int rc = i4_check(0, N, K, 32)) return rc;
    if (!v || !q) return api_fail(GFL_EINVAL, "gfl_pack_i4: NULL argument");
    if (ldv < K || ldv >= GFL_MAX_LD) return api_fail(GFL_EINVAL, "gfl_pack_i4: the row stride must be in [K, GFL_MAX_LD)");
    if (reinterpret_cast<uintptr_t>(q) % 16) return api_fail(GFL_EINVAL, "gfl_pack_i4: q must be 16-byte aligned");
    gfl::launch_pack_i4(v, ldv, N, K, q, reinterpret_cast<hipStream_t>(stream));
    return check_launch("gfl_pack_i4");
}

static int i4_args(gfl::Q4Args& a, const uint8_t* q, const void* scale, int scale_dtype, const uint8_t* zero, int N, int K, int group)
{
    if (scale_dtype != GFL_F16 && scale_dtype != GFL_BF16)
        return api_fail(GFL_EINVAL, "gfl_i4: scale_dtype must be GFL_F16 or GFL_BF16");
    if (!q || !scale) return api_fail(GFL_EINVAL, "gfl_i4: NULL argument");
    if (reinterpret_cast<uintptr_t>(q) % 16) return api_fail(GFL_EINVAL, "gfl_i4: q must be 16-byte aligned");
    a.q = q; a.scale = scale; a.zero = zero;
    a.scale_bf = scale_dtype == GFL_BF16;
    a.N = N; a.K = K; a.group = group;
    a.blocks = (K + 127) / 128;
    return GFL_OK;
}

int gfl_linear_i4(const void* x, int64_t ldx, int dtype, const uint8_t* q, const void* scale, int scale_dtype, const uint8_t* zero,
                  int M, int N, int K, int group, void* out, int64_t ldo, int out_dtype, void* ws, size_t ws_bytes,
                  gfl_stream stream)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16) return api_fail(GFL_EINVAL, "gfl_linear_i4: dtype must be GFL_F16 or GFL_BF16");
    if (out_dtype != GFL_F16 && out_dtype != GFL_BF16 && out_dtype != GFL_F32)
        return api_fail(GFL_EINVAL, "gfl_linear_i4: out_dtype must be GFL_F16, GFL_BF16 or GFL_F32");
    if (int rc = i4_check(M, N, K, group)) return rc;
    if (M == 0) return GFL_OK;
    gfl::Q4Args a;
    if (int rc = i4_args(a, q, scale, scale_dtype, zero, N, K, group)) return rc;
    if (!x || !out) return api_fail(GFL_EINVAL, "gfl_linear_i4: NULL argument");
    if (ldx < K || ldx >= GFL_MAX_LD || ldo < N || ldo >= (1 << 30))
        return api_fail(GFL_EINVAL, "gfl_linear_i4: row strides must be at least the width (x below GFL_MAX_LD, out below 2^30)");
    size_t need = 0;
    gfl_i4_workspace(dtype, out_dtype, M, N, K, group, &need, nullptr);
    if (need && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16))
        return api_fail(GFL_EINVAL, "gfl_linear_i4: workspace missing, too small or not 16-byte aligned");
    if (overlap(Span(x, M, K, ldx, 2), Span(out, M, N, ldo, size_of(out_dtype)))) return api_fail(GFL_EINVAL, "gfl_linear_i4: out overlaps x");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (i4_exact(M, N, K, group, dtype, out_dtype))
    {
        a.x = static_cast<const char*>(x);
        a.ldx = ldx * 2;
        a.M = M;
        a.out = out; a.ldo = ldo; a.odt = out_dtype;
        gfl::launch_linear_i4(a, dtype == GFL_BF16, ws, st);
        return check_launch("gfl_linear_i4");
    }
    const int64_t ldw = i4_ldw(K);
    const size_t wb = up256((size_t)N * ldw * 2);
    gfl::launch_dequant_i4(a, dtype == GFL_BF16, ws, ldw, st);
    if (int rc = check_launch("gfl_linear_i4: weights to 16 bits")) return rc;
    gfl::GmArgs b;
    b.A[0] = b.A[1] = static_cast<const char*>(x);
    b.B[0] = b.B[1] = static_cast<const char*>(ws);
    b.lda = ldx * 2;
    b.ldb = ldw * 2;
    b.M = M; b.N = N; b.K = K;
    b.out[0] = out;
    b.ldo = ldo;
    b.odt = out_dtype;
    b.ragged = K % 8 != 0;
    return gemm16("gfl_linear_i4", dtype, gfl::GM_NT, gfl::EP_OUT, 0, words(x, b.lda), b, static_cast<char*>(ws) + wb,
                  need - wb, 1, st);
}

int gfl_linear_i4_dx(const void* dy, int64_t lddy, int dtype, const uint8_t* q, const void* scale, int scale_dtype,
                     const uint8_t* zero, int M, int N, int K, int group, void* dx, int64_t lddx, void* ws, size_t ws_bytes,
                     gfl_stream stream)
{
    if (dtype != GFL_F16 && dtype != GFL_BF16) return api_fail(GFL_EINVAL, "gfl_linear_i4_dx: dtype must be GFL_F16 or GFL_BF16");
    if (int rc = i4_check(M, N, K, group)) return rc;
    if (M == 0) return GFL_OK;
    gfl::Q4Args a;
    if (int rc = i4_args(a, q, scale, scale_dtype, zero, N, K, group)) return rc;
    if (!dy || !dx) return api_fail(GFL_EINVAL, "gfl_linear_i4_dx: NULL argument");
    if (lddy < N || lddy >= GFL_MAX_LD || lddx < K || lddx >= GFL_MAX_LD)
        return api_fail(GFL_EINVAL, "gfl_linear_i4_dx: row strides must be at least the width and below GFL_MAX_LD");
    size_t need = 0;
    gfl_i4_workspace(dtype, dtype, M, N, K, group, nullptr, &need);
    if (need && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16))
        return api_fail(GFL_EINVAL, "gfl_linear_i4_dx: workspace missing, too small or not 16-byte aligned");
    if (overlap(Span(dy, M, N, lddy, 2), Span(dx, M, K, lddx, 2))) return api_fail(GFL_EINVAL, "gfl_linear_i4_dx: dx overlaps dy");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (gfl::q4_dx_plan(M, N, K).direct)
    {
        a.x = static_cast<const char*>(dy);
        a.ldx = lddy * 2;
        a.M = M;
        a.out = dx;
        a.ldo = lddx;
        a.odt = dtype;
        gfl::launch_linear_i4_dx(a, dtype == GFL_BF16, ws, st);
        return check_launch("gfl_linear_i4_dx");
    }
    const int64_t ldw = i4_ldw(K);
    const size_t wb = up256((size_t)N * ldw * 2);
    gfl::launch_dequant_i4(a, dtype == GFL_BF16, ws, ldw, st);
    if (int rc = check_launch("gfl_linear_i4_dx: weights to 16 bits")) return rc;
    gfl::GmArgs b;
    b.A[0] = b.A[1] = static_cast<const char*>(dy);
    b.B[0] = b.B[1] = static_cast<const char*>(ws);
    b.lda = lddy * 2;
    b.ldb = ldw * 2;
    b.M = M; b.N = K; b.K = N;
    b.out[0] = dx;
    b.ldo = lddx;
    b.odt = dtype;
    b.ragged = N % 8 != 0 || K % 8 != 0;
    return gemm16("gfl_linear_i4_dx", dtype, gfl::GM_NN, gfl::EP_OUT, 0, words(dy, b.lda), b, static_cast<char*>(ws) + wb,
                  need - wb, 1, st);
}

// ---- choice of experts ----

static bool known_dtype(int t) { return t == GFL_F16 || t == GFL_BF16 || t == GFL_F32; }

static int route_check(int dtype, int w_dtype, int M, int E, int topk, int score, float scale)
{
    if (!known_dtype(dtype) || !known_dtype(w_dtype))
        return api_fail(GFL_EINVAL, "gfl_route_experts: dtypes must be GFL_F16, GFL_BF16 or GFL_F32");
    if (M < 0 || M >= GFL_MAX_ROWS) return api_fail(GFL_EINVAL, "gfl_route_experts: need M >= 0 and M < GFL_MAX_ROWS");
    if (E < 1 || E > gfl::MAX_EXPERTS || topk < 1 || topk > E || topk > gfl::MAX_ROUTE_K)
        return api_fail(GFL_EINVAL, "gfl_route_experts: need 1 <= E <= 1024 and 1 <= topk <= min(E, 64)");
    if (score != GFL_SIGMOID && score != GFL_SOFTMAX)
        return api_fail(GFL_EINVAL, "gfl_route_experts: score must be GFL_SIGMOID or GFL_SOFTMAX");
    if (!std::isfinite(scale)) return api_fail(GFL_EINVAL, "gfl_route_experts: scale must be finite");
    return GFL_OK;
}

int gfl_route_experts(const void* logits, int64_t ld, int dtype, const float* bias, int M, int E, int topk, int score, int groups,
                      int top_groups, int group_best, int renorm, float scale, int64_t* sel, void* w, int w_dtype,
                      gfl_stream stream)
{
    if (int rc = route_check(dtype, w_dtype, M, E, topk, score, scale)) return rc;
    if (groups < 1 || groups > gfl::MAX_ROUTE_K || E % groups || top_groups < 1 || top_groups > groups)
        return api_fail(GFL_EINVAL, "gfl_route_experts: groups must be 1..64 and divide E, top_groups 1..groups");
    if (topk > E / groups * top_groups)
        return api_fail(GFL_EINVAL, "gfl_route_experts: topk is more than top_groups groups hold");
    if (group_best != 1 && group_best != 2) return api_fail(GFL_EINVAL, "gfl_route_experts: group_best must be 1 or 2");
    if (M == 0) return GFL_OK;
    if (!logits || !sel || !w) return api_fail(GFL_EINVAL, "gfl_route_experts: NULL argument");
    if (ld < E) return api_fail(GFL_EINVAL, "gfl_route_experts: the row stride must be at least E");
    gfl::RouteArgs a;
    a.logits = logits; a.ld = ld; a.dtype = dtype; a.bias = bias;
    a.M = M; a.E = E; a.topk = topk;
    a.softmax = score == GFL_SOFTMAX;
    a.groups = top_groups == groups ? 1 : groups;   // all of them: nothing to leave out
    a.top_groups = top_groups; a.group_best = group_best;
    a.renorm = renorm != 0;
    a.scale = scale;
    a.sel = sel; a.w = w; a.wdtype = w_dtype;
    if (gfl::launch_route_experts(a, reinterpret_cast<hipStream_t>(stream)))
        return api_fail(GFL_EINVAL, "gfl_route_experts: unsupported shape");
    return check_launch("gfl_route_experts");
}

int gfl_route_experts_backward(const void* dw, int w_dtype, const void* logits, int64_t ld, int dtype, const int64_t* sel, int M,
                               int E, int topk, int score, int renorm, float scale, void* dlogits, int64_t ldd,
                               gfl_stream stream)
{
    if (int rc = route_check(dtype, w_dtype, M, E, topk, score, scale)) return rc;
    if (M == 0) return GFL_OK;
    if (!dw || !logits || !sel || !dlogits) return api_fail(GFL_EINVAL, "gfl_route_experts_backward: NULL argument");
    if (ld < E || ldd < E) return api_fail(GFL_EINVAL, "gfl_route_experts_backward: row strides must be at least E");
    gfl::RouteArgs a;
    a.logits = logits; a.ld = ld; a.dtype = dtype;
    a.M = M; a.E = E; a.topk = topk;
    a.softmax = score == GFL_SOFTMAX;
    a.renorm = renorm != 0;
    a.scale = scale;
    a.wdtype = w_dtype;
    gfl::launch_route_backward(a, dw, sel, dlogits, ldd, reinterpret_cast<hipStream_t>(stream));
    return check_launch("gfl_route_experts_backward");
}

// ---- logits before the draw ----

static_assert(gfl::MAX_BIASES == GFL_MAX_BIASES && GFL_MAX_HISTORY < 1 << 30);   // (a history's count has 31 bits)

int gfl_adjust_logits(const void* logits, int64_t ld, int dtype, int B, int V, const int32_t* history, int64_t ldh, int L,
                      const int32_t* lengths, const int32_t* prompt, const float* repetition, const float* frequency,
                      const float* presence, const int32_t* bias_ids, int64_t ldb, const float* bias, int64_t ldv, int n_bias,
                      const int32_t* allowed, int64_t lda, void* out, int64_t ldo, gfl_stream stream)
{
    if (!known_dtype(dtype)) return api_fail(GFL_EINVAL, "gfl_adjust_logits: dtype must be GFL_F16, GFL_BF16 or GFL_F32");
    if (B < 0 || B > 65535 || V < 1 || V > gfl::MAX_VOCAB)
        return api_fail(GFL_EINVAL, "gfl_adjust_logits: need 0 <= B <= 65535 and 1 <= V <= 2^20");
    if (L < 0 || L > GFL_MAX_HISTORY || n_bias < 0 || n_bias > GFL_MAX_BIASES)
        return api_fail(GFL_EINVAL, "gfl_adjust_logits: need L in 0..GFL_MAX_HISTORY and n_bias in 0..GFL_MAX_BIASES");
    if (!history && (L || lengths || prompt || repetition || frequency || presence))
        return api_fail(GFL_EINVAL, "gfl_adjust_logits: lengths, prompt and penalties need a history");
    if (B == 0) return GFL_OK;
    if (!logits || !out || (n_bias && (!bias_ids || !bias))) return api_fail(GFL_EINVAL, "gfl_adjust_logits: NULL argument");
    if (ld < V || ldo < V || (history && ldh < L) || (n_bias && (ldb < n_bias || ldv < n_bias)) || (allowed && lda < (V + 31) / 32))
        return api_fail(GFL_EINVAL, "gfl_adjust_logits: row strides must be at least the width");
    if (logits == out && ld != ldo && B > 1) return api_fail(GFL_EINVAL, "gfl_adjust_logits: in place, with one row stride");
    if (logits != out && overlap(Span(logits, B, V, ld, size_of(dtype)), Span(out, B, V, ldo, size_of(dtype))))
        return api_fail(GFL_EINVAL, "gfl_adjust_logits: out overlaps the logits without being them");
    gfl::LogitsArgs a;
    a.logits = logits; a.ld = ld; a.out = out; a.ldo = ldo;
    a.dtype = dtype; a.B = B; a.V = V;
    a.history = history; a.ldh = ldh; a.L = history ? L : 0;
    a.lengths = lengths; a.prompt = prompt;
    a.repetition = repetition; a.frequency = frequency; a.presence = presence;
    a.bias_ids = bias_ids; a.ldb = ldb; a.bias = bias; a.ldv = ldv; a.n_bias = n_bias;
    a.allowed = allowed; a.lda = lda;
    gfl::launch_logits(a, reinterpret_cast<hipStream_t>(stream));
    return check_launch("gfl_adjust_logits");
}

}  // extern "C"
