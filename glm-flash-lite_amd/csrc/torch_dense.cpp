// The dense operators (include/gfl_moe.h: gfl_ffn_*, gfl_quant_i8, gfl_gemm_i8, gfl_linear_i8, gfl_*_i4, gfl_route_experts*,
// gfl_adjust_logits, gfl_sample) over torch tensors:
// checks, outputs and workspaces from torch's allocator, the launch on torch's current stream of the tensors' device. In C++
// because a decode step's calls take less time on the GPU (12 us for a shared expert) than their checks take in Python.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <optional>
#include <tuple>

#include "gfl_moe.h"

namespace {

using torch::Tensor;
typedef std::optional<Tensor> OptTensor;

void check_rc(int rc) { TORCH_CHECK(rc == GFL_OK, gfl_last_error()); }

int code_of(at::ScalarType t)
{
    return t == at::kHalf ? GFL_F16 : t == at::kBFloat16 ? GFL_BF16 : t == at::kFloat ? GFL_F32 : -1;
}

int size_of(const char* what, int64_t n)
{
    TORCH_CHECK_VALUE(n <= INT_MAX, what, ": size ", n, " is past 2^31");
    return static_cast<int>(n);
}

// t [..., cols] as rows with one stride between them
struct Rows
{
    int n;
    int64_t ld;
};
Rows rows_of(const char* what, const Tensor& t, int64_t cols)
{
    const int64_t d = t.dim();
    TORCH_CHECK_VALUE(d >= 1 && t.size(-1) == cols, what, " must be [..., ", cols, "]");
    if (t.is_contiguous()) return { size_of(what, cols ? t.numel() / cols : 0), cols };
    TORCH_CHECK_VALUE(d <= 2, what, " with more than two dimensions must be contiguous");
    TORCH_CHECK_VALUE(cols <= 1 || t.stride(-1) == 1, what, " must have contiguous rows");
    if (d == 1 || t.size(0) <= 1) return { d == 1 ? 1 : size_of(what, t.size(0)), cols };
    TORCH_CHECK_VALUE(t.stride(0) >= cols, what, ": rows overlap (row stride ", t.stride(0), ", width ", cols, ")");
    return { size_of(what, t.size(0)), t.stride(0) };
}

// one device for all: that device made current (the C calls launch on the current one), its current stream
struct On
{
    c10::OptionalDeviceGuard guard;
    gfl_stream stream;
    On(const char* what, const Tensor& ref, std::initializer_list<const Tensor*> others)
    {
        TORCH_CHECK_VALUE(ref.is_cuda(), what, ": tensors must be on the device");
        const at::Device dev = ref.device();
        for (const Tensor* t : others)
            TORCH_CHECK_VALUE(!t || !t->defined() || t->device() == dev, what, ": all tensors must be on ", dev);
        guard.reset_device(dev);
        stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    }
};

const Tensor* ptr(const OptTensor& t) { return t ? &*t : nullptr; }
template <typename T = void>
T* addr(const OptTensor& t)
{
    return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// The caller's own output has other values now: a backward pass that saved the old ones is refused.
void written(const OptTensor& out)
{
    if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

Tensor workspace(size_t bytes, const Tensor& ref)
{
    return bytes ? at::empty({ static_cast<int64_t>(bytes) }, ref.options().dtype(at::kByte)) : Tensor();
}
void* addr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Ffn
{
    int H, I, code;
    Ffn(const char* what, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd)
    {
        code = code_of(x.scalar_type());
        TORCH_CHECK_VALUE((code == GFL_F16 || code == GFL_BF16) && x.dim() >= 1, what, ": x must be fp16 or bf16 [..., H]");
        TORCH_CHECK_VALUE(wg.dim() == 2 && wg.size(1) == x.size(-1), what, ": wg must be [I, ", x.size(-1), "]");
        I = size_of(what, wg.size(0));
        H = size_of(what, wg.size(1));
        TORCH_CHECK_VALUE(wu.sizes() == wg.sizes() && wd.dim() == 2 && wd.size(0) == H && wd.size(1) == I, what, ": wu must be [",
                          I, ", ", H, "] and wd [", H, ", ", I, "]");
        for (const Tensor* t : { &wg, &wu, &wd })
            TORCH_CHECK_VALUE(t->scalar_type() == x.scalar_type() && t->is_contiguous(), what,
                              ": the weights must be contiguous, of x's type");
    }
};

std::tuple<Tensor, Tensor, Tensor> ffn_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                                               const OptTensor& out, double act_limit, bool save, bool accumulate)
{
    const char* what = "ffn_forward";
    const Ffn f(what, x, wg, wu, wd);
    const Rows r = rows_of("ffn_forward: x", x, f.H);
    const On on(what, x, { &wg, &wu, &wd, ptr(out) });
    TORCH_CHECK_VALUE(out || !accumulate, "ffn_forward: accumulate needs out");
    TORCH_CHECK_VALUE(!out || (out->sizes() == x.sizes() &&
                               (out->scalar_type() == x.scalar_type() || out->scalar_type() == at::kFloat)),
                      "ffn_forward: out must have x's shape and be of its type or fp32");
    Tensor y = out ? *out : at::empty(x.sizes(), x.options()), g, u;
    const Rows o = rows_of("ffn_forward: out", y, f.H);
    if (save)
    {
        g = at::empty({ r.n, f.I }, x.options().dtype(at::kFloat));
        u = at::empty_like(g);
    }
    size_t need = 0;
    check_rc(gfl_ffn_workspace(f.code, r.n, f.H, f.I, &need, nullptr));
    const Tensor ws = workspace(need, x);
    check_rc(gfl_ffn_forward(x.data_ptr(), r.ld, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), f.code, r.n, f.H, f.I,
                             static_cast<float>(act_limit), static_cast<float*>(addr(g)), static_cast<float*>(addr(u)),
                             y.data_ptr(), o.ld, code_of(y.scalar_type()), accumulate, addr(ws), need, on.stream));
    written(out);
    return { y, g, u };
}

std::tuple<OptTensor, OptTensor, OptTensor, OptTensor> ffn_backward(const Tensor& dy, const Tensor& x, const Tensor& g,
                                                                    const Tensor& u, const Tensor& wg, const Tensor& wu,
                                                                    const Tensor& wd, double act_limit,
                                                                    std::tuple<bool, bool, bool, bool> need)
{
    const char* what = "ffn_backward";
    const Ffn f(what, x, wg, wu, wd);
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
                      "ffn_backward: dy must have x's shape and type");
    const Rows r = rows_of("ffn_backward: x", x, f.H), d = rows_of("ffn_backward: dy", dy, f.H);
    for (const Tensor* t : { &g, &u })
        TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == r.n && t->size(1) == f.I && t->scalar_type() == at::kFloat &&
                              t->is_contiguous(),
                          "ffn_backward: g and u must be contiguous fp32 [", r.n, ", ", f.I, "]");
    const On on(what, x, { &dy, &g, &u, &wg, &wu, &wd });
    auto grad = [](bool wanted, const Tensor& like) {
        return wanted ? OptTensor(at::empty(like.sizes(), like.options())) : OptTensor();
    };
    const OptTensor dx = grad(std::get<0>(need), x), dwg = grad(std::get<1>(need), wg), dwu = grad(std::get<2>(need), wu),
                    dwd = grad(std::get<3>(need), wd);
    size_t bytes = 0;
    check_rc(gfl_ffn_workspace(f.code, r.n, f.H, f.I, nullptr, &bytes));
    const Tensor ws = workspace(bytes, x);
    check_rc(gfl_ffn_backward(dy.data_ptr(), d.ld, x.data_ptr(), r.ld, g.data_ptr<float>(), u.data_ptr<float>(),
                              wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), f.code, r.n, f.H, f.I,
                              static_cast<float>(act_limit), addr(dx), f.H, addr(dwg), addr(dwu), addr(dwd), addr(ws), bytes,
                              on.stream));
    return { dx, dwg, dwu, dwd };
}

int x16_code(const char* what, const Tensor& x)
{
    const int code = code_of(x.scalar_type());
    TORCH_CHECK_VALUE((code == GFL_F16 || code == GFL_BF16) && x.dim() >= 1 && x.size(-1) >= 1, what,
                      ": x must be fp16 or bf16 [..., K]");
    return code;
}

std::tuple<Tensor, Tensor> quant_i8(const Tensor& x)
{
    const int code = x16_code("quant_i8", x), K = size_of("quant_i8", x.size(-1));
    const Rows r = rows_of("quant_i8: x", x, K);
    const On on("quant_i8", x, {});
    Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
    Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    check_rc(gfl_quant_i8(x.data_ptr(), r.ld, code, r.n, K, q.data_ptr<int8_t>(), scale.data_ptr<float>(), on.stream));
    return { q, scale };
}

Rows i8_weight(const char* what, int K, const Tensor& b, const Tensor& sb)
{
    TORCH_CHECK_VALUE(b.scalar_type() == at::kChar && b.dim() == 2 && b.size(1) == K, what, ": b must be int8 [N, ", K, "]");
    const Rows r = rows_of(what, b, K);
    TORCH_CHECK_VALUE(sb.scalar_type() == at::kFloat && sb.dim() == 1 && sb.size(0) == r.n && sb.is_contiguous(), what,
                      ": sb must be contiguous fp32 [", r.n, "]");
    return r;
}

Tensor i8_out(const char* what, const Tensor& a, int N, const OptTensor& out, std::optional<at::ScalarType> dtype,
              at::ScalarType fallback)
{
    at::DimVector shape(a.sizes());
    shape.back() = N;
    if (out)
    {
        TORCH_CHECK_VALUE(!dtype || out->scalar_type() == *dtype, what, ": out's type is not dtype");
        TORCH_CHECK_VALUE(out->sizes() == at::IntArrayRef(shape) && code_of(out->scalar_type()) >= 0, what,
                          ": out must be fp16, bf16 or fp32 ", at::IntArrayRef(shape));
        return *out;
    }
    const at::ScalarType t = dtype.value_or(fallback);
    TORCH_CHECK_VALUE(code_of(t) >= 0, what, ": dtype must be fp16, bf16 or fp32");
    return at::empty(shape, a.options().dtype(t));
}

Tensor gemm_i8(const Tensor& a, const Tensor& sa, const Tensor& b, const Tensor& sb, const OptTensor& out,
               std::optional<at::ScalarType> dtype)
{
    const char* what = "gemm_i8";
    TORCH_CHECK_VALUE(a.scalar_type() == at::kChar && a.dim() >= 1 && a.size(-1) >= 1, "gemm_i8: a must be int8 [..., K]");
    const int K = size_of(what, a.size(-1));
    const Rows r = rows_of("gemm_i8: a", a, K);
    TORCH_CHECK_VALUE(sa.scalar_type() == at::kFloat && sa.sizes() == a.sizes().slice(0, a.dim() - 1) && sa.is_contiguous(),
                      "gemm_i8: sa must be contiguous fp32 ", a.sizes().slice(0, a.dim() - 1));
    const Rows w = i8_weight(what, K, b, sb);
    const On on(what, a, { &sa, &b, &sb, ptr(out) });
    const Tensor y = i8_out(what, a, w.n, out, dtype, at::kHalf);
    const Rows o = rows_of("gemm_i8: out", y, w.n);
    size_t need = 0;
    check_rc(gfl_i8_workspace(r.n, w.n, K, &need, nullptr));
    const Tensor ws = workspace(need, a);
    check_rc(gfl_gemm_i8(a.data_ptr<int8_t>(), r.ld, sa.data_ptr<float>(), b.data_ptr<int8_t>(), w.ld, sb.data_ptr<float>(),
                         r.n, w.n, K, y.data_ptr(), o.ld, code_of(y.scalar_type()), addr(ws), need, on.stream));
    written(out);
    return y;
}

Tensor linear_i8(const Tensor& x, const Tensor& b, const Tensor& sb, const OptTensor& out, std::optional<at::ScalarType> dtype)
{
    const char* what = "linear_i8";
    const int code = x16_code(what, x), K = size_of(what, x.size(-1));
    const Rows r = rows_of("linear_i8: x", x, K), w = i8_weight(what, K, b, sb);
    const On on(what, x, { &b, &sb, ptr(out) });
    const Tensor y = i8_out(what, x, w.n, out, dtype, x.scalar_type());
    const Rows o = rows_of("linear_i8: out", y, w.n);
    size_t need = 0;
    check_rc(gfl_i8_workspace(r.n, w.n, K, nullptr, &need));
    const Tensor ws = workspace(need, x);
    check_rc(gfl_linear_i8(x.data_ptr(), r.ld, code, b.data_ptr<int8_t>(), w.ld, sb.data_ptr<float>(), r.n, w.n, K, y.data_ptr(),
                           o.ld, code_of(y.scalar_type()), addr(ws), need, on.stream));
    written(out);
    return y;
}

int dtype_code(const char* what, const char* name, const Tensor& t)
{
    const int code = code_of(t.scalar_type());
    TORCH_CHECK_VALUE(code >= 0, what, ": ", name, " must be fp32, fp16 or bf16");
    return code;
}

// a 4-bit weight: q [N, ceil(K / 128) * 64], scale (and zero) [ceil(K / group), N]
struct I4
{
    int N, K, group, scale_code;
    I4(const char* what, const Tensor& q, const Tensor& scale, const OptTensor& zero, int64_t k, int64_t g)
    {
        TORCH_CHECK_VALUE(g == 32 || g == 64 || g == 128, what, ": group must be 32, 64 or 128");
        TORCH_CHECK_VALUE(k >= 1 && k < GFL_MAX_LD, what, ": K must be in 1..", GFL_MAX_LD - 1);
        K = static_cast<int>(k);
        group = static_cast<int>(g);
        const int64_t blocks = (k + 127) / 128, groups = (k + g - 1) / g;
        TORCH_CHECK_VALUE(q.scalar_type() == at::kByte && q.dim() == 2 && q.is_contiguous() && q.size(1) == blocks * 64, what,
                          ": q must be contiguous uint8 [N, ", blocks * 64, "], as quant_i4 or pack_i4 made it for ", k, " inputs");
        N = size_of(what, q.size(0));
        scale_code = code_of(scale.scalar_type());
        TORCH_CHECK_VALUE((scale_code == GFL_F16 || scale_code == GFL_BF16) && scale.dim() == 2 && scale.size(0) == groups &&
                              scale.size(1) == N && scale.is_contiguous(),
                          what, ": scale must be contiguous fp16 or bf16 [", groups, ", ", N, "]");
        TORCH_CHECK_VALUE(!zero || (zero->scalar_type() == at::kByte && zero->sizes() == scale.sizes() && zero->is_contiguous()), what,
                          ": zero must be contiguous uint8 [", groups, ", ", N, "]");
    }
};

std::tuple<Tensor, Tensor, OptTensor> quant_i4(const Tensor& w, int64_t group, bool zeros)
{
    const char* what = "quant_i4";
    const int code = x16_code(what, w);
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 1, "quant_i4: the weight must be [N, K]");
    TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128, "quant_i4: group must be 32, 64 or 128");
    const int K = size_of(what, w.size(1));
    const Rows r = rows_of("quant_i4: the weight", w, K);
    const On on(what, w, {});
    const int64_t blocks = (static_cast<int64_t>(K) + 127) / 128, groups = (K + group - 1) / group;
    Tensor q = at::empty({ r.n, blocks * 64 }, w.options().dtype(at::kByte));
    Tensor scale = at::empty({ groups, r.n }, w.options());
    const OptTensor zero = zeros ? OptTensor(at::empty({ groups, r.n }, q.options())) : OptTensor();
    check_rc(gfl_quant_i4(w.data_ptr(), r.ld, code, r.n, K, static_cast<int>(group), q.data_ptr<uint8_t>(), scale.data_ptr(),
                          addr<uint8_t>(zero), on.stream));
    return { q, scale, zero };
}

Tensor pack_i4(const Tensor& v)
{
    const char* what = "pack_i4";
    TORCH_CHECK_VALUE(v.scalar_type() == at::kByte && v.dim() == 2 && v.size(0) >= 1 && v.size(1) >= 1,
                      "pack_i4: the values must be uint8 [N, K]");
    const int K = size_of(what, v.size(1));
    const Rows r = rows_of("pack_i4: the values", v, K);
    const On on(what, v, {});
    Tensor q = at::empty({ r.n, (static_cast<int64_t>(K) + 127) / 128 * 64 }, v.options());
    check_rc(gfl_pack_i4(v.data_ptr<uint8_t>(), r.ld, r.n, K, q.data_ptr<uint8_t>(), on.stream));
    return q;
}

Tensor linear_i4(const Tensor& x, const Tensor& q, const Tensor& scale, const OptTensor& zero, int64_t group, const OptTensor& out,
                 std::optional<at::ScalarType> dtype)
{
    const char* what = "linear_i4";
    const int code = x16_code(what, x);
    const I4 w(what, q, scale, zero, x.size(-1), group);
    const Rows r = rows_of("linear_i4: x", x, w.K);
    const On on(what, x, { &q, &scale, ptr(zero), ptr(out) });
    const Tensor y = i8_out(what, x, w.N, out, dtype, x.scalar_type());
    const Rows o = rows_of("linear_i4: out", y, w.N);
    const int ycode = code_of(y.scalar_type());
    size_t need = 0;
    check_rc(gfl_i4_workspace(code, ycode, r.n, w.N, w.K, w.group, &need, nullptr));
    const Tensor ws = workspace(need, x);
    check_rc(gfl_linear_i4(x.data_ptr(), r.ld, code, q.data_ptr<uint8_t>(), scale.data_ptr(), w.scale_code, addr<uint8_t>(zero), r.n,
                           w.N, w.K, w.group, y.data_ptr(), o.ld, ycode, addr(ws), need, on.stream));
    written(out);
    return y;
}

Tensor linear_i4_dx(const Tensor& dy, const Tensor& q, const Tensor& scale, int64_t K, const OptTensor& zero, int64_t group)
{
    const char* what = "linear_i4_dx";
    const int code = code_of(dy.scalar_type());
    TORCH_CHECK_VALUE((code == GFL_F16 || code == GFL_BF16) && dy.dim() >= 1, "linear_i4_dx: dy must be fp16 or bf16 [..., N]");
    const I4 w(what, q, scale, zero, K, group);
    const Rows r = rows_of("linear_i4_dx: dy", dy, w.N);
    const On on(what, dy, { &q, &scale, ptr(zero) });
    at::DimVector shape(dy.sizes());
    shape.back() = w.K;
    Tensor dx = at::empty(shape, dy.options());
    size_t need = 0;
    check_rc(gfl_i4_workspace(code, code, r.n, w.N, w.K, w.group, nullptr, &need));
    const Tensor ws = workspace(need, dy);
    check_rc(gfl_linear_i4_dx(dy.data_ptr(), r.ld, code, q.data_ptr<uint8_t>(), scale.data_ptr(), w.scale_code, addr<uint8_t>(zero),
                              r.n, w.N, w.K, w.group, dx.data_ptr(), w.K, addr(ws), need, on.stream));
    return dx;
}

int score_code(const char* what, const std::string& score)
{
    TORCH_CHECK_VALUE(score == "sigmoid" || score == "softmax", what, ": score must be 'sigmoid' or 'softmax'");
    return score == "softmax" ? GFL_SOFTMAX : GFL_SIGMOID;
}

std::tuple<Tensor, Tensor> route_experts(const Tensor& logits, int64_t topk, const OptTensor& bias, const std::string& score,
                                         int64_t groups, int64_t top_groups, int64_t group_best, bool renorm, double scale,
                                         std::optional<at::ScalarType> dtype)
{
    const char* what = "route_experts";
    TORCH_CHECK_VALUE(logits.dim() == 2, "route_experts: logits must be [M, E]");
    const int code = dtype_code(what, "logits", logits), E = size_of(what, logits.size(1)), k = size_of(what, topk);
    const Rows r = rows_of("route_experts: logits", logits, E);
    TORCH_CHECK_VALUE(!bias || (bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == E && bias->is_contiguous()),
                      "route_experts: bias must be contiguous fp32 [", E, "]");
    TORCH_CHECK_VALUE(topk >= 1 && topk <= 64 && groups >= 1 && groups <= E && top_groups >= 1 && top_groups <= groups && group_best >= 1 &&
                          group_best <= 2,
                      "route_experts: need topk in 1..64, 1 <= top_groups <= groups <= E and group_best 1 or 2");
    const int by = score_code(what, score);
    const On on(what, logits, { ptr(bias) });
    Tensor sel = at::empty({ r.n, topk }, logits.options().dtype(at::kLong));
    Tensor w = at::empty({ r.n, topk }, logits.options().dtype(dtype.value_or(at::kHalf)));
    check_rc(gfl_route_experts(logits.data_ptr(), r.ld, code, addr<float>(bias), r.n, E, k, by, static_cast<int>(groups),
                               static_cast<int>(top_groups), static_cast<int>(group_best), renorm, static_cast<float>(scale),
                               sel.data_ptr<int64_t>(), w.data_ptr(), dtype_code(what, "dtype", w), on.stream));
    return { sel, w };
}

Tensor route_experts_backward(const Tensor& dw, const Tensor& logits, const Tensor& sel, const std::string& score, bool renorm,
                              double scale)
{
    const char* what = "route_experts_backward";
    TORCH_CHECK_VALUE(logits.dim() == 2, "route_experts_backward: logits must be [M, E]");
    const int code = dtype_code(what, "logits", logits), E = size_of(what, logits.size(1)), wcode = dtype_code(what, "dw", dw);
    const Rows r = rows_of("route_experts_backward: logits", logits, E);
    TORCH_CHECK_VALUE(sel.scalar_type() == at::kLong && sel.dim() == 2 && sel.size(0) == r.n && sel.is_contiguous(),
                      "route_experts_backward: sel must be contiguous int64 [", r.n, ", topk]");
    TORCH_CHECK_VALUE(dw.sizes() == sel.sizes() && dw.is_contiguous(), "route_experts_backward: dw must be contiguous, of sel's shape");
    const int by = score_code(what, score);
    const On on(what, logits, { &dw, &sel });
    Tensor dx = at::empty(logits.sizes(), logits.options());
    check_rc(gfl_route_experts_backward(dw.data_ptr(), wcode, logits.data_ptr(), r.ld, code, sel.data_ptr<int64_t>(), r.n, E,
                                        size_of(what, sel.size(1)), by, renorm, static_cast<float>(scale), dx.data_ptr(), E,
                                        on.stream));
    return dx;
}

Tensor adjust_logits(const Tensor& logits, const OptTensor& history, const OptTensor& lengths, const OptTensor& prompt,
                     const OptTensor& repetition, const OptTensor& frequency, const OptTensor& presence, const OptTensor& bias_ids,
                     const OptTensor& bias, const OptTensor& allowed, const OptTensor& out)
{
    const char* what = "adjust_logits";
    TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) >= 1, "adjust_logits: logits must be [B, V]");
    const int code = dtype_code(what, "logits", logits), V = size_of(what, logits.size(1));
    const Rows r = rows_of("adjust_logits: logits", logits, V);
    auto per_row = [&](const char* name, const Tensor* t, at::ScalarType type) {
        TORCH_CHECK_VALUE(!t || (t->scalar_type() == type && t->dim() == 1 && t->size(0) == r.n && t->is_contiguous()),
                          "adjust_logits: ", name, " must be contiguous ", type, " [", r.n, "]");
    };
    auto rows = [&](const char* name, const Tensor* t, at::ScalarType type, int64_t cols) {
        if (!t) return Rows{ 0, 0 };
        TORCH_CHECK_VALUE(t->scalar_type() == type && t->dim() == 2 && t->size(0) == r.n && t->size(1) == cols, "adjust_logits: ", name,
                          " must be ", type, " [", r.n, ", ", cols, "]");
        return rows_of(name, *t, cols);
    };
    const int64_t L = history && history->dim() == 2 ? history->size(1) : 0, n = bias_ids && bias_ids->dim() == 2 ? bias_ids->size(1) : 0;
    const Rows h = rows("history", ptr(history), at::kInt, L);
    per_row("lengths", ptr(lengths), at::kInt);
    per_row("prompt", ptr(prompt), at::kInt);
    per_row("repetition", ptr(repetition), at::kFloat);
    per_row("frequency", ptr(frequency), at::kFloat);
    per_row("presence", ptr(presence), at::kFloat);
    TORCH_CHECK_VALUE(history || !(lengths || prompt || repetition || frequency || presence),
                      "adjust_logits: lengths, prompt and penalties need a history");
    TORCH_CHECK_VALUE(!bias_ids == !bias, "adjust_logits: bias_ids and bias are given together");
    const Rows bi = rows("bias_ids", ptr(bias_ids), at::kInt, n), bv = rows("bias", ptr(bias), at::kFloat, n);
    const Rows m = rows("allowed", ptr(allowed), at::kInt, (static_cast<int64_t>(V) + 31) / 32);
    TORCH_CHECK_VALUE(!out || (out->sizes() == logits.sizes() && out->scalar_type() == logits.scalar_type()),
                      "adjust_logits: out must be of logits' shape and type");
    const On on(what, logits, { ptr(history), ptr(lengths), ptr(prompt), ptr(repetition), ptr(frequency), ptr(presence),
                                ptr(bias_ids), ptr(bias), ptr(allowed), ptr(out) });
    const Tensor y = out ? *out : at::empty(logits.sizes(), logits.options());
    const Rows o = rows_of("adjust_logits: out", y, V);
    // a history of no columns has no address
    check_rc(gfl_adjust_logits(logits.data_ptr(), r.ld, code, r.n, V, L ? addr<int32_t>(history) : nullptr, h.ld, size_of(what, L),
                               L ? addr<int32_t>(lengths) : nullptr, L ? addr<int32_t>(prompt) : nullptr,
                               L ? addr<float>(repetition) : nullptr, L ? addr<float>(frequency) : nullptr,
                               L ? addr<float>(presence) : nullptr, addr<int32_t>(bias_ids), bi.ld, addr<float>(bias), bv.ld,
                               size_of(what, n), addr<int32_t>(allowed), m.ld, y.data_ptr(), o.ld, on.stream));
    written(out);
    return y;
}

std::tuple<Tensor, Tensor> sample(const Tensor& logits, const Tensor& u, const OptTensor& temperature, const OptTensor& top_k,
                                  const OptTensor& top_p, const OptTensor& min_p)
{
    const char* what = "sample";
    const int code = code_of(logits.scalar_type());
    TORCH_CHECK_VALUE(logits.dim() == 2 && code >= 0 && logits.size(1) >= 1, "sample: logits must be fp32, fp16 or bf16 [B, V]");
    const int V = size_of(what, logits.size(1));
    const Rows r = rows_of("sample: logits", logits, V);
    auto per_row = [&](const char* name, const Tensor* t, at::ScalarType type) {
        TORCH_CHECK_VALUE(!t || (t->scalar_type() == type && t->dim() == 1 && t->size(0) == r.n && t->is_contiguous()), "sample: ",
                          name, " must be contiguous ", type, " [", r.n, "]");
    };
    per_row("u", &u, at::kFloat);
    per_row("temperature", ptr(temperature), at::kFloat);
    per_row("top_k", ptr(top_k), at::kInt);
    per_row("top_p", ptr(top_p), at::kFloat);
    per_row("min_p", ptr(min_p), at::kFloat);
    const On on(what, logits, { &u, ptr(temperature), ptr(top_k), ptr(top_p), ptr(min_p) });
    Tensor token = at::empty({ r.n }, logits.options().dtype(at::kLong));
    Tensor prob = at::empty({ r.n }, logits.options().dtype(at::kFloat));
    size_t need = 0;
    check_rc(gfl_sample_workspace(r.n, V, &need));
    const Tensor ws = workspace(need, logits);
    check_rc(gfl_sample(logits.data_ptr(), r.ld, code, r.n, V, addr<float>(temperature), addr<int32_t>(top_k), addr<float>(top_p),
                        addr<float>(min_p), u.data_ptr<float>(), token.data_ptr<int64_t>(), prob.data_ptr<float>(), addr(ws),
                        need, on.stream));
    return { token, prob };
}

}  // namespace

void bind_dense(pybind11::module& m)
{
    m.def("ffn_forward", &ffn_forward);
    m.def("ffn_backward", &ffn_backward);
    m.def("quant_i8", &quant_i8);
    m.def("gemm_i8", &gemm_i8);
    m.def("linear_i8", &linear_i8);
    m.def("quant_i4", &quant_i4);
    m.def("pack_i4", &pack_i4);
    m.def("linear_i4", &linear_i4);
    m.def("linear_i4_dx", &linear_i4_dx);
    m.def("route_experts", &route_experts);
    m.def("route_experts_backward", &route_experts_backward);
    m.def("adjust_logits", &adjust_logits);
    m.def("sample", &sample);
}
