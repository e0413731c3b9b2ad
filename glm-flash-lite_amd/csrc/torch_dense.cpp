// The dense operators (include/gfl_moe.h: gfl_ffn_*, gfl_quant_i8, gfl_gemm_i8, gfl_linear_i8, gfl_sample) over torch tensors:
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
    m.def("sample", &sample);
}
