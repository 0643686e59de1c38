// PyTorch extension: torch.ops.hfuse_b200.* for the five DL kernels, their ten fused pairs and the
// language-model operators.
//
// Stands in for the torch C++ extension the reference's Python harness calls
// (TorchKernel's build.sh / call_{1080,v100}.py, README.md:68,84-95 of aoli-al/HFuse).  It only
// checks tensors, allocates the outputs and forwards raw pointers plus the current stream to the C
// ABI in include/hfuse_b200.h; all device code lives in libhfuse_b200.so.  CUDA tensors only.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <optional>
#include <tuple>

#include "../../include/hfuse_b200.h"

namespace {

using at::Tensor;
using IntList = at::IntArrayRef;

void check_in(const Tensor& t, const char* what, int dims = -1) {
    TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor: hfuse_b200 has no CPU path");
    TORCH_CHECK(t.scalar_type() == at::kFloat, what, " must be float32");
    TORCH_CHECK(t.is_contiguous(), what, " must be contiguous (NCHW)");
    TORCH_CHECK(dims < 0 || t.dim() == dims, what, " must be ", dims, "-D");
}
void ok(int rc, const char* fn) { TORCH_CHECK(rc == HFUSE_OK, fn, ": ", hfuse_error_string(rc), " (", rc, ")"); }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
int i32(int64_t v) { return static_cast<int>(v); }

// ---- one descriptor per operator: shapes, outputs, and the C-ABI argument values -------------------
struct Im2col {
    Tensor x, col;
    int N, C, H, W, kh, kw, ph, pw, sh, sw, dh, dw;
    Im2col(const Tensor& x_, IntList k, IntList p, IntList s, IntList d) : x(x_) {
        check_in(x, "im2col input", 4);
        TORCH_CHECK(k.size() == 2 && p.size() == 2 && s.size() == 2 && d.size() == 2, "im2col: 2-element lists expected");
        N = i32(x.size(0)); C = i32(x.size(1)); H = i32(x.size(2)); W = i32(x.size(3));
        kh = i32(k[0]); kw = i32(k[1]); ph = i32(p[0]); pw = i32(p[1]); sh = i32(s[0]); sw = i32(s[1]); dh = i32(d[0]); dw = i32(d[1]);
        TORCH_CHECK(sh > 0 && sw > 0 && dh > 0 && dw > 0 && kh > 0 && kw > 0, "im2col: bad kernel/stride/dilation");
        const int64_t Hc = (H + 2 * ph - (dh * (kh - 1) + 1)) / sh + 1, Wc = (W + 2 * pw - (dw * (kw - 1) + 1)) / sw + 1;
        TORCH_CHECK(Hc > 0 && Wc > 0, "im2col: kernel does not fit the padded input");
        col = at::empty({N, (int64_t)C * kh * kw, Hc * Wc}, x.options());
    }
};
#define IM2COL_ARGS(o) (o).x.data_ptr<float>(), (o).N, (o).C, (o).H, (o).W, (o).kh, (o).kw, (o).ph, (o).pw, (o).sh, (o).sw, (o).dh, (o).dw, (o).col.data_ptr<float>()

struct MaxPool {
    Tensor x, out, idx;
    int N, C, H, W, pH, pW, kh, kw, sh, sw, ph, pw, dh, dw;
    MaxPool(const Tensor& x_, IntList k, IntList s, IntList p, IntList d) : x(x_) {
        check_in(x, "max_pool input", 4);
        TORCH_CHECK(k.size() == 2 && p.size() == 2 && s.size() == 2 && d.size() == 2, "max_pool: 2-element lists expected");
        N = i32(x.size(0)); C = i32(x.size(1)); H = i32(x.size(2)); W = i32(x.size(3));
        kh = i32(k[0]); kw = i32(k[1]); sh = i32(s[0]); sw = i32(s[1]); ph = i32(p[0]); pw = i32(p[1]); dh = i32(d[0]); dw = i32(d[1]);
        TORCH_CHECK(sh > 0 && sw > 0 && dh > 0 && dw > 0 && kh > 0 && kw > 0, "max_pool: bad kernel/stride/dilation");
        pH = (H + 2 * ph - dh * (kh - 1) - 1) / sh + 1; pW = (W + 2 * pw - dw * (kw - 1) - 1) / sw + 1;
        TORCH_CHECK(pH > 0 && pW > 0, "max_pool: window does not fit the padded input");
        out = at::empty({N, C, pH, pW}, x.options());
        idx = at::empty({N, C, pH, pW}, x.options().dtype(at::kLong));
    }
};
#define MAXPOOL_ARGS(o) (o).x.data_ptr<float>(), (o).N, (o).C, (o).H, (o).W, (o).pH, (o).pW, (o).kh, (o).kw, (o).sh, (o).sw, (o).ph, (o).pw, (o).dh, (o).dw, (o).out.data_ptr<float>(), (o).idx.data_ptr<int64_t>()

// zero-initialised scratch for the statistics kernel, one per (device, stream, channels)
Tensor bn_workspace(const Tensor& like, int C) {
    static std::mutex mu;
    static std::map<std::tuple<int, void*, int>, Tensor> cache;
    std::lock_guard<std::mutex> lk(mu);
    auto key = std::make_tuple((int)like.get_device(), stream(), C);
    auto it = cache.find(key);
    if (it == cache.end())
        it = cache.emplace(key, at::zeros({(int64_t)hfuse_bnstats_workspace_bytes(1, C, 1)}, like.options().dtype(at::kByte))).first;
    return it->second;
}
struct BnStats {
    Tensor x, mean, invstd, ws;
    int N, C, HW;
    float eps;
    BnStats(const Tensor& x_, double eps_) : x(x_), eps((float)eps_) {
        check_in(x, "batch_norm input");
        TORCH_CHECK(x.dim() >= 2 && x.numel() > 0, "batch_norm input must have at least 2 dimensions and be non-empty");
        N = i32(x.size(0)); C = i32(x.size(1)); HW = i32(x.numel() / ((int64_t)N * C));
        mean = at::empty({C}, x.options()); invstd = at::empty({C}, x.options());
        ws = bn_workspace(x, C);
    }
};
#define BNSTATS_ARGS(o) (o).x.data_ptr<float>(), (o).N, (o).C, (o).HW, (o).eps, (o).mean.data_ptr<float>(), (o).invstd.data_ptr<float>(), (double*)nullptr, (o).ws.data_ptr(), (size_t)(o).ws.numel()

struct Upsample {
    Tensor x, out;
    int N, C, H, W, oH, oW, align;
    Upsample(const Tensor& x_, IntList size, bool align_corners) : x(x_), align(align_corners) {
        check_in(x, "upsample input", 4);
        TORCH_CHECK(size.size() == 2 && size[0] > 0 && size[1] > 0, "upsample: output size must be two positive ints");
        N = i32(x.size(0)); C = i32(x.size(1)); H = i32(x.size(2)); W = i32(x.size(3)); oH = i32(size[0]); oW = i32(size[1]);
        out = at::empty({N, C, oH, oW}, x.options());
    }
};
#define UPSAMPLE_ARGS(o) (o).x.data_ptr<float>(), (o).N, (o).C, (o).H, (o).W, (o).oH, (o).oW, (o).align, (o).out.data_ptr<float>()

struct Histc {
    Tensor x, counts;
    int64_t n;
    int bins;
    float lo, hi;
    Histc(const Tensor& x_, int64_t bins_, double lo_, double hi_) : x(x_), n(x_.numel()), bins(i32(bins_)), lo((float)lo_), hi((float)hi_) {
        check_in(x, "histc input");
        TORCH_CHECK(bins > 0, "histc: bins must be positive");
        TORCH_CHECK(lo < hi, "histc: max must be larger than min");
        counts = at::empty({bins}, x.options().dtype(at::kInt));      // uint32 counts in int32 storage
    }
};
#define HISTC_ARGS(o) (o).n ? (o).x.data_ptr<float>() : nullptr, (o).n, (o).bins, (o).lo, (o).hi, (uint32_t*)(o).counts.data_ptr<int>()

// ---- standalone operators -----------------------------------------------------------------------------
Tensor im2col(const Tensor& x, IntList k, IntList p, IntList s, IntList d) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Im2col a(x, k, p, s, d);
    ok(hfuse_im2col_f32(IM2COL_ARGS(a), stream()), "hfuse_im2col_f32");
    return a.col;
}
std::tuple<Tensor, Tensor> max_pool2d_with_indices(const Tensor& x, IntList k, IntList s, IntList p, IntList d) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    MaxPool a(x, k, s, p, d);
    ok(hfuse_maxpool2d_f32(MAXPOOL_ARGS(a), stream()), "hfuse_maxpool2d_f32");
    return {a.out, a.idx};
}
std::tuple<Tensor, Tensor> batch_norm_stats(const Tensor& x, double eps) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    BnStats a(x, eps);
    ok(hfuse_bnstats_f32(BNSTATS_ARGS(a), stream()), "hfuse_bnstats_f32");
    return {a.mean, a.invstd};
}
Tensor upsample_bilinear2d(const Tensor& x, IntList size, bool align_corners) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Upsample a(x, size, align_corners);
    ok(hfuse_upsample_bilinear2d_f32(UPSAMPLE_ARGS(a), stream()), "hfuse_upsample_bilinear2d_f32");
    return a.out;
}
Tensor histc(const Tensor& x, int64_t bins, double lo, double hi) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Histc a(x, bins, lo, hi);
    ok(hfuse_histc_f32(HISTC_ARGS(a), stream()), "hfuse_histc_f32");
    return a.counts;
}

// ---- fused pairs: K1's arguments, then K2's; outputs in the same order ---------------------------------
std::tuple<Tensor, Tensor, Tensor> im2col_maxpool(const Tensor& x, IntList k, IntList p, IntList s, IntList d,
                                                  const Tensor& y, IntList k2, IntList s2, IntList p2, IntList d2) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Im2col a(x, k, p, s, d); MaxPool b(y, k2, s2, p2, d2);
    ok(hfuse_im2col_maxpool_f32(IM2COL_ARGS(a), MAXPOOL_ARGS(b), stream()), "hfuse_im2col_maxpool_f32");
    return {a.col, b.out, b.idx};
}
std::tuple<Tensor, Tensor, Tensor> im2col_bnstats(const Tensor& x, IntList k, IntList p, IntList s, IntList d,
                                                  const Tensor& y, double eps) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Im2col a(x, k, p, s, d); BnStats b(y, eps);
    ok(hfuse_im2col_bnstats_f32(IM2COL_ARGS(a), BNSTATS_ARGS(b), stream()), "hfuse_im2col_bnstats_f32");
    return {a.col, b.mean, b.invstd};
}
std::tuple<Tensor, Tensor> im2col_histc(const Tensor& x, IntList k, IntList p, IntList s, IntList d, const Tensor& y,
                                        int64_t bins, double lo, double hi) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Im2col a(x, k, p, s, d); Histc b(y, bins, lo, hi);
    ok(hfuse_im2col_histc_f32(IM2COL_ARGS(a), HISTC_ARGS(b), stream()), "hfuse_im2col_histc_f32");
    return {a.col, b.counts};
}
std::tuple<Tensor, Tensor> im2col_upsample(const Tensor& x, IntList k, IntList p, IntList s, IntList d, const Tensor& y,
                                           IntList size, bool align_corners) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Im2col a(x, k, p, s, d); Upsample b(y, size, align_corners);
    ok(hfuse_im2col_upsample_f32(IM2COL_ARGS(a), UPSAMPLE_ARGS(b), stream()), "hfuse_im2col_upsample_f32");
    return {a.col, b.out};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> maxpool_bnstats(const Tensor& x, IntList k, IntList s, IntList p, IntList d,
                                                           const Tensor& y, double eps) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    MaxPool a(x, k, s, p, d); BnStats b(y, eps);
    ok(hfuse_maxpool_bnstats_f32(MAXPOOL_ARGS(a), BNSTATS_ARGS(b), stream()), "hfuse_maxpool_bnstats_f32");
    return {a.out, a.idx, b.mean, b.invstd};
}
std::tuple<Tensor, Tensor, Tensor> maxpool_upsample(const Tensor& x, IntList k, IntList s, IntList p, IntList d,
                                                    const Tensor& y, IntList size, bool align_corners) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    MaxPool a(x, k, s, p, d); Upsample b(y, size, align_corners);
    ok(hfuse_maxpool_upsample_f32(MAXPOOL_ARGS(a), UPSAMPLE_ARGS(b), stream()), "hfuse_maxpool_upsample_f32");
    return {a.out, a.idx, b.out};
}
std::tuple<Tensor, Tensor, Tensor> histc_maxpool(const Tensor& x, int64_t bins, double lo, double hi, const Tensor& y,
                                                 IntList k, IntList s, IntList p, IntList d) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Histc a(x, bins, lo, hi); MaxPool b(y, k, s, p, d);
    ok(hfuse_histc_maxpool_f32(HISTC_ARGS(a), MAXPOOL_ARGS(b), stream()), "hfuse_histc_maxpool_f32");
    return {a.counts, b.out, b.idx};
}
std::tuple<Tensor, Tensor> histc_upsample(const Tensor& x, int64_t bins, double lo, double hi, const Tensor& y, IntList size,
                                          bool align_corners) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Histc a(x, bins, lo, hi); Upsample b(y, size, align_corners);
    ok(hfuse_histc_upsample_f32(HISTC_ARGS(a), UPSAMPLE_ARGS(b), stream()), "hfuse_histc_upsample_f32");
    return {a.counts, b.out};
}
std::tuple<Tensor, Tensor, Tensor> upsample_bnstats(const Tensor& x, IntList size, bool align_corners, const Tensor& y,
                                                    double eps) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Upsample a(x, size, align_corners); BnStats b(y, eps);
    ok(hfuse_upsample_bnstats_f32(UPSAMPLE_ARGS(a), BNSTATS_ARGS(b), stream()), "hfuse_upsample_bnstats_f32");
    return {a.out, b.mean, b.invstd};
}
std::tuple<Tensor, Tensor, Tensor> histc_bnstats(const Tensor& x, int64_t bins, double lo, double hi, const Tensor& y,
                                                 double eps) {
    check_in(x, "first input");
    c10::cuda::CUDAGuard g(x.device());
    Histc a(x, bins, lo, hi); BnStats b(y, eps);
    ok(hfuse_histc_bnstats_f32(HISTC_ARGS(a), BNSTATS_ARGS(b), stream()), "hfuse_histc_bnstats_f32");
    return {a.counts, b.mean, b.invstd};
}

// ---- operators of a language model's token path ---------------------------------------------------------
using OptTensor = const std::optional<Tensor>&;

// These operators are called for single tokens too, where the host's time counts: no dispatch for each buffer (a layer norm of
// one row 7.8 us a call instead of 8.9, a recurrence step 7.1 instead of 8.1).  Dispatch modes do not see these buffers.
Tensor buffer(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

int lm_type(const Tensor& t, const char* what) {
    TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor: hfuse_b200 has no CPU path");
    switch (t.scalar_type()) {
    case at::kFloat: return HFUSE_F32;
    case at::kBFloat16: return HFUSE_BF16;
    case at::kHalf: return HFUSE_F16;
    default: break;
    }
    TORCH_CHECK(false, what, " must be float32, bfloat16 or float16");
    return -1;
}
void check_unit(const Tensor& t, const char* what) {
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, what, " must have a last dimension of at least 1");
    TORCH_CHECK(t.size(-1) == 1 || t.stride(-1) == 1, what, " must have stride 1 in its last dimension");
    TORCH_CHECK(t.size(-1) <= INT32_MAX, what, " has too long rows");
}
void check_like(const Tensor& t, const Tensor& like, at::ScalarType type, const char* what) {
    TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor: hfuse_b200 has no CPU path");
    TORCH_CHECK(t.device() == like.device(), what, " must be on ", like.device(), ", is on ", t.device());
    TORCH_CHECK(t.scalar_type() == type, what, " must be ", type, ", is ", t.scalar_type());
}
void check_vec(const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef shape, const char* what) {
    check_like(t, like, type, what);
    TORCH_CHECK(t.sizes() == shape, what, " must have shape ", shape, ", has ", t.sizes());
    TORCH_CHECK(t.is_contiguous(), what, " must be contiguous");
}
const void* opt_ptr(OptTensor t) { return t ? t->data_ptr() : nullptr; }
const float* opt_f32(OptTensor t) { return t ? t->data_ptr<float>() : nullptr; }

// elements between two rows (all dimensions but the last, which must follow each other evenly)
int64_t row_stride(const Tensor& t, const char* what) {
    int64_t ld = -1, span = 0;
    if (t.numel() == 0) return t.size(-1);
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (ld < 0) ld = t.stride(d);
        else TORCH_CHECK(t.stride(d) == span, what, " must have rows that are evenly spaced in memory");
        span = t.stride(d) * t.size(d);
    }
    if (ld < 0) return t.size(-1);
    TORCH_CHECK(ld >= t.size(-1), what, " must have rows that do not overlap");
    return ld;
}
// type of weight and bias (the input's where there is neither)
at::ScalarType norm_params(const Tensor& x, OptTensor weight, OptTensor bias) {
    const auto type = weight ? weight->scalar_type() : bias ? bias->scalar_type() : x.scalar_type();
    TORCH_CHECK(type == x.scalar_type() || type == at::kFloat, "weight and bias must have the input's type or float32");
    const int64_t D[1] = {x.size(-1)};
    if (weight) check_vec(*weight, x, type, D, "weight");
    if (bias) check_vec(*bias, x, type, D, "bias");
    return type;
}
int code_of(at::ScalarType t) { return t == at::kFloat ? HFUSE_F32 : t == at::kBFloat16 ? HFUSE_BF16 : HFUSE_F16; }

std::tuple<Tensor, Tensor, Tensor> layer_norm(const Tensor& x, OptTensor weight, OptTensor bias, double eps) {
    const int type = lm_type(x, "layer_norm input");
    check_unit(x, "layer_norm input");
    TORCH_CHECK(eps >= 0, "layer_norm: eps must not be negative");
    const auto wt = norm_params(x, weight, bias);
    const int64_t D = x.size(-1), ld = row_stride(x, "layer_norm input");
    c10::cuda::CUDAGuard g(x.device());
    Tensor y = buffer(x.sizes(), x.scalar_type(), x);
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    Tensor mean = buffer(lead, at::kFloat, x), invstd = buffer(lead, at::kFloat, x);
    ok(hfuse_layernorm(x.data_ptr(), x.numel() / D, i32(D), ld, type, opt_ptr(weight), opt_ptr(bias), code_of(wt), (float)eps,
                       y.data_ptr(), mean.data_ptr<float>(), invstd.data_ptr<float>(), stream()), "hfuse_layernorm");
    return {y, mean, invstd};
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& x, const Tensor& grad_out, const Tensor& mean,
                                                       const Tensor& invstd, OptTensor weight) {
    const int type = lm_type(x, "layer_norm input");
    check_unit(x, "layer_norm input");
    check_like(grad_out, x, x.scalar_type(), "layer_norm grad_out");
    TORCH_CHECK(grad_out.sizes() == x.sizes(), "layer_norm grad_out must have the shape of the input");
    check_unit(grad_out, "layer_norm grad_out");
    check_vec(mean, x, at::kFloat, x.sizes().slice(0, x.dim() - 1), "mean");
    check_vec(invstd, x, at::kFloat, x.sizes().slice(0, x.dim() - 1), "invstd");
    const auto wt = norm_params(x, weight, std::nullopt);
    const int64_t D = x.size(-1), rows = x.numel() / D;
    const int64_t ldx = row_stride(x, "layer_norm input"), ldg = row_stride(grad_out, "layer_norm grad_out");
    c10::cuda::CUDAGuard g(x.device());
    Tensor dx = buffer(x.sizes(), x.scalar_type(), x), dw = buffer({D}, wt, x), db = buffer({D}, wt, x);
    Tensor ws = buffer({(int64_t)hfuse_layernorm_backward_workspace_bytes(rows, i32(D))}, at::kByte, x);
    ok(hfuse_layernorm_backward(x.data_ptr(), ldx, grad_out.data_ptr(), ldg, rows, i32(D), type, mean.data_ptr<float>(),
                                invstd.data_ptr<float>(), opt_ptr(weight), code_of(wt), dx.data_ptr(), dw.data_ptr(),
                                db.data_ptr(), ws.data_ptr(), (size_t)ws.numel(), stream()), "hfuse_layernorm_backward");
    return {dx, dw, db};
}

void check_ids(const Tensor& ids, const Tensor& like) {
    TORCH_CHECK(ids.is_cuda(), "ids must be a CUDA tensor: hfuse_b200 has no CPU path");
    TORCH_CHECK(ids.device() == like.device(), "ids must be on ", like.device(), ", is on ", ids.device());
    TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "ids must be int64 or int32");
    TORCH_CHECK(ids.is_contiguous(), "ids must be contiguous");
}
Tensor embedding(const Tensor& table, const Tensor& ids, double scale) {
    const int type = lm_type(table, "embedding table");
    TORCH_CHECK(table.dim() == 2 && table.numel() > 0 && table.is_contiguous(), "embedding table must be 2-D, contiguous and not empty");
    TORCH_CHECK(table.size(1) <= INT32_MAX, "embedding table has too long rows");
    check_ids(ids, table);
    c10::cuda::CUDAGuard g(table.device());
    auto shape = ids.sizes().vec();
    shape.push_back(table.size(1));
    Tensor out = buffer(shape, table.scalar_type(), table);
    ok(hfuse_embedding(table.data_ptr(), table.size(0), i32(table.size(1)), type, ids.data_ptr(), ids.numel(),
                       i32(ids.element_size()), (float)scale, out.data_ptr(), stream()), "hfuse_embedding");
    return out;
}
Tensor embedding_backward(const Tensor& grad_out, const Tensor& ids, int64_t rows, double scale, int64_t padding_id) {
    const int type = lm_type(grad_out, "embedding grad_out");
    check_ids(ids, grad_out);
    TORCH_CHECK(grad_out.dim() == ids.dim() + 1 && grad_out.sizes().slice(0, ids.dim()) == ids.sizes() && grad_out.size(-1) >= 1,
                "embedding grad_out must have the shape of ids and one dimension more");
    TORCH_CHECK(grad_out.is_contiguous(), "embedding grad_out must be contiguous");
    TORCH_CHECK(rows >= 1, "embedding_backward: rows must be positive");
    const int64_t D = grad_out.size(-1), n = ids.numel();
    TORCH_CHECK(D <= INT32_MAX, "embedding grad_out has too long rows");
    c10::cuda::CUDAGuard g(grad_out.device());
    Tensor grad = buffer({rows, D}, grad_out.scalar_type(), grad_out);
    Tensor ws = buffer({(int64_t)hfuse_embedding_backward_workspace_bytes(n, rows, i32(D))}, at::kByte, grad_out);
    ok(hfuse_embedding_backward(grad_out.data_ptr(), ids.data_ptr(), n, i32(ids.element_size()), rows, i32(D), type, (float)scale,
                                padding_id, grad.data_ptr(), ws.data_ptr(), (size_t)ws.numel(), stream()),
       "hfuse_embedding_backward");
    return grad;
}

int check_steps(const Tensor& t, const char* what) {
    const int type = lm_type(t, what);
    TORCH_CHECK(t.dim() == 3 && t.numel() > 0, what, " must be 3-D and not empty");
    check_unit(t, what);
    return type;
}
void check_steps_like(const Tensor& t, const Tensor& like, const char* what) {
    check_like(t, like, like.scalar_type(), what);
    TORCH_CHECK(t.sizes() == like.sizes(), what, " must have shape ", like.sizes(), ", has ", t.sizes());
    check_unit(t, what);
}
std::tuple<Tensor, Tensor, Tensor> gated_recurrence(const Tensor& gate, const Tensor& x, OptTensor h0, bool save_states) {
    const int type = check_steps(gate, "gate");
    check_steps_like(x, gate, "x");
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), BD[2] = {B, D};
    if (h0) check_vec(*h0, x, at::kFloat, BD, "h0");
    c10::cuda::CUDAGuard g(x.device());
    Tensor out = buffer(x.sizes(), x.scalar_type(), x), last = buffer({B, D}, at::kFloat, x);
    Tensor states = save_states ? buffer({B, hfuse_gated_recurrence_chunks(T), D}, at::kFloat, x) : buffer({0}, at::kFloat, x);
    ok(hfuse_gated_recurrence(gate.data_ptr(), gate.stride(0), gate.stride(1), x.data_ptr(), x.stride(0), x.stride(1), B, T, i32(D),
                              type, opt_f32(h0), out.data_ptr(), last.data_ptr<float>(),
                              save_states ? states.data_ptr<float>() : nullptr, stream()), "hfuse_gated_recurrence");
    return {out, last, states};
}
std::tuple<Tensor, Tensor, Tensor> gated_recurrence_backward(const Tensor& gate, const Tensor& x, const Tensor& states,
                                                             const Tensor& grad_out, OptTensor grad_last) {
    const int type = check_steps(gate, "gate");
    check_steps_like(x, gate, "x");
    check_steps_like(grad_out, gate, "grad_out");
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), BD[2] = {B, D}, S[3] = {B, hfuse_gated_recurrence_chunks(T), D};
    check_vec(states, x, at::kFloat, S, "states");
    if (grad_last) check_vec(*grad_last, x, at::kFloat, BD, "grad_last");
    c10::cuda::CUDAGuard g(x.device());
    Tensor dgate = buffer(x.sizes(), x.scalar_type(), x), dx = buffer(x.sizes(), x.scalar_type(), x);
    Tensor dh0 = buffer({B, D}, at::kFloat, x);
    ok(hfuse_gated_recurrence_backward(gate.data_ptr(), gate.stride(0), gate.stride(1), x.data_ptr(), x.stride(0), x.stride(1),
                                       states.data_ptr<float>(), grad_out.data_ptr(), grad_out.stride(0), grad_out.stride(1),
                                       opt_f32(grad_last), B, T, i32(D), type, dgate.data_ptr(), dx.data_ptr(),
                                       dh0.data_ptr<float>(), stream()), "hfuse_gated_recurrence_backward");
    return {dgate, dx, dh0};
}

}  // namespace

TORCH_LIBRARY(hfuse_b200, m) {
    m.def("im2col(Tensor x, int[2] kernel_size, int[2] padding, int[2] stride, int[2] dilation) -> Tensor", &im2col);
    m.def("max_pool2d_with_indices(Tensor x, int[2] kernel_size, int[2] stride, int[2] padding, int[2] dilation) -> (Tensor, Tensor)", &max_pool2d_with_indices);
    m.def("batch_norm_stats(Tensor x, float eps) -> (Tensor, Tensor)", &batch_norm_stats);
    m.def("upsample_bilinear2d(Tensor x, int[2] output_size, bool align_corners) -> Tensor", &upsample_bilinear2d);
    m.def("histc(Tensor x, int bins, float min, float max) -> Tensor", &histc);
    m.def("im2col_maxpool(Tensor x, int[2] kernel_size, int[2] padding, int[2] stride, int[2] dilation, Tensor y, int[2] pool_kernel, int[2] pool_stride, int[2] pool_padding, int[2] pool_dilation) -> (Tensor, Tensor, Tensor)", &im2col_maxpool);
    m.def("im2col_bnstats(Tensor x, int[2] kernel_size, int[2] padding, int[2] stride, int[2] dilation, Tensor y, float eps) -> (Tensor, Tensor, Tensor)", &im2col_bnstats);
    m.def("im2col_histc(Tensor x, int[2] kernel_size, int[2] padding, int[2] stride, int[2] dilation, Tensor y, int bins, float min, float max) -> (Tensor, Tensor)", &im2col_histc);
    m.def("im2col_upsample(Tensor x, int[2] kernel_size, int[2] padding, int[2] stride, int[2] dilation, Tensor y, int[2] output_size, bool align_corners) -> (Tensor, Tensor)", &im2col_upsample);
    m.def("maxpool_bnstats(Tensor x, int[2] kernel_size, int[2] stride, int[2] padding, int[2] dilation, Tensor y, float eps) -> (Tensor, Tensor, Tensor, Tensor)", &maxpool_bnstats);
    m.def("maxpool_upsample(Tensor x, int[2] kernel_size, int[2] stride, int[2] padding, int[2] dilation, Tensor y, int[2] output_size, bool align_corners) -> (Tensor, Tensor, Tensor)", &maxpool_upsample);
    m.def("histc_maxpool(Tensor x, int bins, float min, float max, Tensor y, int[2] kernel_size, int[2] stride, int[2] padding, int[2] dilation) -> (Tensor, Tensor, Tensor)", &histc_maxpool);
    m.def("histc_upsample(Tensor x, int bins, float min, float max, Tensor y, int[2] output_size, bool align_corners) -> (Tensor, Tensor)", &histc_upsample);
    m.def("upsample_bnstats(Tensor x, int[2] output_size, bool align_corners, Tensor y, float eps) -> (Tensor, Tensor, Tensor)", &upsample_bnstats);
    m.def("histc_bnstats(Tensor x, int bins, float min, float max, Tensor y, float eps) -> (Tensor, Tensor, Tensor)", &histc_bnstats);
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)", &layer_norm);
    m.def("layer_norm_backward(Tensor x, Tensor grad_out, Tensor mean, Tensor invstd, Tensor? weight) -> (Tensor, Tensor, Tensor)", &layer_norm_backward);
    m.def("embedding(Tensor table, Tensor ids, float scale) -> Tensor", &embedding);
    m.def("embedding_backward(Tensor grad_out, Tensor ids, int rows, float scale, int padding_id) -> Tensor", &embedding_backward);
    m.def("gated_recurrence(Tensor gate, Tensor x, Tensor? h0, bool save_states) -> (Tensor, Tensor, Tensor)", &gated_recurrence);
    m.def("gated_recurrence_backward(Tensor gate, Tensor x, Tensor states, Tensor grad_out, Tensor? grad_last) -> (Tensor, Tensor, Tensor)", &gated_recurrence_backward);
}
