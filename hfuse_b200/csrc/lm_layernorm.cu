// Layer norm over the last dimension, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   forward   mu = sum x / D,  var = sum (x - mu)^2 / D,  r = 1 / sqrt(var + eps),  y = (x - mu) r w + b
//   backward  xh = (x - mu) r,  g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
#include "launch.cuh"
#include "lm_common.cuh"

using namespace hfuse;

namespace {

struct LnFwdArgs {
    const void *x, *w, *b;
    void* y;
    float *mean, *invstd;
    long long rows, ldx;
    int D;
    float inv_d, eps;
};

struct LnBwdArgs {
    const void *x, *dy, *w;
    const float *mean, *invstd;
    void *dx, *dw, *db;
    float* part;             // [slices][2][D]
    long long rows, ldx, lddy, slice_rows;
    int D, slices;
    float inv_d;
};

// ---- any width: one block per row, the row read again from L2 for each step ---------------------
template <class T, class W>
__global__ void __launch_bounds__(512) ln_fwd_wide(const LnFwdArgs a) {
    __shared__ float sh[16];
    const W* w = static_cast<const W*>(a.w);
    const W* b = static_cast<const W*>(a.b);
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        T* y = static_cast<T*>(a.y) + r * a.D;
        float s = 0.f;
        for (int i = threadIdx.x; i < a.D; i += blockDim.x) s += to_f32(x[i]);
        const float mu = block_sum(s, sh) * a.inv_d;
        float q = 0.f;
        for (int i = threadIdx.x; i < a.D; i += blockDim.x) {
            const float d = to_f32(x[i]) - mu;
            q = fmaf(d, d, q);
        }
        const float is = 1.f / sqrtf(fmaf(block_sum(q, sh), a.inv_d, a.eps));
        for (int i = threadIdx.x; i < a.D; i += blockDim.x)
            y[i] = from_f32<T>(fmaf((to_f32(x[i]) - mu) * is, w ? to_f32(w[i]) : 1.f, b ? to_f32(b[i]) : 0.f));
        if (threadIdx.x == 0) {
            a.mean[r] = mu;
            a.invstd[r] = is;
        }
    }
}

template <class T, class W>
__global__ void __launch_bounds__(512) ln_bwd_rows(const LnBwdArgs a) {
    __shared__ float sh[16];
    const W* w = static_cast<const W*>(a.w);
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
        T* dx = static_cast<T*>(a.dx) + r * a.D;
        const float mu = a.mean[r], is = a.invstd[r];
        float s = 0.f, d = 0.f;
        for (int i = threadIdx.x; i < a.D; i += blockDim.x) {
            const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.f);
            s += g;
            d = fmaf(g, (to_f32(x[i]) - mu) * is, d);
        }
        const float ms = block_sum(s, sh) * a.inv_d, md = block_sum(d, sh) * a.inv_d;
        for (int i = threadIdx.x; i < a.D; i += blockDim.x) {
            const float g = to_f32(dy[i]) * (w ? to_f32(w[i]) : 1.f);
            dx[i] = from_f32<T>(is * (g - ms - (to_f32(x[i]) - mu) * is * md));
        }
    }
}

// column sums of dy xh and dy over one slice of the rows
template <class T>
__global__ void __launch_bounds__(256) ln_bwd_cols(const LnBwdArgs a) {
    __shared__ float sw[8][32], sb[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + tx;
    const long long r0 = blockIdx.y * a.slice_rows, r1 = min(a.rows, r0 + a.slice_rows);
    float dw = 0.f, db = 0.f;
    if (c < a.D)
        for (long long r = r0 + ty; r < r1; r += 8) {
            const float dy = to_f32(static_cast<const T*>(a.dy)[r * a.lddy + c]);
            dw = fmaf(dy, (to_f32(static_cast<const T*>(a.x)[r * a.ldx + c]) - a.mean[r]) * a.invstd[r], dw);
            db += dy;
        }
    sw[ty][tx] = dw;
    sb[ty][tx] = db;
    __syncthreads();
    if (ty == 0 && c < a.D) {
        for (int k = 1; k < 8; ++k) {
            dw += sw[k][tx];
            db += sb[k][tx];
        }
        a.part[(2LL * blockIdx.y) * a.D + c] = dw;
        a.part[(2LL * blockIdx.y + 1) * a.D + c] = db;
    }
}

// the slices' sums, added in slice order
template <class W>
__global__ void __launch_bounds__(256) ln_bwd_fold(const LnBwdArgs a) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.D) return;
    float dw = 0.f, db = 0.f;
    for (int s = 0; s < a.slices; ++s) {
        dw += a.part[(2LL * s) * a.D + c];
        db += a.part[(2LL * s + 1) * a.D + c];
    }
    if (a.dw) static_cast<W*>(a.dw)[c] = from_f32<W>(dw);
    if (a.db) static_cast<W*>(a.db)[c] = from_f32<W>(db);
}

int ln_slices(int64_t rows) {
    const int64_t s = (rows + 31) / 32;
    return (int)(s < 1 ? 1 : s > 296 ? 296 : s);
}

bool ln_shape_ok(int64_t rows, int D, int64_t ld) { return rows >= 0 && D > 0 && (rows <= 1 || ld >= D); }

}  // namespace

extern "C" {

int hfuse_layernorm(const void* x, int64_t rows, int D, int64_t ld_x, int dtype, const void* weight, const void* bias,
                    int weight_dtype, float eps, void* y, float* mean, float* invstd, hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || (weight_dtype != dtype && weight_dtype != HFUSE_F32)) return HFUSE_ERR_BAD_ARG;
    if (!ln_shape_ok(rows, D, ld_x) || !(eps >= 0.f)) return HFUSE_ERR_BAD_ARG;
    if (rows == 0) return HFUSE_OK;
    if (!x || !y || !mean || !invstd) return HFUSE_ERR_BAD_ARG;
    const size_t es = lm_type_size(dtype), ws = lm_type_size(weight_dtype);
    if (!aligned_to(x, es) || !aligned_to(y, es) || !aligned_to(weight, ws) || !aligned_to(bias, ws) || !aligned_to(mean, 4) ||
        !aligned_to(invstd, 4))
        return HFUSE_ERR_ALIGNMENT;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    LnFwdArgs a{x, weight, bias, y, mean, invstd, rows, ld_x, D, 1.f / (float)D, eps};
    return by_types(dtype, weight_dtype, [&](auto t, auto w) {
        using T = typename decltype(t)::type;
        using W = typename decltype(w)::type;
        const int grid = (int)(rows < f.sms * 4LL ? rows : f.sms * 4LL);
        return launch_kernel(ln_fwd_wide<T, W>, grid, 512, 0, static_cast<cudaStream_t>(stream), false, a);
    });
}

size_t hfuse_layernorm_backward_workspace_bytes(int64_t rows, int D) {
    if (rows < 0 || D <= 0) return 0;
    return (size_t)ln_slices(rows) * 2 * (size_t)D * sizeof(float);
}

int hfuse_layernorm_backward(const void* x, int64_t ld_x, const void* grad_out, int64_t ld_grad_out, int64_t rows, int D,
                             int dtype, const float* mean, const float* invstd, const void* weight, int weight_dtype,
                             void* grad_in, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                             hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || (weight_dtype != dtype && weight_dtype != HFUSE_F32)) return HFUSE_ERR_BAD_ARG;
    if (!ln_shape_ok(rows, D, ld_x) || !ln_shape_ok(rows, D, ld_grad_out)) return HFUSE_ERR_BAD_ARG;
    if (rows > 0 && (!x || !grad_out || !mean || !invstd)) return HFUSE_ERR_BAD_ARG;
    const bool want_w = grad_weight || grad_bias;
    const size_t es = lm_type_size(dtype), ws = lm_type_size(weight_dtype);
    if (!aligned_to(x, es) || !aligned_to(grad_out, es) || !aligned_to(grad_in, es) || !aligned_to(weight, ws) ||
        !aligned_to(grad_weight, ws) || !aligned_to(grad_bias, ws) || !aligned_to(mean, 4) || !aligned_to(invstd, 4) ||
        !aligned_to(workspace, 16))
        return HFUSE_ERR_ALIGNMENT;
    if (want_w && (!workspace || workspace_bytes < hfuse_layernorm_backward_workspace_bytes(rows, D))) return HFUSE_ERR_WORKSPACE;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int slices = ln_slices(rows);
    LnBwdArgs a{x, grad_out, weight, mean, invstd, grad_in, grad_weight, grad_bias, static_cast<float*>(workspace),
                rows, ld_x, ld_grad_out, (rows + slices - 1) / slices, D, slices, 1.f / (float)D};
    return by_types(dtype, weight_dtype, [&](auto t, auto w) {
        using T = typename decltype(t)::type;
        using W = typename decltype(w)::type;
        if (grad_in && rows > 0) {
            const int grid = (int)(rows < f.sms * 4LL ? rows : f.sms * 4LL);
            if (int rc = launch_kernel(ln_bwd_rows<T, W>, grid, 512, 0, s, false, a)) return rc;
        }
        if (!want_w) return (int)HFUSE_OK;
        ln_bwd_cols<T><<<dim3((unsigned)((D + 31) / 32), (unsigned)slices), 256, 0, s>>>(a);
        if (int rc = check_launch()) return rc;
        return launch_kernel(ln_bwd_fold<W>, (D + 255) / 256, 256, 0, s, false, a);
    });
}

}  // extern "C"
