// Gated linear recurrence along the steps of a sequence, forward and backward.
//
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  out_t = h_t      (per batch item and channel)
//   e_t = dout_t + a_{t+1} e_{t+1},  dx_t = (1 - a_t) e_t,  dgate_t = e_t (h_{t-1} - x_t) a_t (1 - a_t),  dh_0 = a_1 e_1
//
// A gate of -infinity starts afresh (h_t = x_t), one of +infinity holds the state.
#include "launch.cuh"
#include "lm_common.cuh"

using namespace hfuse;

namespace {

constexpr int kSaved = HFUSE_RECURRENCE_CHUNK;

struct RecArgs {
    const void *gate, *x, *dy;
    const float *h0, *dlast;
    void *y, *dgate, *dx;
    float *last, *states, *dh0;
    long long gate_b, gate_t, x_b, x_t, dy_b, dy_t;       // strides of a batch item and of a step
    int B, T, D, chunks;
};

// a = sigmoid(g) and 1 - a, the smaller of the two without cancellation; a NaN stays one
__device__ __forceinline__ void gates(float g, float& a, float& z) {
    const float e = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + e), s = e * r;
    a = g >= 0.f ? r : s;
    z = g >= 0.f ? s : r;
}

template <class T>
__global__ void __launch_bounds__(128) rec_fwd(const RecArgs p) {
    for (long long i = (long long)blockIdx.x * 128 + threadIdx.x; i < (long long)p.B * p.D; i += (long long)gridDim.x * 128) {
        const long long b = i / p.D, d = i - b * p.D;
        const T* g = static_cast<const T*>(p.gate) + b * p.gate_b + d;
        const T* x = static_cast<const T*>(p.x) + b * p.x_b + d;
        T* y = static_cast<T*>(p.y) + b * p.T * p.D + d;
        float h = p.h0 ? p.h0[i] : 0.f;
        for (int t = 0; t < p.T; ++t) {
            if (p.states && t % kSaved == 0) p.states[(b * p.chunks + t / kSaved) * p.D + d] = h;
            float a, z;
            gates(to_f32(g[t * p.gate_t]), a, z);
            h = fmaf(a, h, z * to_f32(x[t * p.x_t]));
            y[(long long)t * p.D] = from_f32<T>(h);
        }
        p.last[i] = h;
    }
}

template <class T>
__global__ void __launch_bounds__(128) rec_bwd(const RecArgs p) {
    for (long long i = (long long)blockIdx.x * 128 + threadIdx.x; i < (long long)p.B * p.D; i += (long long)gridDim.x * 128) {
        const long long b = i / p.D, d = i - b * p.D;
        const T* g = static_cast<const T*>(p.gate) + b * p.gate_b + d;
        const T* x = static_cast<const T*>(p.x) + b * p.x_b + d;
        const T* dy = static_cast<const T*>(p.dy) + b * p.dy_b + d;
        T* dg = static_cast<T*>(p.dgate) + b * p.T * p.D + d;
        T* dx = static_cast<T*>(p.dx) + b * p.T * p.D + d;
        float e = p.dlast ? p.dlast[i] : 0.f;
        float before[kSaved];                              // the state before each step of the chunk, run again
        for (int c = p.chunks - 1; c >= 0; --c) {
            const int t0 = c * kSaved, t1 = min(p.T, t0 + kSaved);
            float h = p.states[(b * p.chunks + c) * p.D + d], a, z;
            for (int t = t0; t < t1; ++t) {
                before[t - t0] = h;
                gates(to_f32(g[t * p.gate_t]), a, z);
                h = fmaf(a, h, z * to_f32(x[t * p.x_t]));
            }
            for (int t = t1 - 1; t >= t0; --t) {
                gates(to_f32(g[t * p.gate_t]), a, z);
                e += to_f32(dy[t * p.dy_t]);
                dx[(long long)t * p.D] = from_f32<T>(e * z);
                dg[(long long)t * p.D] = from_f32<T>(e * (before[t - t0] - to_f32(x[t * p.x_t])) * (a * z));
                e *= a;
            }
        }
        p.dh0[i] = e;
    }
}

bool rec_shape_ok(int64_t B, int64_t T, int D) { return B > 0 && T > 0 && D > 0; }
constexpr long long kMax32 = (1LL << 31) - 1;

}  // namespace

extern "C" {

int64_t hfuse_gated_recurrence_chunks(int64_t T) { return T > 0 ? (T + kSaved - 1) / kSaved : 0; }

int hfuse_gated_recurrence(const void* gate, int64_t gate_stride_b, int64_t gate_stride_t, const void* x, int64_t x_stride_b,
                           int64_t x_stride_t, int64_t B, int64_t T, int D, int dtype, const float* h0, void* out, float* h_last,
                           float* states, hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || !rec_shape_ok(B, T, D) || !gate || !x || !out || !h_last) return HFUSE_ERR_BAD_ARG;
    if (gate_stride_b < 0 || gate_stride_t < 0 || x_stride_b < 0 || x_stride_t < 0) return HFUSE_ERR_BAD_ARG;
    if (B > kMax32 || T > kMax32 - 65536 || B * D > kMax32) return HFUSE_ERR_TOO_LARGE;
    const size_t es = lm_type_size(dtype);
    if (!aligned_to(gate, es) || !aligned_to(x, es) || !aligned_to(out, es) || !aligned_to(h0, 4) || !aligned_to(h_last, 4) ||
        !aligned_to(states, 4))
        return HFUSE_ERR_ALIGNMENT;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    RecArgs a{};
    a.gate = gate; a.x = x; a.h0 = h0; a.y = out; a.last = h_last; a.states = states;
    a.gate_b = gate_stride_b; a.gate_t = gate_stride_t; a.x_b = x_stride_b; a.x_t = x_stride_t;
    a.B = (int)B; a.T = (int)T; a.D = D; a.chunks = (int)hfuse_gated_recurrence_chunks(T);
    return by_type(dtype, [&](auto t) {
        using E = typename decltype(t)::type;
        const long long want = (B * D + 127) / 128, most = f.sms * 16LL;
        return launch_kernel(rec_fwd<E>, (int)(want < most ? want : most), 128, 0, static_cast<cudaStream_t>(stream), false, a);
    });
}

int hfuse_gated_recurrence_backward(const void* gate, int64_t gate_stride_b, int64_t gate_stride_t, const void* x,
                                    int64_t x_stride_b, int64_t x_stride_t, const float* states, const void* grad_out,
                                    int64_t grad_out_stride_b, int64_t grad_out_stride_t, const float* grad_h_last, int64_t B,
                                    int64_t T, int D, int dtype, void* grad_gate, void* grad_x, float* grad_h0,
                                    hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || !rec_shape_ok(B, T, D) || !gate || !x || !states || !grad_out || !grad_gate || !grad_x || !grad_h0)
        return HFUSE_ERR_BAD_ARG;
    if (gate_stride_b < 0 || gate_stride_t < 0 || x_stride_b < 0 || x_stride_t < 0 || grad_out_stride_b < 0 || grad_out_stride_t < 0)
        return HFUSE_ERR_BAD_ARG;
    if (B > kMax32 || T > kMax32 - 65536 || B * D > kMax32) return HFUSE_ERR_TOO_LARGE;
    const size_t es = lm_type_size(dtype);
    if (!aligned_to(gate, es) || !aligned_to(x, es) || !aligned_to(grad_out, es) || !aligned_to(grad_gate, es) ||
        !aligned_to(grad_x, es) || !aligned_to(states, 4) || !aligned_to(grad_h_last, 4) || !aligned_to(grad_h0, 4))
        return HFUSE_ERR_ALIGNMENT;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    RecArgs a{};
    a.gate = gate; a.x = x; a.dy = grad_out; a.dlast = grad_h_last; a.states = const_cast<float*>(states);
    a.dgate = grad_gate; a.dx = grad_x; a.dh0 = grad_h0;
    a.gate_b = gate_stride_b; a.gate_t = gate_stride_t; a.x_b = x_stride_b; a.x_t = x_stride_t;
    a.dy_b = grad_out_stride_b; a.dy_t = grad_out_stride_t;
    a.B = (int)B; a.T = (int)T; a.D = D; a.chunks = (int)hfuse_gated_recurrence_chunks(T);
    return by_type(dtype, [&](auto t) {
        using E = typename decltype(t)::type;
        const long long want = (B * D + 127) / 128, most = f.sms * 16LL;
        return launch_kernel(rec_bwd<E>, (int)(want < most ? want : most), 128, 0, static_cast<cudaStream_t>(stream), false, a);
    });
}

}  // extern "C"
