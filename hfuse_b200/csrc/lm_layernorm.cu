// Layer norm over the last dimension, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   forward   mu = sum x / D,  var = sum (x - mu)^2 / D,  r = 1 / sqrt(var + eps),  y = (x - mu) r w + b
//   backward  xh = (x - mu) r,  g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
#include <type_traits>

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
    int lanes;               // threads that share a row
    float inv_d, eps;
};

struct LnBwdArgs {
    const void *x, *dy, *w;
    const float *mean, *invstd;
    void *dx, *dw, *db;
    float* part;             // [slices][2][D]
    long long rows, ldx, lddy, slice_rows;
    int D, slices, lanes;
    float inv_d;
};

// A row lives in the registers of the threads that share it, NV accesses of EV elements each: it is read once, the mean
// and the sum of squares around it are formed there, and y is written.  MANY: 2^k <= 32 lanes share a row and a
// block has many, without any barrier; otherwise the whole block shares one, its warps' moments meet in shared memory behind one
// barrier.  Each thread keeps its columns from row to row, so their weights stay in registers too (KEEP), and
// the next row is loaded (AHEAD) before this one is reduced.
template <int NV, int EV, class T>
struct Row {
    Pack<T, EV> v[NV];
};
template <class T, int EV, int NV>
__device__ __forceinline__ void load_row(Row<NV, EV, T>& r, const T* p, int at, int lanes, int packs) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (at + k * lanes < packs) r.v[k] = load_stream<T, EV>(p + (at + k * lanes) * EV);
}
// f(pair index, value) over a pack; an odd element is a pair with a second value of zero
template <class T, int EV>
__device__ __forceinline__ float2 elements(const Pack<T, EV>& p, int k) {
    if constexpr (EV == 1) return make_float2(to_f32(p.v[0]), 0.f);
    else return pair_of(p, k);
}
template <int EV>
constexpr int kPairs = (EV + 1) / 2;

template <bool MANY>
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    if constexpr (MANY) {
        for (int o = lanes >> 1; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    } else {
        return warp_sum(v);
    }
}

template <class T, class W, int EV, int NV, bool MANY, int MAXT>
__global__ void __launch_bounds__(MAXT) ln_fwd(const LnFwdArgs a) {
    constexpr bool KEEP = NV * EV * (int)sizeof(W) <= 64 && MAXT <= 512, AHEAD = MAXT <= 512;
    __shared__ float2 moments[2][32];
    const T* x = static_cast<const T*>(a.x);
    const W* w = static_cast<const W*>(a.w);
    const W* b = static_cast<const W*>(a.b);
    const int lanes = MANY ? a.lanes : blockDim.x, packs = a.D / EV;
    const int at = MANY ? threadIdx.x & (lanes - 1) : threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = MANY ? blockDim.x / lanes : 1;
    const long long step = (long long)gridDim.x * per;
    long long r = (long long)blockIdx.x * per + (MANY ? threadIdx.x / lanes : 0);
    long long head = MANY ? (long long)blockIdx.x * per + warp * (32 / lanes) : r;      // the warp's first row
    // elements that warp number `lane` of the block holds
    float count = 0.f, inv_count = 0.f;
    if constexpr (!MANY) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) n += min(max(packs - k * lanes - 32 * lane, 0), min(32, max(lanes - 32 * lane, 0)));
        count = (float)(n * EV);
        inv_count = n ? 1.f / count : 0.f;
    }
    const float mine = MANY ? 0.f : __shfl_sync(0xffffffffu, inv_count, warp);
    Pack<W, EV> kw[NV], kb[NV];
    if constexpr (KEEP) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (at + k * lanes < packs) {
                if (w) load_weights<W, EV>(w + (at + k * lanes) * EV, kw[k]);
                if (b) load_weights<W, EV>(b + (at + k * lanes) * EV, kb[k]);
            }
    }
    Row<NV, EV, T> row, ahead;
    if (r < a.rows) load_row<T, EV, NV>(row, x + r * a.ldx, at, lanes, packs);
    for (int turn = 0; head < a.rows; head += step, r += step, turn ^= 1) {
        const bool in = !MANY || r < a.rows;
        if constexpr (AHEAD) {
            if (r + step < a.rows) load_row<T, EV, NV>(ahead, x + (r + step) * a.ldx, at, lanes, packs);
        } else if (r >= step && in) {
            load_row<T, EV, NV>(row, x + r * a.ldx, at, lanes, packs);
        }
        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (in && at + k * lanes < packs) {
#pragma unroll
                for (int q = 0; q < kPairs<EV>; ++q) s2 = add2(s2, elements<T, EV>(row.v[k], q));
            }
        float s = lanes_sum<MANY>(s2.x + s2.y, lanes);
        const float mid = MANY ? s * a.inv_d : s * mine;              // of the row, or of the warp's part of it
        float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (in && at + k * lanes < packs) {
#pragma unroll
                for (int q = 0; q < kPairs<EV>; ++q) {
                    float2 d = add2(elements<T, EV>(row.v[k], q), make_float2(-mid, -mid));
                    if (EV == 1) d.y = 0.f;
                    q2 = fma2(d, d, q2);
                }
            }
        float q = lanes_sum<MANY>(q2.x + q2.y, lanes), mu = mid;
        if constexpr (!MANY) {
            if (lane == 0) moments[turn][warp] = make_float2(s, q);
            __syncthreads();
            // lane l takes warp l's part: sums of squares around the parts' means, moved to the row's mean
            const float2 m = lane < (lanes >> 5) ? moments[turn][lane] : make_float2(0.f, 0.f);
            mu = warp_sum(m.x) * a.inv_d;
            const float d = m.x * inv_count - mu;
            q = warp_sum(fmaf(count * d, d, m.y));
        }
        const float is = 1.f / sqrtf(fmaf(q, a.inv_d, a.eps));
        if (in) {
            T* y = static_cast<T*>(a.y) + r * a.D;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int p = at + k * lanes;
                if (p >= packs) continue;
                if constexpr (!KEEP) {
                    if (w) load_weights<W, EV>(w + p * EV, kw[k]);
                    if (b) load_weights<W, EV>(b + p * EV, kb[k]);
                }
                float o[2 * kPairs<EV>];
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j) {
                    float2 d = mul2(add2(elements<T, EV>(row.v[k], j), make_float2(-mu, -mu)), make_float2(is, is));
                    if (w) d = mul2(d, elements<W, EV>(kw[k], j));
                    if (b) d = add2(d, elements<W, EV>(kb[k], j));
                    o[2 * j] = d.x;
                    o[2 * j + 1] = d.y;
                }
                if constexpr (EV == 1) store_stream<T, 1>(y + p, Pack<T, 1>{{from_f32<T>(o[0])}});
                else store_stream<T, EV>(y + p * EV, pack_f32<T, EV>(o));
            }
            if (at == 0) {
                a.mean[r] = mu;
                a.invstd[r] = is;
            }
        }
        if constexpr (AHEAD) row = ahead;
    }
}

// The same layout backwards: x and dy of a row are in registers, the two row sums are reduced together, and each
// thread adds up dy xh and dy of its columns over all rows of its block.  The blocks' sums go to the workspace, [block][2][D].
template <class T, class W, int EV, int NV, bool MANY, int MAXT>
__global__ void __launch_bounds__(MAXT) ln_bwd(const LnBwdArgs a) {
    constexpr bool AHEAD = MAXT <= 512;
    extern __shared__ float shared_sums[];                  // MANY: 2 EV NV floats of every thread
    __shared__ float2 sums[2][32];
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    const W* w = static_cast<const W*>(a.w);
    const int lanes = MANY ? a.lanes : blockDim.x, packs = a.D / EV;
    const int at = MANY ? threadIdx.x & (lanes - 1) : threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = MANY ? blockDim.x / lanes : 1;
    const long long step = (long long)gridDim.x * per;
    long long r = (long long)blockIdx.x * per + (MANY ? threadIdx.x / lanes : 0);
    long long head = MANY ? (long long)blockIdx.x * per + warp * (32 / lanes) : r;
    Pack<W, EV> kw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (w && at + k * lanes < packs) load_weights<W, EV>(w + (at + k * lanes) * EV, kw[k]);
    float2 dw[NV][kPairs<EV>], db[NV][kPairs<EV>];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < kPairs<EV>; ++j) dw[k][j] = db[k][j] = make_float2(0.f, 0.f);
    Row<NV, EV, T> rx, rd, nx, nd;
    float mu = 0.f, is = 0.f, nmu = 0.f, nis = 0.f;
    if (r < a.rows) {
        load_row<T, EV, NV>(rx, x + r * a.ldx, at, lanes, packs);
        load_row<T, EV, NV>(rd, dy + r * a.lddy, at, lanes, packs);
        mu = __ldg(a.mean + r);
        is = __ldg(a.invstd + r);
    }
    for (int turn = 0; head < a.rows; head += step, r += step, turn ^= 1) {
        const bool in = !MANY || r < a.rows;
        if (!AHEAD && r >= step && in) {
            load_row<T, EV, NV>(rx, x + r * a.ldx, at, lanes, packs);
            load_row<T, EV, NV>(rd, dy + r * a.lddy, at, lanes, packs);
            mu = __ldg(a.mean + r);
            is = __ldg(a.invstd + r);
        }
        if (AHEAD && r + step < a.rows) {
            load_row<T, EV, NV>(nx, x + (r + step) * a.ldx, at, lanes, packs);
            load_row<T, EV, NV>(nd, dy + (r + step) * a.lddy, at, lanes, packs);
            nmu = __ldg(a.mean + r + step);
            nis = __ldg(a.invstd + r + step);
        }
        const float2 mu2 = make_float2(-mu, -mu), is2 = make_float2(is, is);
        float2 s = make_float2(0.f, 0.f), d = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (in && at + k * lanes < packs) {
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j) {
                    const float2 xh = mul2(add2(elements<T, EV>(rx.v[k], j), mu2), is2), g0 = elements<T, EV>(rd.v[k], j);
                    const float2 g = w ? mul2(g0, elements<W, EV>(kw[k], j)) : g0;
                    dw[k][j] = fma2(g0, xh, dw[k][j]);
                    db[k][j] = add2(db[k][j], g0);
                    s = add2(s, g);
                    d = fma2(g, xh, d);
                }
            }
        float2 both = make_float2(lanes_sum<MANY>(s.x + s.y, lanes), lanes_sum<MANY>(d.x + d.y, lanes));
        if constexpr (!MANY) {
            if (lane == 0) sums[turn][warp] = both;
            __syncthreads();
            both = make_float2(0.f, 0.f);
            for (int k = 0; k < (lanes >> 5); ++k) both = add2(both, sums[turn][k]);
        }
        if (in && a.dx) {
            const float2 ms = make_float2(-both.x * a.inv_d, -both.x * a.inv_d), md = make_float2(-both.y * a.inv_d, -both.y * a.inv_d);
            T* dx = static_cast<T*>(a.dx) + r * a.D;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int p = at + k * lanes;
                if (p >= packs) continue;
                float o[2 * kPairs<EV>];
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j) {
                    const float2 xh = mul2(add2(elements<T, EV>(rx.v[k], j), mu2), is2), g0 = elements<T, EV>(rd.v[k], j);
                    const float2 g = w ? mul2(g0, elements<W, EV>(kw[k], j)) : g0;
                    const float2 v = mul2(is2, fma2(xh, md, add2(g, ms)));
                    o[2 * j] = v.x;
                    o[2 * j + 1] = v.y;
                }
                if constexpr (EV == 1) store_stream<T, 1>(dx + p, Pack<T, 1>{{from_f32<T>(o[0])}});
                else store_stream<T, EV>(dx + p * EV, pack_f32<T, EV>(o));
            }
        }
        if constexpr (AHEAD) {
            rx = nx;
            rd = nd;
            mu = nmu;
            is = nis;
        }
    }
    if (!a.part) return;
    float* part = a.part + 2LL * blockIdx.x * a.D;
    if constexpr (MANY) {
        // the block's groups of lanes, added in their order; [value][thread]
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < EV; ++j) {
                shared_sums[(2 * (k * EV + j)) * 256 + threadIdx.x] = j & 1 ? dw[k][j / 2].y : dw[k][j / 2].x;
                shared_sums[(2 * (k * EV + j) + 1) * 256 + threadIdx.x] = j & 1 ? db[k][j / 2].y : db[k][j / 2].x;
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * NV * EV * lanes; i += 256) {
            const int l = i & (lanes - 1), v = i / lanes, c = ((v >> 1) / EV * lanes + l) * EV + (v >> 1) % EV;
            if (c >= a.D) continue;
            float t = 0.f;
            for (int g = 0; g < per; ++g) t += shared_sums[v * 256 + g * lanes + l];
            part[(v & 1) * (long long)a.D + c] = t;
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (at + k * lanes < packs) {
#pragma unroll
                for (int j = 0; j < EV; ++j) {
                    const int c = (at + k * lanes) * EV + j;
                    part[c] = j & 1 ? dw[k][j / 2].y : dw[k][j / 2].x;
                    part[a.D + c] = j & 1 ? db[k][j / 2].y : db[k][j / 2].x;
                }
            }
    }
}

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

// The slices' (or blocks') sums: 32 columns and 8 runs of slices to a block, the runs added in their order.  Launched
// as the programmatic dependent of the kernel that makes the sums.
template <class W>
__global__ void __launch_bounds__(256) ln_bwd_fold(const LnBwdArgs a) {
    __shared__ float sh[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long long i = blockIdx.x * 32LL + tx;                   // of 2 D values
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float t = 0.f;
    if (i < 2LL * a.D) {
        const int per = (a.slices + 7) / 8, s0 = ty * per, s1 = min(a.slices, s0 + per);
#pragma unroll 8
        for (int s = s0; s < s1; ++s) t += a.part[2LL * s * a.D + i];
    }
    sh[ty][tx] = t;
    __syncthreads();
    if (ty == 0 && i < 2LL * a.D) {
        for (int k = 1; k < 8; ++k) t += sh[k][tx];
        W* out = static_cast<W*>(i < a.D ? a.dw : a.db);
        if (out) out[i < a.D ? i : i - a.D] = from_f32<W>(t);
    }
}

constexpr int kMaxParts = 592;        // blocks whose sums the workspace holds: 4 on each of 148 SMs

// rows of the column sums of rows too wide for registers
int ln_slices(int64_t rows) {
    const int64_t s = (rows + 31) / 32;
    return (int)(s < 1 ? 1 : s > 296 ? 296 : s);
}

using Yes = std::bool_constant<true>;
using No = std::bool_constant<false>;
template <int N>
using Num = std::integral_constant<int, N>;

// How a row of `packs` accesses is shared: by `lanes` threads with `nv` accesses each (nv = 0: too wide).  Up to 32
// threads: `many` rows to a block.  Above: blocks of about 256 threads while two accesses of each do, then up to 512, then
// (`big`) up to 1024 with half the registers.
struct LnShape {
    int nv, lanes;
    bool many, big;
};
LnShape ln_shape(long long packs, int max_nv_many, int max_nv) {
    LnShape s{};
    for (int nv = 1; nv <= max_nv_many; nv *= 2)
        if (packs <= 32LL * nv) {
            s.nv = nv;
            s.many = true;
            s.lanes = 32;
            while (s.lanes > 1 && (long long)(s.lanes / 2) * nv >= packs) s.lanes /= 2;
            return s;
        }
    for (int nv = 1; nv <= max_nv; nv *= 2)
        if (packs <= (nv == max_nv ? 1024LL : 256LL) * nv) {
            s.nv = nv;
            s.lanes = (int)((packs + 32LL * nv - 1) / (32LL * nv) * 32);
            s.big = s.lanes > 512;
            return s;
        }
    return s;
}

template <class T, class W, int EV, int NV, bool MANY, int MAXT>
int ln_fwd_launch(LnFwdArgs a, LnShape h, int sms, cudaStream_t s) {
    auto kern = ln_fwd<T, W, EV, NV, MANY, MAXT>;
    const int block = MANY ? 256 : h.lanes, per = MANY ? 256 / h.lanes : 1;
    const long long want = (a.rows + per - 1) / per, most = (long long)sms * resident_blocks((const void*)kern, block, 0);
    a.lanes = h.lanes;
    return launch_kernel(kern, (int)(want < most ? want : most), block, 0, s, false, a);
}
template <class T, class W, int EV, int NV, bool MANY, int MAXT>
int ln_bwd_launch(LnBwdArgs& a, LnShape h, int sms, cudaStream_t s) {
    auto kern = ln_bwd<T, W, EV, NV, MANY, MAXT>;
    const int block = MANY ? 256 : h.lanes, per = MANY ? 256 / h.lanes : 1;
    const size_t smem = MANY ? (size_t)2 * NV * EV * 256 * 4 : 0;
    const long long want = (a.rows + per - 1) / per;
    long long most = (long long)sms * resident_blocks((const void*)kern, block, smem);
    most = most < kMaxParts ? most : kMaxParts;
    a.lanes = h.lanes;
    a.slices = (int)(want < most ? want : most);
    return launch_kernel(kern, a.slices, block, smem, s, false, a);
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
    LnFwdArgs a{x, weight, bias, y, mean, invstd, rows, ld_x, D, 0, 1.f / (float)D, eps};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = aligned_to(x, 16) && aligned_to(y, 16) && aligned_to(weight, 16) && aligned_to(bias, 16) &&
                      D * es % 16 == 0 && ld_x * es % 16 == 0;
    return by_types(dtype, weight_dtype, [&](auto t, auto w) {
        using T = typename decltype(t)::type;
        using W = typename decltype(w)::type;
        constexpr int EV = 16 / sizeof(T);
        const LnShape h = ln_shape(wide ? D / EV : D, 4, 4);
        if (h.nv == 0) {
            const int grid = (int)(rows < f.sms * 4LL ? rows : f.sms * 4LL);
            return launch_kernel(ln_fwd_wide<T, W>, grid, 512, 0, s, false, a);
        }
        auto go = [&](auto many, auto nv, auto maxt) {
            constexpr bool MANY = decltype(many)::value;
            constexpr int NV = decltype(nv)::value, MAXT = decltype(maxt)::value;
            return wide ? ln_fwd_launch<T, W, EV, NV, MANY, MAXT>(a, h, f.sms, s) : ln_fwd_launch<T, W, 1, NV, MANY, MAXT>(a, h, f.sms, s);
        };
        if (h.many)
            return h.nv == 1 ? go(Yes{}, Num<1>{}, Num<256>{}) : h.nv == 2 ? go(Yes{}, Num<2>{}, Num<256>{}) : go(Yes{}, Num<4>{}, Num<256>{});
        if (h.big) return go(No{}, Num<4>{}, Num<1024>{});
        return h.nv == 1 ? go(No{}, Num<1>{}, Num<512>{}) : h.nv == 2 ? go(No{}, Num<2>{}, Num<512>{}) : go(No{}, Num<4>{}, Num<512>{});
    });
}

size_t hfuse_layernorm_backward_workspace_bytes(int64_t rows, int D) {
    if (rows < 0 || D <= 0) return 0;
    return (size_t)(rows < 1 ? 1 : rows < kMaxParts ? rows : kMaxParts) * 2 * (size_t)D * sizeof(float);
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
    LnBwdArgs a{x, grad_out, weight, mean, invstd, grad_in, grad_weight, grad_bias, want_w ? static_cast<float*>(workspace) : nullptr,
                rows, ld_x, ld_grad_out, (rows + slices - 1) / slices, D, slices, 0, 1.f / (float)D};
    const bool wide = aligned_to(x, 16) && aligned_to(grad_out, 16) && aligned_to(grad_in, 16) && aligned_to(weight, 16) &&
                      D * es % 16 == 0 && ld_x * es % 16 == 0 && ld_grad_out * es % 16 == 0;
    return by_types(dtype, weight_dtype, [&](auto t, auto w) {
        using T = typename decltype(t)::type;
        using W = typename decltype(w)::type;
        constexpr int EV = 16 / sizeof(T);
        const LnShape h = rows > 0 ? ln_shape(wide ? D / EV : D, 2, wide ? EV == 8 ? 2 : 4 : 8) : LnShape{};
        int rc;
        if (h.nv == 0) {
            if (grad_in && rows > 0) {
                const int grid = (int)(rows < f.sms * 4LL ? rows : f.sms * 4LL);
                if ((rc = launch_kernel(ln_bwd_rows<T, W>, grid, 512, 0, s, false, a))) return rc;
            }
            if (!want_w) return (int)HFUSE_OK;
            ln_bwd_cols<T><<<dim3((unsigned)((D + 31) / 32), (unsigned)slices), 256, 0, s>>>(a);
            rc = check_launch();
        } else {
            auto go = [&](auto many, auto nv, auto maxt) {
                constexpr bool MANY = decltype(many)::value;
                constexpr int NV = decltype(nv)::value, MAXT = decltype(maxt)::value;
                if (!wide) return ln_bwd_launch<T, W, 1, NV, MANY, MAXT>(a, h, f.sms, s);
                if constexpr (NV * EV <= 16) return ln_bwd_launch<T, W, EV, NV, MANY, MAXT>(a, h, f.sms, s);
                else return (int)HFUSE_ERR_BAD_ARG;                    // ln_shape gives no such shape
            };
            if (h.many) rc = h.nv == 1 ? go(Yes{}, Num<1>{}, Num<256>{}) : go(Yes{}, Num<2>{}, Num<256>{});
            else if (h.big)
                rc = h.nv == 2 ? go(No{}, Num<2>{}, Num<1024>{}) : h.nv == 4 ? go(No{}, Num<4>{}, Num<1024>{}) : go(No{}, Num<8>{}, Num<1024>{});
            else
                rc = h.nv == 1   ? go(No{}, Num<1>{}, Num<512>{})
                     : h.nv == 2 ? go(No{}, Num<2>{}, Num<512>{})
                     : h.nv == 4 ? go(No{}, Num<4>{}, Num<512>{})
                                 : go(No{}, Num<8>{}, Num<512>{});
        }
        if (rc || !want_w) return rc;
        return launch_kernel(ln_bwd_fold<W>, (int)((2LL * D + 31) / 32), 256, 0, s, true, a);
    });
}

}  // extern "C"
