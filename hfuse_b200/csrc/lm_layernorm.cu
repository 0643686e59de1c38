// Layer norm over the last dimension, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   forward   mu = sum x / D,  var = sum (x - mu)^2 / D,  r = 1 / sqrt(var + eps),  y = (x - mu) r w + b
//   backward  xh = (x - mu) r,  g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Memory-bound: a row is read once, its mean and the sum of squares around it are formed on chip, and the result is written.
// Three layouts, by the length of a row:
//   short rows   2^k <= 32 lanes share a row and a block has many; no barrier at all, the next row is on its way into
//                registers while one is reduced;
//   rows         one-dimensional bulk (TMA) copies bring whole rows into shared memory ahead of their use, so
//                that the bytes in flight cost neither registers nor threads; forward, one warp (or a few that share a named
//                barrier) takes a row; backward, a block takes a few rows at a time and each thread keeps its columns, for
//                which it adds up dw and db in registers over all of the block's rows;
//   long rows    a block per row that reads it again from L2 for each step.
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
    float inv_d, eps;
    int lanes;               // short rows: threads that share a row
    int team, stages;        // rows: warps that share a row, buffers of each team
    int buf, wbytes;         // bytes of a row buffer and of the weights in shared memory
    int period;              // rows: see Cut
};

struct LnBwdArgs {
    const void *x, *dy, *w;
    const float *mean, *invstd;
    void *dx, *dw, *db;
    float* part;             // [slices][2][D]
    long long rows, ldx, lddy, slice_rows;
    int D, slices;
    float inv_d;
    int lanes, stages, buf;
    int period;              // rows: see Cut
};

// ---- short rows: NV accesses of EV elements in the registers of each of the 2^k <= 32 lanes that share a row ---------
// Each thread keeps its columns from row to row, so their weights stay in registers too.
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
template <int EV>
constexpr int kPairs = (EV + 1) / 2;

// sum over the first n lanes, the others being zero; the same in all lanes up to the next power of two
__device__ __forceinline__ float few_sum(float v, int n) {
    if (n > 16) v += __shfl_xor_sync(0xffffffffu, v, 16);
    if (n > 8) v += __shfl_xor_sync(0xffffffffu, v, 8);
    if (n > 4) v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 2);
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return __shfl_sync(0xffffffffu, v, 0);
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = lanes >> 1; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// 1 / sqrt(var + eps): rsqrt is off by 2 units in the last place at most
__device__ __forceinline__ float inv_std(float q, float inv_d, float eps) {
    return rsqrtf(fmaf(q, inv_d, eps));
}

template <class W, int EV>
__device__ __forceinline__ void weights_of(const W* from, int p, float2 (&to)[kPairs<EV>], float none) {
    Pack<W, EV> q = {};
    if (from) q = load_cached<W, EV>(from + p * EV);
#pragma unroll
    for (int j = 0; j < kPairs<EV>; ++j) to[j] = from ? pair_of<W, EV>(q, j) : make_float2(none, none);
}

template <class T, class W, int EV, int NV>
__global__ void __launch_bounds__(256, NV * EV == 16 ? 3 : 1) ln_fwd_short(const LnFwdArgs a) {
    const T* x = static_cast<const T*>(a.x);
    const int lanes = a.lanes, packs = a.D / EV, per = 256 / lanes, at = threadIdx.x & (lanes - 1);
    const long long step = (long long)gridDim.x * per;
    long long r = (long long)blockIdx.x * per + threadIdx.x / lanes;
    long long head = (long long)blockIdx.x * per + (threadIdx.x >> 5) * (32 / lanes);      // the warp's first row
    float2 kw[NV][kPairs<EV>], kb[NV][kPairs<EV>];
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (at + k * lanes < packs) {
            weights_of<W, EV>(static_cast<const W*>(a.w), at + k * lanes, kw[k], 1.f);
            weights_of<W, EV>(static_cast<const W*>(a.b), at + k * lanes, kb[k], 0.f);
        }
    Row<NV, EV, T> row, ahead;
    if (r < a.rows) load_row<T, EV, NV>(row, x + r * a.ldx, at, lanes, packs);
    for (; head < a.rows; head += step, r += step) {
        const bool in = r < a.rows;
        if (r + step < a.rows) load_row<T, EV, NV>(ahead, x + (r + step) * a.ldx, at, lanes, packs);
        float2 f[NV][kPairs<EV>], s2 = make_float2(0.f, 0.f), q2 = s2;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (in && at + k * lanes < packs) {
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j) {
                    f[k][j] = pair_of<T, EV>(row.v[k], j);
                    s2 = add2(s2, f[k][j]);
                }
            }
        const float mu = lanes_sum(s2.x + s2.y, lanes) * a.inv_d;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (in && at + k * lanes < packs) {
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j) {
                    f[k][j] = add2(f[k][j], make_float2(-mu, -mu));
                    if (EV == 1) f[k][j].y = 0.f;
                    q2 = fma2(f[k][j], f[k][j], q2);
                }
            }
        const float is = inv_std(lanes_sum(q2.x + q2.y, lanes), a.inv_d, a.eps);
        if (in) {
            T* y = static_cast<T*>(a.y) + r * a.D;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (at + k * lanes >= packs) continue;
                float2 o[kPairs<EV>];
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j) o[j] = fma2(f[k][j], mul2(kw[k][j], make_float2(is, is)), kb[k][j]);
                store_stream<T, EV>(y + (at + k * lanes) * EV, pack_pairs<T, EV>(o));
            }
            if (at == 0) {
                a.mean[r] = mu;
                a.invstd[r] = is;
            }
        }
        row = ahead;
    }
}

// The same layout backwards: x and dy of a row are in registers, the two row sums are reduced together, and each
// thread adds up dy xh and dy of its columns over all its rows.  The blocks' sums go to the workspace, [block][2][D].
template <class T, class W, int EV, int NV>
__global__ void __launch_bounds__(256, NV * EV == 16 ? 2 : 1) ln_bwd_short(const LnBwdArgs a) {
    extern __shared__ float shared_sums[];                  // 2 EV NV floats of every thread, [value][thread]
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    const int lanes = a.lanes, packs = a.D / EV, per = 256 / lanes, at = threadIdx.x & (lanes - 1);
    const long long step = (long long)gridDim.x * per;
    long long r = (long long)blockIdx.x * per + threadIdx.x / lanes;
    long long head = (long long)blockIdx.x * per + (threadIdx.x >> 5) * (32 / lanes);
    float2 kw[NV][kPairs<EV>], dw[NV][kPairs<EV>], db[NV][kPairs<EV>];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (at + k * lanes < packs) weights_of<W, EV>(static_cast<const W*>(a.w), at + k * lanes, kw[k], 1.f);
#pragma unroll
        for (int j = 0; j < kPairs<EV>; ++j) dw[k][j] = db[k][j] = make_float2(0.f, 0.f);
    }
    Row<NV, EV, T> rx, rd, nx, nd;
    float mu = 0.f, is = 0.f, nmu = 0.f, nis = 0.f;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the sums' last step waits for this grid's end
    if (r < a.rows) {
        load_row<T, EV, NV>(rx, x + r * a.ldx, at, lanes, packs);
        load_row<T, EV, NV>(rd, dy + r * a.lddy, at, lanes, packs);
        mu = __ldg(a.mean + r);
        is = __ldg(a.invstd + r);
    }
    for (; head < a.rows; head += step, r += step) {
        const bool in = r < a.rows;
        if (r + step < a.rows) {
            load_row<T, EV, NV>(nx, x + (r + step) * a.ldx, at, lanes, packs);
            load_row<T, EV, NV>(nd, dy + (r + step) * a.lddy, at, lanes, packs);
            nmu = __ldg(a.mean + r + step);
            nis = __ldg(a.invstd + r + step);
        }
        const float2 mu2 = make_float2(-mu, -mu), is2 = make_float2(is, is);
        float2 s = make_float2(0.f, 0.f), d = s, xh[NV][kPairs<EV>], g[NV][kPairs<EV>];
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (in && at + k * lanes < packs) {
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j) {
                    const float2 g0 = pair_of<T, EV>(rd.v[k], j);
                    xh[k][j] = mul2(add2(pair_of<T, EV>(rx.v[k], j), mu2), is2);
                    g[k][j] = mul2(g0, kw[k][j]);
                    dw[k][j] = fma2(g0, xh[k][j], dw[k][j]);
                    db[k][j] = add2(db[k][j], g0);
                    s = add2(s, g[k][j]);
                    d = fma2(g[k][j], xh[k][j], d);
                }
            }
        const float ms = -lanes_sum(s.x + s.y, lanes) * a.inv_d, md = -lanes_sum(d.x + d.y, lanes) * a.inv_d;
        if (in && a.dx) {
            T* dx = static_cast<T*>(a.dx) + r * a.D;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (at + k * lanes >= packs) continue;
                float2 o[kPairs<EV>];
#pragma unroll
                for (int j = 0; j < kPairs<EV>; ++j)
                    o[j] = mul2(is2, fma2(xh[k][j], make_float2(md, md), add2(g[k][j], make_float2(ms, ms))));
                store_stream<T, EV>(dx + (at + k * lanes) * EV, pack_pairs<T, EV>(o));
            }
        }
        rx = nx;
        rd = nd;
        mu = nmu;
        is = nis;
    }
    if (!a.part) return;
    float* part = a.part + 2LL * blockIdx.x * a.D;
    // the block's groups of lanes, added in their order
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
}

// ---- rows in shared memory ---------------------------------------------------------------------------------
// A bulk copy begins on a 16-byte boundary and has a multiple of 16 bytes, so a row that does not is copied with what
// shares its first and last 16 bytes, as far as that belongs to the tensor; the first and the last row may lack some
// elements at the tensor's very ends, which are fetched one by one (patch).  Element 0 is `shift` bytes into the buffer.
struct Span {
    const unsigned char *lo, *hi;      // what is copied
    int shift;
};
template <class T>
__device__ __forceinline__ Span row_span(const T* base, long long ld, long long rows, int D, long long r) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(base), end = reinterpret_cast<uintptr_t>(base + (rows - 1) * ld + D);
    const uintptr_t p = reinterpret_cast<uintptr_t>(base + r * ld), q = p + (size_t)D * sizeof(T);
    Span s;
    s.shift = (int)(p & 15);
    uintptr_t lo = p & ~(uintptr_t)15, hi = (q + 15) & ~(uintptr_t)15;
    if (lo < begin) lo += 16;
    if (hi > end) hi -= 16;
    s.lo = reinterpret_cast<const unsigned char*>(lo);
    s.hi = reinterpret_cast<const unsigned char*>(hi);
    return s;
}
// announces and starts the copy of a row (one thread)
template <class T>
__device__ __forceinline__ void fetch_row(unsigned char* buf, unsigned long long* bar, const T* base, long long ld, long long rows, int D,
                                          long long r) {
    const Span s = row_span(base, ld, rows, D, r);
    const long long bytes = s.hi - s.lo;
    if (bytes > 0) {
        mbar_expect_tx(bar, (uint32_t)bytes);
        const uintptr_t row = reinterpret_cast<uintptr_t>(base + r * ld) & ~(uintptr_t)15;
        bulk_load(buf + (reinterpret_cast<uintptr_t>(s.lo) - row), s.lo, (uint32_t)bytes, bar);
    } else {
        mbar_arrive(bar);
    }
}
// whether patch_row has something to do; every thread of the team, then a barrier of the team
template <class T>
__device__ __forceinline__ bool row_lacks(const T* base, long long ld, long long rows, int D, long long r) {
    if (r != 0 && r != rows - 1) return false;
    const Span s = row_span(base, ld, rows, D, r);
    const uintptr_t p = reinterpret_cast<uintptr_t>(base + r * ld);
    return reinterpret_cast<uintptr_t>(s.lo) > p || reinterpret_cast<uintptr_t>(s.hi) < p + (size_t)D * sizeof(T);
}
template <class T>
__device__ __forceinline__ void patch_row(unsigned char* buf, const T* base, long long ld, long long rows, int D, long long r, int at,
                                          int lanes) {
    const Span s = row_span(base, ld, rows, D, r);
    const T* p = base + r * ld;
    T* to = reinterpret_cast<T*>(buf + s.shift);
    for (int i = at; i < D; i += lanes) {
        const unsigned char* q = reinterpret_cast<const unsigned char*>(p + i);
        if (q < s.lo || q >= s.hi) to[i] = p[i];
    }
    fence_proxy_async_shared();        // a later copy may write there
}
// the 16-byte boundary's distance from row r, in bytes; the low bits of a product need no wide multiplication
template <class T>
__device__ __forceinline__ int shift_of(const T* base, long long ld, long long r) {
    return (int)(((unsigned)reinterpret_cast<uintptr_t>(base) + (unsigned)r * ((unsigned)ld * (unsigned)sizeof(T))) & 15u);
}
// Rows of a width that is no multiple of 16 bytes.  Where all tensors' rows begin equally far behind a 16-byte boundary, that
// distance comes back after `period` rows (8 for an odd number of 16-bit elements), so a team that takes every period-th row
// has one distance, and its threads the same columns in each of its rows: `packs` whole 16-byte accesses from element
// `lead` on, and up to 14 elements before and behind them, one to a lane of the team's first warp.  16384 rows of 2047 16-bit
// elements take 35 us forward and 57 backward (of 2048: 25 and 47); as single elements they took 58 and 76.
struct Cut {
    int lead, packs, edges;       // edges: elements before and behind
    int column;                   // this thread's one, or -1
};
template <bool PHASED, int EV, class T>
__device__ __forceinline__ Cut cut_rows(const T* x, long long ld, int D, int first, int at) {
    if constexpr (!PHASED) return {0, D / EV, 0, -1};
    const int lead = (EV - shift_of(x, ld, first) / (int)sizeof(T)) & (EV - 1), packs = (D - lead) / EV, edges = D - packs * EV;
    return {lead, packs, edges, at < lead ? at : at < edges ? at + packs * EV : -1};
}
template <class W>
__device__ __forceinline__ float weight_of(const void* w, int c, float none) {
    return w ? to_f32(static_cast<const W*>(w)[c]) : none;
}
constexpr unsigned long long kRowWaitNs = 2000000000ull;

// the warps of a team meet at their own named barrier
__device__ __forceinline__ void team_sync(int team, int warps) {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(warps * 32) : "memory");
}

// A row's elements in the registers of a team: accesses of EV elements, or (EV = 1) single elements in pairs of
// accesses.  VALUES pairs.
template <class T, int EV, int NV>
struct Team {
    static constexpr int VALUES = NV * EV / 2;
    Pack<T, EV> v[NV];
    __device__ __forceinline__ void read(uint32_t row, const int (&place)[NV]) {
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = load_shared<T, EV>(row + place[k]);
    }
    // places behind `last` read that one; the minimum is kept from being taken ahead, which would cost a register each
    __device__ __forceinline__ void read_until(uint32_t row, const int (&place)[NV], int last) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            int p;
            asm volatile("min.s32 %0, %1, %2;" : "=r"(p) : "r"(place[k]), "r"(last));
            v[k] = load_shared<T, EV>(row + p);
        }
    }
    __device__ __forceinline__ float2 get(int i) const {
        if constexpr (EV == 1) return make_float2(pair_of<T, 1>(v[2 * i], 0).x, pair_of<T, 1>(v[2 * i + 1], 0).x);
        else return pair_of<T, EV>(v[i / (EV / 2)], i % (EV / 2));
    }
};
// where in a row's buffer a thread's accesses are; a place beyond the row is the row's last access again: who adds up has to
// leave it out
template <class T, int EV, int NV>
__device__ __forceinline__ void places(int (&place)[NV], int at, int lanes, int packs) {
#pragma unroll
    for (int k = 0; k < NV; ++k) place[k] = min(at + k * lanes, packs - 1) * EV * (int)sizeof(T);
}
// which of a pair's elements exist
template <int EV>
__device__ __forceinline__ void exists(int i, int at, int lanes, int packs, bool& x, bool& y) {
    if constexpr (EV == 1) {
        x = at + 2 * i * lanes < packs;
        y = at + (2 * i + 1) * lanes < packs;
    } else {
        x = y = at + i / (EV / 2) * lanes < packs;
    }
}

// The weights are in shared memory as floats, the halves of eight-element accesses in planes of their own, so that
// neighbouring lanes read neighbouring 16 bytes.
template <int EV>
__device__ __forceinline__ int weight_at(int c, int packs) {
    if constexpr (EV == 8) return ((c & 4) ? packs * 4 : 0) + (c >> 3) * 4 + (c & 3);
    else return c;
}
template <int EV>
__device__ __forceinline__ void weight_pairs(const float* w, int p, int packs, float2 (&to)[kPairs<EV>]) {
    if constexpr (EV == 1) {
        to[0] = make_float2(w[p], 0.f);
    } else {
#pragma unroll
        for (int h = 0; h < EV / 4; ++h) {
            const float4 v = *reinterpret_cast<const float4*>(w + h * packs * 4 + p * 4);
            to[2 * h] = make_float2(v.x, v.y);
            to[2 * h + 1] = make_float2(v.z, v.w);
        }
    }
}

// Bound by memory: 16384 rows of 4096 bf16 in 50 us, 5.4 TB/s (with rows loaded to registers: 60).
template <class T, class W, int EV, int NV, bool PHASED>
__global__ void __launch_bounds__(512) ln_fwd_rows(const LnFwdArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int VALUES = NV * EV / 2;
    const T* x = static_cast<const T*>(a.x);
    const int M = a.team, lane = threadIdx.x & 31, warp = warp_index(), warps = blockDim.x >> 5, teams = warps / M;
    const int team = warp / M, part = warp - team * M, lanes = 32 * M, at = part * 32 + lane;
    const int period = PHASED ? a.period : 1, first = blockIdx.x & (period - 1);                // of the block's rows
    const Cut cut = cut_rows<PHASED, EV>(x, a.ldx, a.D, first, at);
    const int packs = cut.packs;
    float* sw = reinterpret_cast<float*>(smem);
    float* sb = reinterpret_cast<float*>(smem + a.wbytes);
    unsigned char* ring = smem + 2 * a.wbytes + (size_t)team * a.stages * a.buf;
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + 2 * a.wbytes + (size_t)teams * a.stages * a.buf) + team * a.stages;
    float2* moments = reinterpret_cast<float2*>(smem + 2 * a.wbytes + (size_t)teams * a.stages * (a.buf + 8));    // [2][warps]
    const long long step = (long long)period * teams * (((int)gridDim.x - first + period - 1) / period);
    long long r = first + (long long)period * (blockIdx.x / period * teams + team);
    const bool lead = part == 0 && lane == 0;
    auto fetch = [&](long long row, int s) {
        if constexpr (PHASED) {
            mbar_expect_tx(bars + s, (uint32_t)packs * 16);
            bulk_load(ring + (size_t)s * a.buf, x + row * a.ldx + cut.lead, (uint32_t)packs * 16, bars + s);
        } else {
            fetch_row(ring + (size_t)s * a.buf, bars + s, x, a.ldx, a.rows, a.D, row);
        }
    };
    if (lead) {
        for (int s = 0; s < a.stages; ++s) mbar_init(bars + s, 1);
        fence_mbar_init();
        for (int s = 0; s < a.stages; ++s)
            if (r + s * step < a.rows) fetch(r + s * step, s);
    }
    // the thread's single element, a row ahead
    const T* edge_at = x + r * a.ldx + max(cut.column, 0);
    float edge_w = 0.f, edge_b = 0.f, edge = 0.f, edge_next = 0.f;
    if (PHASED && cut.column >= 0) {
        edge_w = weight_of<W>(a.w, cut.column, 1.f);
        edge_b = weight_of<W>(a.b, cut.column, 0.f);
        if (r < a.rows) edge_next = to_f32(*edge_at);
    }
    for (int i = threadIdx.x; PHASED && i < packs * EV; i += blockDim.x) {
        sw[weight_at<EV>(i, packs)] = weight_of<W>(a.w, cut.lead + i, 1.f);
        sb[weight_at<EV>(i, packs)] = weight_of<W>(a.b, cut.lead + i, 0.f);
    }
    for (int p = threadIdx.x; !PHASED && p < packs; p += blockDim.x) {
        float2 w[kPairs<EV>], b[kPairs<EV>];
        weights_of<W, EV>(static_cast<const W*>(a.w), p, w, 1.f);
        weights_of<W, EV>(static_cast<const W*>(a.b), p, b, 0.f);
#pragma unroll
        for (int j = 0; j < EV; ++j) {
            sw[weight_at<EV>(p * EV + j, packs)] = j & 1 ? w[j / 2].y : w[j / 2].x;
            sb[weight_at<EV>(p * EV + j, packs)] = j & 1 ? b[j / 2].y : b[j / 2].x;
        }
    }
    // elements that the team's warp number `lane` holds
    float count = 0.f, inv_count = 0.f;
    if (M > 1 && lane < M) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) n += min(max(packs - k * lanes - 32 * lane, 0), 32);
        count = (float)(n * EV + (lane == 0 ? cut.edges : 0));
        inv_count = n ? 1.f / count : 0.f;
    }
    const float mine = M > 1 ? __shfl_sync(0xffffffffu, inv_count, part) : a.inv_d;
    const bool whole = packs == NV * lanes;                // no place beyond the row
    int place[NV];
    places<T, EV, NV>(place, at, lanes, packs);
    __syncthreads();
    int stage = 0, parity = 0;
    for (int turn = 0; r < a.rows; r += step, turn ^= 1) {
        unsigned char* buf = ring + (size_t)stage * a.buf;
        const bool there = mbar_wait(bars + stage, parity, kRowWaitNs);
        int shift = 0;
        if constexpr (EV == 1) {
            shift = shift_of(x, a.ldx, r);
            if (row_lacks(x, a.ldx, a.rows, a.D, r)) {
                patch_row(buf, x, a.ldx, a.rows, a.D, r, at, lanes);
                team_sync(team, M);
            }
        }
        float2 f[VALUES], s2 = make_float2(0.f, 0.f), q2 = s2;
        if constexpr (PHASED) {
            edge = edge_next;
            s2.x = edge;
            edge_at += step * a.ldx;
            if (cut.column >= 0 && r + step < a.rows) edge_next = to_f32(*edge_at);
        }
        {
            Team<T, EV, NV> row;
            row.read(smem_u32(buf) + shift, place);
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                f[i] = row.get(i);
                if (whole) {
                    s2 = add2(s2, f[i]);
                } else {
                    bool ex, ey;
                    exists<EV>(i, at, lanes, packs, ex, ey);
                    s2 = add2(s2, make_float2(ex ? f[i].x : 0.f, ey ? f[i].y : 0.f));
                }
            }
        }
        const float s = warp_sum(s2.x + s2.y), mid = s * mine;                   // the mean of the warp's part
        if constexpr (PHASED) {
            edge = cut.column >= 0 ? edge - mid : 0.f;
            q2.x = edge * edge;
        }
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            f[i] = add2(f[i], make_float2(-mid, -mid));
            if (whole) {
                q2 = fma2(f[i], f[i], q2);
            } else {
                bool ex, ey;
                exists<EV>(i, at, lanes, packs, ex, ey);
                const float2 d = make_float2(ex ? f[i].x : 0.f, ey ? f[i].y : 0.f);
                q2 = fma2(d, d, q2);
            }
        }
        float q = warp_sum(q2.x + q2.y), mu = mid;
        if (M == 1) {
            __syncwarp();
        } else {
            float2* mine2 = moments + turn * warps + team * M;
            if (lane == 0) mine2[part] = make_float2(s, q);
            team_sync(team, M);
            // lane l takes warp l's part: sums of squares around the parts' means, moved to the row's mean
            const float2 m = lane < M ? mine2[lane] : make_float2(0.f, 0.f);
            mu = few_sum(m.x, M) * a.inv_d;
            const float d = m.x * inv_count - mu;
            q = few_sum(fmaf(count * d, d, m.y), M);
        }
        // the whole team has read the buffer
        if (lead && r + a.stages * step < a.rows) fetch(r + a.stages * step, stage);
        if (++stage == a.stages) {
            stage = 0;
            parity ^= 1;
        }
        float is = inv_std(q, a.inv_d, a.eps);
        if (!there) mu = is = __int_as_float(0x7fc00000);
        // f is relative to the mean of the warp's part: y = (f + (mid - mu)) is w + b
        const float2 is2 = make_float2(is, is), move = make_float2((mid - mu) * is, (mid - mu) * is);
        T* y = static_cast<T*>(a.y) + r * a.D + cut.lead;
        if (PHASED && cut.column >= 0) y[cut.column - cut.lead] = from_f32<T>(fmaf(fmaf(edge, is, move.x), edge_w, edge_b));
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int p = at + k * lanes;
            if (p >= packs) continue;
            float2 w[kPairs<EV>], b[kPairs<EV>], o[kPairs<EV>];
            weight_pairs<EV>(sw, p, packs, w);
            weight_pairs<EV>(sb, p, packs, b);
#pragma unroll
            for (int j = 0; j < kPairs<EV>; ++j) {
                float2 v;
                if constexpr (EV == 1) v = make_float2(k & 1 ? f[k / 2].y : f[k / 2].x, 0.f);
                else v = f[k * (EV / 2) + j];
                o[j] = fma2(fma2(v, is2, move), w[j], b[j]);
            }
            store_stream<T, EV>(y + p * EV, pack_pairs<T, EV>(o));
        }
        if (lead) {
            a.mean[r] = mu;
            a.invstd[r] = is;
        }
    }
}

// The sums over a warp of 4 values of each lane, in 6 shuffles instead of 20: halves of the lanes take over halves of the
// values.  Lane l gets value l / 8's sum (the same in its 8 lanes).
__device__ __forceinline__ float warp_sum4(float a, float b, float c, float d, int lane) {
    const bool up = lane & 16;
    const float u = (up ? c : a) + __shfl_xor_sync(0xffffffffu, up ? a : c, 16);
    const float v = (up ? d : b) + __shfl_xor_sync(0xffffffffu, up ? b : d, 16);
    const bool odd = lane & 8;
    float t = (odd ? v : u) + __shfl_xor_sync(0xffffffffu, odd ? u : v, 8);
    t += __shfl_xor_sync(0xffffffffu, t, 4);
    t += __shfl_xor_sync(0xffffffffu, t, 2);
    t += __shfl_xor_sync(0xffffffffu, t, 1);
    return t;
}

// Teams of warps take two rows at a time, [team][stage][x, dy][row] buffers; the block's teams add up their dw and db in
// the same memory at the end.  x and dy are read from shared memory twice, which leaves registers for the columns' sums.  8192
// rows of 2048 floats take 33 us (under ncu), 6.2 TB/s, bound by memory; 16-bit rows (16384 of 2048: 47 us with the join below, of
// 1000 elements 32) by the latency of 16 warps with two barriers for a pair of rows.
template <class T, class W, int EV, int NV, bool PHASED>
__global__ void __launch_bounds__(512) ln_bwd_rows(const LnBwdArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int VALUES = NV * EV / 2;
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    const W* w = static_cast<const W*>(a.w);
    const int lanes = a.lanes, warps = lanes >> 5, lane = threadIdx.x & 31, team = warp_index() / warps, warp = warp_index() - team * warps;
    const int teams = blockDim.x / lanes, at = warp * 32 + lane;
    const int period = PHASED ? a.period : 1, number = blockIdx.x * teams + team, first = number & (period - 1);
    const Cut cut = cut_rows<PHASED, EV>(x, a.ldx, a.D, first, at);
    const int packs = cut.packs;
    unsigned char* ring = smem + (size_t)team * a.stages * 4 * a.buf;
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(smem + (size_t)teams * a.stages * 4 * a.buf) + team * 2;
    float* sums = reinterpret_cast<float*>(smem + (size_t)teams * (a.stages * 4 * (size_t)a.buf + 16)) + team * 8 * warps;   // [2][warps][4]
    float2 kw[VALUES], dw[VALUES], db[VALUES];
    {
        Team<W, EV, NV> t;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            t.v[k] = {};
            if (!PHASED && w && at + k * lanes < packs) t.v[k] = load_cached<W, EV>(w + (at + k * lanes) * EV);
        }
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            bool ex, ey;
            exists<EV>(i, at, lanes, packs, ex, ey);
            kw[i] = w ? t.get(i) : make_float2(ex ? 1.f : 0.f, ey ? 1.f : 0.f);
            if (PHASED && w && ex) {
                const int c = cut.lead + (at + i / (EV / 2) * lanes) * EV + 2 * (i % (EV / 2));
                kw[i] = make_float2(to_f32(w[c]), to_f32(w[c + 1]));
            }
            dw[i] = db[i] = make_float2(0.f, 0.f);
        }
    }
    // Places beyond the row read x's last access again and zeros as dy, which keep out of the row sums whatever the row
    // holds (as x, a zero could be infinitely many deviations from the mean); nothing is stored for them.
    const int none = EV > 1 ? packs * EV * (int)sizeof(T) : a.buf - 32;
    const int last = (packs - 1) * EV * (int)sizeof(T);
    int place[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
        place[k] = EV > 1 ? min(at + k * lanes, packs) * EV * (int)sizeof(T) : at + k * lanes < packs ? (at + k * lanes) * (int)sizeof(T) : none;
    // the thread's single elements of the next two rows
    float edge_w = 0.f, edge_dw = 0.f, edge_db = 0.f, ex[2] = {0.f, 0.f}, ed[2] = {0.f, 0.f};
    if (PHASED && cut.column >= 0) edge_w = weight_of<W>(w, cut.column, 1.f);
    auto edges = [&](long long r) {
        if (PHASED && cut.column >= 0) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const long long row = r + g * period;
                if (row >= a.rows) continue;
                ex[g] = to_f32(x[row * a.ldx + cut.column]);
                ed[g] = to_f32(dy[row * a.lddy + cut.column]);
            }
        }
    };
    // a pair of rows, r and r + period; lanes 0 to 3 of the team's first warp fetch one row each
    const long long step = 2LL * period * (((int)gridDim.x * teams - first + period - 1) / period);
    auto fetch = [&](long long r, int s) {
        if (warp == 0 && lane < 4) {
            const long long row = r + (lane & 1) * period;
            unsigned char* buf = ring + (size_t)(4 * s + lane) * a.buf;
            if (row >= a.rows) {
                mbar_arrive(bars + s);
            } else if constexpr (PHASED) {
                mbar_expect_tx(bars + s, (uint32_t)packs * 16);
                bulk_load(buf, (lane < 2 ? x + row * a.ldx : dy + row * a.lddy) + cut.lead, (uint32_t)packs * 16, bars + s);
            }
            else if (lane < 2) fetch_row(buf, bars + s, x, a.ldx, a.rows, a.D, row);
            else fetch_row(buf, bars + s, dy, a.lddy, a.rows, a.D, row);
        }
    };
    // mean and invstd of a pair of rows in lanes 0 to 3
    auto stats = [&](long long r) {
        const long long row = r + (lane & 1) * period;
        return lane < 4 && row < a.rows ? __ldg((lane < 2 ? a.mean : a.invstd) + row) : 0.f;
    };
    if (at == 0) {
        mbar_init(bars, 4);
        mbar_init(bars + 1, 4);
        fence_mbar_init();
    }
    team_sync(team, warps);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the sums' last step waits for this grid's end
    long long r = first + 2LL * period * (number / period);
    for (int s = 0; s < a.stages; ++s)
        if (r + s * step < a.rows) fetch(r + s * step, s);
    if (at + (NV - 1) * lanes >= packs)                    // who reads the zeros writes them
        for (int b = 0; b < 4 * a.stages; ++b)
#pragma unroll
            for (int h = 0; h < (EV == 1 ? 2 : 1); ++h)
                reinterpret_cast<float4*>(ring + (size_t)b * a.buf + none)[h] = make_float4(0.f, 0.f, 0.f, 0.f);
    float now = stats(r), next = 0.f;
    edges(r);
    int stage = 0, parity = 0;
    for (int turn = 0; r < a.rows; r += step, turn ^= 1) {
        next = stats(r + step);
        unsigned char* buf = ring + (size_t)4 * stage * a.buf;
        const bool there = mbar_wait(bars + stage, parity, kRowWaitNs);
        const uint32_t at_buf = smem_u32(buf);
        const int two = r + period < a.rows ? 2 : 1;
        int shift[4] = {0, 0, 0, 0};
        if constexpr (EV == 1) {
            bool lacks = false;
            for (int g = 0; g < two; ++g) {
                shift[g] = shift_of(x, a.ldx, r + g);
                shift[2 + g] = shift_of(dy, a.lddy, r + g);
                if (row_lacks(x, a.ldx, a.rows, a.D, r + g)) {
                    patch_row(buf + (size_t)g * a.buf, x, a.ldx, a.rows, a.D, r + g, at, lanes);
                    lacks = true;
                }
                if (row_lacks(dy, a.lddy, a.rows, a.D, r + g)) {
                    patch_row(buf + (size_t)(2 + g) * a.buf, dy, a.lddy, a.rows, a.D, r + g, at, lanes);
                    lacks = true;
                }
            }
            if (lacks) team_sync(team, warps);
        }
        float2 s[2], d[2];
        float exh[2], egw[2];                              // of the single elements
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            s[g] = d[g] = make_float2(0.f, 0.f);
            exh[g] = egw[g] = 0.f;
            if (g >= two) continue;
            const float mu = __shfl_sync(0xffffffffu, now, g), is = __shfl_sync(0xffffffffu, now, 2 + g);
            const float2 is2 = make_float2(is, is), off = make_float2(-mu, -mu);
            if (PHASED && cut.column >= 0) {
                exh[g] = (ex[g] - mu) * is;
                egw[g] = ed[g] * edge_w;
                edge_dw = fmaf(ed[g], exh[g], edge_dw);
                edge_db += ed[g];
                s[g].x = egw[g];
                d[g].x = egw[g] * exh[g];
            }
            Team<T, EV, NV> vx, vd;
            vx.read_until(at_buf + g * a.buf + shift[g], place, last);
            vd.read(at_buf + (2 + g) * a.buf + shift[2 + g], place);
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                const float2 xh = mul2(add2(vx.get(i), off), is2), g0 = vd.get(i), gw = mul2(g0, kw[i]);
                dw[i] = fma2(g0, xh, dw[i]);
                db[i] = add2(db[i], g0);
                s[g] = add2(s[g], gw);
                d[g] = fma2(gw, xh, d[g]);
            }
        }
        edges(r + step);
        const float t4 = warp_sum4(s[0].x + s[0].y, d[0].x + d[0].y, s[1].x + s[1].y, d[1].x + d[1].y, lane);
        float* set = sums + turn * warps * 4;
        if ((lane & 7) == 0) set[warp * 4 + (lane >> 3)] = t4;
        team_sync(team, warps);
        // lane l adds value l % 4 of warps l / 4, l / 4 + 8, ..
        float total = 0.f;
        for (int k = lane >> 2; k < warps; k += 8) total += set[k * 4 + (lane & 3)];
        total += __shfl_xor_sync(0xffffffffu, total, 4);
        total += __shfl_xor_sync(0xffffffffu, total, 8);
        total += __shfl_xor_sync(0xffffffffu, total, 16);
        total *= -a.inv_d;
        if (!there) {                                      // a copy that never came: no number comes out
            total = __int_as_float(0x7fc00000);
#pragma unroll
            for (int i = 0; i < VALUES; ++i) dw[i] = db[i] = make_float2(total, total);
            edge_dw = edge_db = total;
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const float mu = __shfl_sync(0xffffffffu, now, g), is = __shfl_sync(0xffffffffu, now, 2 + g);
            const float ms = __shfl_sync(0xffffffffu, total, 2 * g), md = __shfl_sync(0xffffffffu, total, 2 * g + 1);
            if (g >= two || !a.dx) continue;
            const float2 is2 = make_float2(is, is), off = make_float2(-mu, -mu), ms2 = make_float2(ms, ms), md2 = make_float2(md, md);
            Team<T, EV, NV> vx, vd;
            vx.read_until(at_buf + g * a.buf + shift[g], place, last);
            vd.read(at_buf + (2 + g) * a.buf + shift[2 + g], place);
            T* dx = static_cast<T*>(a.dx) + (r + g * period) * a.D + cut.lead;
            if (PHASED && cut.column >= 0) dx[cut.column - cut.lead] = from_f32<T>(is * fmaf(exh[g], md, egw[g] + ms));
            float2 o[VALUES];
#pragma unroll
            for (int i = 0; i < VALUES; ++i) {
                const float2 xh = mul2(add2(vx.get(i), off), is2);
                o[i] = mul2(is2, fma2(xh, md2, fma2(vd.get(i), kw[i], ms2)));
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (at + k * lanes >= packs) continue;
                if constexpr (EV == 1) {
                    dx[at + k * lanes] = from_f32<T>(k & 1 ? o[k / 2].y : o[k / 2].x);
                } else {
                    float2 part[EV / 2];
#pragma unroll
                    for (int j = 0; j < EV / 2; ++j) part[j] = o[k * (EV / 2) + j];
                    store_stream<T, EV>(dx + (at + k * lanes) * EV, pack_pairs<T, EV>(part));
                }
            }
        }
        team_sync(team, warps);                            // the whole team has read the stage
        if (r + a.stages * step < a.rows) fetch(r + a.stages * step, stage);
        if (++stage == a.stages) {
            stage = 0;
            parity ^= 1;
        }
        now = next;
    }
    if (!a.part) return;
    // every copy has been waited for, so the buffers are free: [team][2][D]
    __syncthreads();
    float* all = reinterpret_cast<float*>(smem);
    auto put = [&](float* to) {
        if (PHASED && cut.column >= 0) {
            to[cut.column] = edge_dw;
            to[a.D + cut.column] = edge_db;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (at + k * lanes < packs) {
#pragma unroll
                for (int j = 0; j < EV; ++j) {
                    const int c = cut.lead + (at + k * lanes) * EV + j, i = (k * EV + j) / 2;
                    to[c] = (k * EV + j) & 1 ? dw[i].y : dw[i].x;
                    to[a.D + c] = (k * EV + j) & 1 ? db[i].y : db[i].x;
                }
            }
    };
    float* part = a.part + 2LL * blockIdx.x * a.D;
    if (teams == 1) {
        put(part);
        return;
    }
    put(all + 2LL * team * a.D);
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.D; c += blockDim.x) {
        float t = all[c];
        for (int k = 1; k < teams; ++k) t += all[2LL * k * a.D + c];
        part[c] = t;
    }
}

// ---- long rows: one block per row, the row read again from L2 for each step ---------------------
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
__global__ void __launch_bounds__(512) ln_bwd_wide(const LnBwdArgs a) {
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

// A few rows: one launch without a workspace.  Blocks below `rows` take a row each; dw and db need no row sums, so the
// blocks above add them up for 32 columns each at the same time, from the same inputs.  In a replayed graph, with it and with the
// kernels for more rows: 256 rows of 1024 bf16 4.4 and 7.3 us, 384 8.1 and 8.4, 512 11.4 and 8.6; 128 rows of 8192 bf16 7.4
// and 18.7, 1024 32.6 and 30.3.
constexpr long long kFewRows = 256, kFewElements = 1 << 20;
template <class T, class W>
__global__ void __launch_bounds__(512) ln_bwd_few(const LnBwdArgs a) {
    __shared__ float sh[2][16][33];
    const T* x = static_cast<const T*>(a.x);
    const T* dy = static_cast<const T*>(a.dy);
    const W* w = static_cast<const W*>(a.w);
    if (blockIdx.x < a.rows) {
        if (!a.dx) return;
        const long long r = blockIdx.x;
        const T *px = x + r * a.ldx, *pd = dy + r * a.lddy;
        T* dx = static_cast<T*>(a.dx) + r * a.D;
        const float mu = a.mean[r], is = a.invstd[r];
        float s = 0.f, d = 0.f;
#pragma unroll 4
        for (int i = threadIdx.x; i < a.D; i += 512) {
            const float g = to_f32(pd[i]) * (w ? to_f32(w[i]) : 1.f);
            s += g;
            d = fmaf(g, (to_f32(px[i]) - mu) * is, d);
        }
        s = warp_sum(s);
        d = warp_sum(d);
        if ((threadIdx.x & 31) == 0) {
            sh[0][threadIdx.x >> 5][0] = s;
            sh[1][threadIdx.x >> 5][0] = d;
        }
        __syncthreads();
        s = d = 0.f;
        for (int k = 0; k < 16; ++k) {
            s += sh[0][k][0];
            d += sh[1][k][0];
        }
        s *= a.inv_d;
        d *= a.inv_d;
#pragma unroll 4
        for (int i = threadIdx.x; i < a.D; i += 512) {
            const float g = to_f32(pd[i]) * (w ? to_f32(w[i]) : 1.f);
            dx[i] = from_f32<T>(is * (g - s - (to_f32(px[i]) - mu) * is * d));
        }
        return;
    }
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = (int)(blockIdx.x - a.rows) * 32 + tx;
    float dw = 0.f, db = 0.f;
    if (c < a.D) {
#pragma unroll 4
        for (long long r = ty; r < a.rows; r += 16) {
            const float g = to_f32(dy[r * a.lddy + c]);
            dw = fmaf(g, (to_f32(x[r * a.ldx + c]) - a.mean[r]) * a.invstd[r], dw);
            db += g;
        }
    }
    sh[0][ty][tx] = dw;
    sh[1][ty][tx] = db;
    __syncthreads();
    if (ty < 2 && c < a.D) {
        float t = 0.f;
        for (int k = 0; k < 16; ++k) t += sh[ty][k][tx];
        W* out = static_cast<W*>(ty ? a.db : a.dw);
        if (out) out[c] = from_f32<W>(t);
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

// The slices' (or blocks') sums: 32 columns and 32 runs of slices to a block, the runs added in a fixed order.  Launched
// as the programmatic dependent of the kernel that makes the sums.  148 blocks' sums of 2048 columns: 7.2 us by itself and cold,
// under ncu.
template <class W>
__global__ void __launch_bounds__(1024) ln_bwd_fold(const LnBwdArgs a) {
    __shared__ float sh[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long long i = blockIdx.x * 32LL + tx;                   // of 2 D values
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float t = 0.f;
    if (i < 2LL * a.D) {
        const int per = (a.slices + 31) / 32, s0 = ty * per, s1 = min(a.slices, s0 + per);
#pragma unroll 16
        for (int s = s0; s < s1; ++s) t += a.part[2LL * s * a.D + i];
    }
    sh[ty][tx] = t;
    __syncthreads();
    t = warp_sum(sh[tx][ty]);                                     // warp k adds column k
    const long long o = blockIdx.x * 32LL + ty;
    if (tx == 0 && o < 2LL * a.D) {
        W* out = static_cast<W*>(o < a.D ? a.dw : a.db);
        if (out) out[o < a.D ? o : o - a.D] = from_f32<W>(t);
    }
}

constexpr int kMaxParts = 1184;       // blocks whose sums the workspace holds: 8 on each of 148 SMs

// slices of the column sums of long rows
int ln_slices(int64_t rows) {
    const int64_t s = (rows + 31) / 32;
    return (int)(s < 1 ? 1 : s > 296 ? 296 : s);
}

template <int N>
using Num = std::integral_constant<int, N>;

// lanes that share a short row of `packs` accesses, nv each: the fewest, a power of two
int short_lanes(long long packs, int nv) {
    int lanes = 32;
    while (lanes > 1 && (long long)(lanes / 2) * nv >= packs) lanes /= 2;
    return lanes;
}

constexpr size_t kRowSmem = 200 * 1024;      // of the 227 KB that a block may have

template <class T, class W, int EV, int NV>
int ln_fwd_short_launch(LnFwdArgs a, int sms, cudaStream_t s) {
    auto kern = ln_fwd_short<T, W, EV, NV>;
    a.lanes = short_lanes(a.D / EV, NV);
    const int per = 256 / a.lanes;
    const long long want = (a.rows + per - 1) / per, most = (long long)sms * resident_blocks((const void*)kern, 256, 0);
    return launch_kernel(kern, (int)(want < most ? want : most), 256, 0, s, false, a);
}

// One block of up to 16 warps to an SM; as many teams as there are rows for, as many buffers as fit (up to 4).
template <class T, class W, int EV, int NV, bool PHASED = false>
int ln_fwd_rows_launch(LnFwdArgs a, int team, int sms, cudaStream_t s) {
    const long long per_sm = (a.rows + sms - 1) / sms;
    int teams = 16 / team;
    if (per_sm < teams) teams = (int)per_sm;
    a.team = team;
    a.buf = (int)((a.D * sizeof(T) + 15) / 16 * 16 + (EV == 1 ? 16 : 0));
    a.wbytes = (a.D * 4 + 15) / 16 * 16;
    while (teams > 1 && 2 * (size_t)a.wbytes + (size_t)teams * a.buf > kRowSmem) --teams;
    const size_t room = (kRowSmem - 2 * (size_t)a.wbytes) / ((size_t)teams * a.buf);
    a.stages = (int)(room > 4 ? 4 : room);
    const size_t smem = 2 * (size_t)a.wbytes + (size_t)teams * a.stages * (a.buf + 8) + 2 * (size_t)teams * team * sizeof(float2);
    const long long want = (a.rows + teams - 1) / teams;
    int grid = (int)(want < sms ? want : sms);
    if (PHASED && grid < a.period) grid = a.period;          // each distance has a block
    return launch_kernel(ln_fwd_rows<T, W, EV, NV, PHASED>, grid, teams * team * 32, smem, s, false, a);
}

template <class T, class W, int EV, int NV>
int ln_bwd_short_launch(LnBwdArgs& a, int sms, cudaStream_t s) {
    auto kern = ln_bwd_short<T, W, EV, NV>;
    a.lanes = short_lanes(a.D / EV, NV);
    const int per = 256 / a.lanes;
    const size_t smem = (size_t)2 * NV * EV * 256 * 4;
    const long long want = (a.rows + per - 1) / per;
    long long most = (long long)sms * resident_blocks((const void*)kern, 256, smem);
    most = most < kMaxParts ? most : kMaxParts;
    a.slices = (int)(want < most ? want : most);
    return launch_kernel(kern, a.slices, 256, smem, s, false, a);
}

// Teams of as many warps as the row's columns need, 16 columns to a thread: up to 16 warps and as many teams to a block as
// fit with two stages each (one team with one stage for the longest rows).
template <class T, class W, int EV, int NV, bool PHASED = false>
int ln_bwd_rows_launch(LnBwdArgs& a, int sms, cudaStream_t s) {
    auto kern = ln_bwd_rows<T, W, EV, NV, PHASED>;
    a.lanes = (int)((a.D / EV + 32 * NV - 1) / (32 * NV) * 32);
    // a row (EV = 1: that begins up to 15 bytes into its buffer), then zeros for one access where there are places beyond it
    const size_t row = (a.D * sizeof(T) + 15) / 16 * 16 + (EV == 1 ? 16 : 0);
    a.buf = PHASED || a.D / EV % (NV * a.lanes) != 0 ? (int)(row + (EV == 1 ? 32 : 16) + 127) / 128 * 128 : (int)row;
    a.stages = 8 * row <= kRowSmem ? 2 : 1;
    const long long pairs = (a.rows + 1) / 2;
    int teams = 512 / a.lanes;
    while (teams > 1 && ((size_t)teams * a.stages * 4 * row > kRowSmem || (long long)(teams - 1) * sms >= pairs)) --teams;
    // a team's dw and db, 8 D bytes, fit its buffers: 16 D with two stages of 16-bit rows
    const size_t smem = (size_t)teams * (a.stages * 4 * (size_t)a.buf + 16 + (size_t)(a.lanes / 32) * 32);
    const long long want = (pairs + teams - 1) / teams;
    long long most = (long long)sms * resident_blocks((const void*)kern, teams * a.lanes, smem);
    most = most < kMaxParts ? most : kMaxParts;
    a.slices = (int)(want < most ? want : most);
    if (PHASED && a.slices * teams < a.period) a.slices = (a.period + teams - 1) / teams;      // each distance has a team
    return launch_kernel(kern, a.slices, teams * a.lanes, smem, s, false, a);
}

// rows at p begin as far behind a 16-byte boundary as those of x [..][D] without gaps
bool rows_alike(const void* x, const void* p, int64_t ld, int D, size_t es) {
    return ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0 && (ld - D) * (int64_t)es % 16 == 0;
}
// rows after which that distance comes back
int rows_period(int D, size_t es) {
    int n = 1;
    while (n * (D * es % 16) % 16 != 0) n *= 2;
    return n;
}
bool ln_shape_ok(int64_t rows, int D, int64_t ld) { return rows >= 0 && D > 0 && (rows <= 1 || ld >= D); }

}  // namespace

extern "C" {

int hfuse_layernorm(const void* x, int64_t rows, int D, int64_t ld_x, int dtype, const void* weight, const void* bias,
                    int weight_dtype, float eps, void* y, float* mean, float* invstd, hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || (weight_dtype != dtype && weight_dtype != HFUSE_F32)) return HFUSE_ERR_BAD_ARG;
    if (!ln_shape_ok(rows, D, ld_x) || !(eps >= 0.f)) return HFUSE_ERR_BAD_ARG;
    if (D > kMaxWidth) return HFUSE_ERR_TOO_LARGE;
    if (rows == 0) return HFUSE_OK;
    if (!x || !y || !mean || !invstd) return HFUSE_ERR_BAD_ARG;
    const size_t es = lm_type_size(dtype), ws = lm_type_size(weight_dtype);
    if (!aligned_to(x, es) || !aligned_to(y, es) || !aligned_to(weight, ws) || !aligned_to(bias, ws) || !aligned_to(mean, 4) ||
        !aligned_to(invstd, 4))
        return HFUSE_ERR_ALIGNMENT;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    LnFwdArgs a{};
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.invstd = invstd;
    a.rows = rows; a.ldx = ld_x; a.D = D; a.inv_d = 1.f / (float)D; a.eps = eps;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = aligned_to(x, 16) && aligned_to(y, 16) && aligned_to(weight, 16) && aligned_to(bias, 16) &&
                      D * es % 16 == 0 && ld_x * es % 16 == 0;
    const bool phased = !wide && rows_alike(x, x, ld_x, D, es) && rows_alike(x, y, D, D, es);
    a.period = rows_period(D, es);
    return by_types(dtype, weight_dtype, [&](auto t, auto w) {
        using T = typename decltype(t)::type;
        using W = typename decltype(w)::type;
        constexpr int EV = 16 / sizeof(T);
        const long long packs = wide ? D / EV : D;
        // short rows: up to 4 accesses of 32 lanes (unaligned: 2)
        if (wide && packs <= 32) return ln_fwd_short_launch<T, W, EV, 1>(a, f.sms, s);
        if (wide && packs <= 64) return ln_fwd_short_launch<T, W, EV, 2>(a, f.sms, s);
        if (!wide && packs <= 32) return ln_fwd_short_launch<T, W, 1, 1>(a, f.sms, s);
        if (!wide && packs <= 64) return ln_fwd_short_launch<T, W, 1, 2>(a, f.sms, s);
        // Rows that fit shared memory beside their weights.  Few rows are spread over twice the warps each: 4096 bf16 wide, in a
        // replayed graph, 296 rows take 4.5 instead of 5.6 us, 592 5.1 and 5.6, 888 6.9 and 6.4, 2368 11.5 and 10.1.
        const bool few = rows < 4LL * f.sms;
        auto team = [&](int nv) { return (int)(((phased ? D / EV : packs) + 32LL * nv - 1) / (32LL * nv)); };
        if (8 * (size_t)D + D * es + 64 <= kRowSmem) {
            if (phased && D / EV <= 32 * 4 * 16 && (few || D / EV <= 32 * 4))
                return ln_fwd_rows_launch<T, W, EV, 4, true>(a, team(4), f.sms, s);
            if (phased && D / EV <= 32 * 8 * 16) return ln_fwd_rows_launch<T, W, EV, 8, true>(a, team(8), f.sms, s);
            if (wide && packs <= 32 * 4 * 16 && (few || packs <= 32 * 4)) return ln_fwd_rows_launch<T, W, EV, 4>(a, team(4), f.sms, s);
            if (wide && packs <= 32 * 8 * 16) return ln_fwd_rows_launch<T, W, EV, 8>(a, team(8), f.sms, s);
            if (!wide && packs <= 32 * 8 * 16 && (few || packs <= 32 * 8)) return ln_fwd_rows_launch<T, W, 1, 8>(a, team(8), f.sms, s);
            if (!wide && packs <= 32 * 32 * 16) return ln_fwd_rows_launch<T, W, 1, 32>(a, team(32), f.sms, s);
        }
        const int grid = (int)(rows < f.sms * 4LL ? rows : f.sms * 4LL);
        return launch_kernel(ln_fwd_wide<T, W>, grid, 512, 0, s, false, a);
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
    if (D > kMaxWidth) return HFUSE_ERR_TOO_LARGE;
    if (rows > 0 && (!x || !grad_out || !mean || !invstd)) return HFUSE_ERR_BAD_ARG;
    const bool want_w = grad_weight || grad_bias;
    if (!want_w && (rows == 0 || !grad_in)) return HFUSE_OK;
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
    LnBwdArgs a{};
    a.x = x; a.dy = grad_out; a.w = weight; a.mean = mean; a.invstd = invstd;
    a.dx = grad_in; a.dw = grad_weight; a.db = grad_bias; a.part = want_w ? static_cast<float*>(workspace) : nullptr;
    a.rows = rows; a.ldx = ld_x; a.lddy = ld_grad_out; a.D = D; a.inv_d = 1.f / (float)D;
    a.slices = slices; a.slice_rows = (rows + slices - 1) / slices;
    const bool wide = aligned_to(x, 16) && aligned_to(grad_out, 16) && aligned_to(grad_in, 16) && aligned_to(weight, 16) &&
                      D * es % 16 == 0 && ld_x * es % 16 == 0 && ld_grad_out * es % 16 == 0;
    const bool phased = rows_alike(x, x, ld_x, D, es) && rows_alike(x, grad_out, ld_grad_out, D, es) && (!grad_in || rows_alike(x, grad_in, D, D, es));
    a.period = rows_period(D, es);
    return by_types(dtype, weight_dtype, [&](auto t, auto w) {
        using T = typename decltype(t)::type;
        using W = typename decltype(w)::type;
        constexpr int EV = 16 / sizeof(T), NV = 16 / EV;               // 16 columns to a thread
        const long long packs = wide ? D / EV : D;
        int rc;
        // one launch instead of two: 8.3 instead of 10 to 12 us a call of a few rows, which is the host's time
        if (rows <= kFewRows && rows * (long long)D <= kFewElements)
            return launch_kernel(ln_bwd_few<T, W>, (int)rows + (want_w ? (D + 31) / 32 : 0), 512, 0, s, false, a);
        if (rows > 0 && packs <= 64) {
            rc = wide ? packs <= 32 ? ln_bwd_short_launch<T, W, EV, 1>(a, f.sms, s) : ln_bwd_short_launch<T, W, EV, 2>(a, f.sms, s)
                      : packs <= 32 ? ln_bwd_short_launch<T, W, 1, 1>(a, f.sms, s) : ln_bwd_short_launch<T, W, 1, 2>(a, f.sms, s);
        } else if (rows > 0 && D <= 16 * 512) {
            rc = wide           ? ln_bwd_rows_launch<T, W, EV, NV>(a, f.sms, s)
                 : phased       ? ln_bwd_rows_launch<T, W, EV, NV, true>(a, f.sms, s)
                 : D <= 8 * 512 ? ln_bwd_rows_launch<T, W, 1, 8>(a, f.sms, s) : ln_bwd_rows_launch<T, W, 1, 16>(a, f.sms, s);
        } else {
            if (grad_in && rows > 0) {
                const int grid = (int)(rows < f.sms * 4LL ? rows : f.sms * 4LL);
                if ((rc = launch_kernel(ln_bwd_wide<T, W>, grid, 512, 0, s, false, a))) return rc;
            }
            if (!want_w) return (int)HFUSE_OK;
            ln_bwd_cols<T><<<dim3((unsigned)((D + 31) / 32), (unsigned)slices), 256, 0, s>>>(a);
            rc = check_launch();
        }
        if (rc || !want_w) return rc;
        return launch_kernel(ln_bwd_fold<W>, (int)((2LL * D + 31) / 32), 1024, 0, s, true, a);
    });
}

}  // extern "C"
