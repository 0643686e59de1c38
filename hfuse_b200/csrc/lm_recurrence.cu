// Gated linear recurrence along the steps of a sequence, forward and backward.
//
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  out_t = h_t      (per batch item and channel)
//   e_t = dout_t + a_{t+1} e_{t+1},  dx_t = (1 - a_t) e_t,  dgate_t = e_t (h_{t-1} - x_t) a_t (1 - a_t),  dh_0 = a_1 e_1
//
// A gate of -infinity starts afresh (h_t = x_t), one of +infinity holds the state.
//
// Steps s .. t together map a state h to A h + H with A the product of their a and H their result from zero, and two
// such maps make one: (A2, H2) after (A1, H1) is (A2 A1, A2 H1 + H2).  So a block takes 32 lanes' worth of channels
// of one sequence, each of its warps runs kSteps steps of them from zero in registers, the warps' maps meet in
// shared memory, and each warp adds what the state before its first step contributes: A_t times that state.  One
// pass over the data: gate and x are read once and out is written once; the block moves on through the sequence
// with the state in registers.  The backward pass does the same from the end (its maps are e -> A e + E),
// with the states before each step run again from the ones that the forward pass saved every 256 steps.
//
// The next pieces of the sequence are on their way into shared memory while one is worked on: as TMA tiles where the tensors
// allow it (the results take the places of the inputs and leave as tiles too, all issued by a warp of its own, so that
// the others only compute), else by cp.async.  Where there are fewer groups of channels than the GPU has room for, a
// cluster of blocks shares a group: each takes a piece in turn and the blocks' maps are exchanged through
// distributed shared memory.
#include <cuda.h>

#include <initializer_list>

#include "launch.cuh"
#include "lm_common.cuh"

using namespace hfuse;

namespace {

constexpr int kSaved = HFUSE_RECURRENCE_CHUNK;
constexpr int kWarpsFwd = 8, kWarpsBwd = 16, kSteps = 16;     // a whole piece of the backward pass is kSaved steps
static_assert(kWarpsBwd * kSteps == kSaved && kSaved % kSteps == 0, "pieces begin where states are saved");
constexpr int kMaxCluster = 8;

struct RecArgs {
    const void *gate, *x, *dy;
    const float *h0, *dlast;
    void *y, *dgate, *dx;
    float *last, *states, *dh0;
    long long gate_b, gate_t, x_b, x_t, dy_b, dy_t;       // strides of a batch item and of a step
    int B, T, D, chunks;
    int groups;              // groups of channels per sequence
    int split;               // blocks that share a group
};

// a = sigmoid(g) and z = 1 - a = sigmoid(-g): with e = exp(-g), a = 1 / (1 + e) and z = e a.  From e = 2^126 on (gates below
// -87.3, -infinity among them) the reciprocal is flushed to zero; e a would then be zero or no number, and z is one.  The
// exponent is a product rounded to 32 bits, so e's relative error grows with the gate: about (4 + 1.3 |g|) 2^-24, and a few
// roundings more for a and z.  A gate that is a NaN makes both one.
__device__ __forceinline__ void gates2(float2 g, float2& a, float2& z) {
    const float2 t = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    float2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    const float2 d = add2(e, make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a.y) : "f"(d.y));
    z = mul2(e, a);
    z.x = a.x == 0.f ? 1.f : z.x;
    z.y = a.y == 0.f ? 1.f : z.y;
}

// ---- staging: `rows` steps of 32 * CPL channels into shared memory ----------------------------------------
// ALIGN: bytes that every row's begin and the number of channels are a multiple of (16, 4, or one 16-bit element)
__device__ __forceinline__ void cp_async16(uint32_t s, const void* g) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(__cvta_generic_to_global(g)) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t s, const void* g) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s), "l"(__cvta_generic_to_global(g)) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Steps from T on get `beyond` (a gate of +infinity and an x of zero leave the state as it is), channels from D on are
// left alone: no result of theirs is stored.
template <class T, int CPL, int ALIGN, int S>
__device__ __forceinline__ void stage_rows(T* dst, const T* src, long long stride, int t0, int rows, int d0, int T_end, int D,
                                           float beyond) {
    constexpr int C = 32 * CPL, E = ALIGN >= (int)sizeof(T) ? ALIGN / (int)sizeof(T) : 1, PER = C / E;
    constexpr int COLS = PER < 32 ? PER : 32;                // accesses of a row that a warp has in its lanes
    constexpr int COUNT = S * COLS / 32;                     // accesses of a thread in its column: rows / step
    const int step = blockDim.x / COLS, r0 = threadIdx.x / COLS, in = T_end - t0;
#pragma unroll
    for (int k0 = 0; k0 < PER; k0 += COLS) {
        const int k = (k0 + threadIdx.x % COLS) * E;
        if (d0 + k >= D) continue;
        const T* from = src + (long long)(t0 + r0) * stride + d0 + k;
        T* to = dst + r0 * C + k;
        const long long ahead = step * stride;
        const uint32_t s0 = smem_u32(to), sahead = step * C * (int)sizeof(T);
        if (in >= rows) {                                    // all pieces but a sequence's last one
#pragma unroll
            for (int j = 0; j < COUNT; ++j) {
                if constexpr (ALIGN == 16) cp_async16(s0 + j * sahead, from + j * ahead);
                else if constexpr (ALIGN == 4) cp_async4(s0 + j * sahead, from + j * ahead);
                else to[j * step * C] = from[j * ahead];
            }
        } else {
            for (int j = 0; j < COUNT; ++j) {
                if (r0 + j * step < in) {
                    if constexpr (ALIGN == 16) cp_async16(s0 + j * sahead, from + j * ahead);
                    else if constexpr (ALIGN == 4) cp_async4(s0 + j * sahead, from + j * ahead);
                    else to[j * step * C] = from[j * ahead];
                } else {
#pragma unroll
                    for (int q = 0; q < E; ++q) to[j * step * C + q] = from_f32<T>(beyond);
                }
            }
        }
    }
}

// Elements are worked on in pairs: the two channels of a lane, or two steps of its only channel.
template <class T, int CPL>
__device__ __forceinline__ float2 read_pair(const T* at, int i) {
    constexpr int C = 32 * CPL;
    if constexpr (CPL == 2) {
        return pair_of(*reinterpret_cast<const Pack<T, 2>*>(at + i * C), 0);
    } else {
        return make_float2(to_f32(at[2 * i * C]), to_f32(at[(2 * i + 1) * C]));
    }
}
// h -> a h + b over a pair; `all` are the results (before: what h was ahead of each)
template <int CPL>
__device__ __forceinline__ float2 run_pair(float2 a, float2 b, float (&h)[CPL], float2* before = nullptr) {
    if constexpr (CPL == 2) {
        const float2 old = make_float2(h[0], h[1]), r = fma2(a, old, b);
        h[0] = r.x;
        h[1] = r.y;
        if (before) *before = old;
        return r;
    } else {
        const float x = fmaf(a.x, h[0], b.x), y = fmaf(a.y, x, b.y);
        if (before) *before = make_float2(h[0], x);
        h[0] = y;
        return make_float2(x, y);
    }
}
// the same for a product
template <int CPL>
__device__ __forceinline__ float2 scale_pair(float2 a, float (&A)[CPL]) {
    if constexpr (CPL == 2) {
        const float2 r = mul2(a, make_float2(A[0], A[1]));
        A[0] = r.x;
        A[1] = r.y;
        return r;
    } else {
        const float x = a.x * A[0], y = a.y * x;
        A[0] = y;
        return make_float2(x, y);
    }
}
template <int CPL>
__device__ __forceinline__ float2 both(const float (&v)[CPL]) { return make_float2(v[0], v[CPL - 1]); }

// a pair to its place: `steps` steps and `left` channels are there
template <class T, int CPL, bool WHOLE>
__device__ __forceinline__ void write_pair(T* at, long long stride, int i, float2 v, int steps, int left) {
    if constexpr (CPL == 2) {
        if constexpr (WHOLE) {             // rows keep the alignment of two elements, D is even
            const float2 w[1] = {v};
            if (i < steps && left > 0) store_stream<T, 2>(at + i * stride, pack_pairs<T, 2>(w));
        } else if (i < steps) {
            if (left > 0) at[i * stride] = from_f32<T>(v.x);
            if (left > 1) at[i * stride + 1] = from_f32<T>(v.y);
        }
    } else if (left > 0) {
        if (2 * i < steps) at[2 * i * stride] = from_f32<T>(v.x);
        if (2 * i + 1 < steps) at[(2 * i + 1) * stride] = from_f32<T>(v.y);
    }
}
template <int CPL>
__device__ __forceinline__ void read_state(const float* p, float (&v)[CPL], int left) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) v[c] = p && c < left ? p[c] : 0.f;
}
template <int CPL>
__device__ __forceinline__ void write_state(float* p, const float (&v)[CPL], int left) {
#pragma unroll
    for (int c = 0; c < CPL; ++c)
        if (c < left) p[c] = v[c];
}

// ---- maps h -> A h + H of one stretch of steps in shared memory: a lane's A, then its H ---------------------
template <int CPL>
__device__ __forceinline__ void write_map(float* m, const float (&A)[CPL], const float (&H)[CPL]) {
    if constexpr (CPL == 2) *reinterpret_cast<float4*>(m) = make_float4(A[0], A[1], H[0], H[1]);
    else *reinterpret_cast<float2*>(m) = make_float2(A[0], H[0]);
}
template <int CPL>
__device__ __forceinline__ void apply_map(const float* m, float (&h)[CPL]) {
    if constexpr (CPL == 2) {
        const float4 r = *reinterpret_cast<const float4*>(m);
        const float2 n = fma2(make_float2(r.x, r.y), make_float2(h[0], h[1]), make_float2(r.z, r.w));
        h[0] = n.x;
        h[1] = n.y;
    } else {
        const float2 r = *reinterpret_cast<const float2*>(m);
        h[0] = fmaf(r.x, h[0], r.y);
    }
}
// the map of the steps so far, then m's
template <int CPL>
__device__ __forceinline__ void join_map(const float* m, float (&A)[CPL], float (&H)[CPL]) {
    apply_map<CPL>(m, H);
#pragma unroll
    for (int c = 0; c < CPL; ++c) A[c] *= m[c];
}

// ---- cluster: the blocks that share a group of channels --------------------------------------------------
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_peer(const void* p, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    return at;
}
// two floats of a map into a peer's shared memory; their 8 bytes are counted on the peer's mbarrier, so neither side
// needs a fence or a barrier of the whole cluster
__device__ __forceinline__ void send_two(uint32_t to, uint32_t bar, float A, float H) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(A), "f"(H),
                 "r"(bar)
                 : "memory");
}
constexpr unsigned long long kPeerWaitNs = 2000000000ull;

// The maps of all blocks of the cluster: sets of maps that alternate, each with an mbarrier.  A block sends a set only
// after all its warps have read the last one, and it receives a set only after every block has sent the one before,
// so no set is written while it is read.
template <int CPL>
struct Peers {
    static constexpr int C = 32 * CPL;
    float* sets;                   // [2][kMaxCluster][C]{A, H}
    unsigned long long* bars;      // [2]
    int split, rank;
    bool lost = false;             // a wait ran out: results become NaN

    __device__ __forceinline__ Peers(float* at, int split_, int rank_)
        : sets(at), bars(reinterpret_cast<unsigned long long*>(at + 2 * kMaxCluster * C * 2)), split(split_), rank(rank_) {}
    __device__ __forceinline__ void spoil(float (&u)[CPL], float (&v)[CPL]) const {
        if (!lost) return;
#pragma unroll
        for (int c = 0; c < CPL; ++c) u[c] = v[c] = __int_as_float(0x7fc00000);
    }
    __device__ __forceinline__ void begin() {
        if (threadIdx.x == 0) {
            mbar_init(bars, 1);
            mbar_init(bars + 1, 1);
            fence_mbar_init();
        }
        __syncthreads();
        cluster_sync();            // every block's barriers are there
    }
    // called by the warps below `split`: warp j sends to block j
    __device__ __forceinline__ void send(int it, int warp, int lane, const float (&A)[CPL], const float (&H)[CPL]) {
        if (threadIdx.x == 0) mbar_expect_tx(bars + (it & 1), (uint32_t)(split * C * 8));
        const uint32_t bar = at_peer(bars + (it & 1), warp);
        const uint32_t to = at_peer(sets + (((it & 1) * kMaxCluster + rank) * C + lane * CPL) * 2, warp);
        if constexpr (CPL == 2) {
            send_two(to, bar, A[0], A[1]);
            send_two(to + 8, bar, H[0], H[1]);
        } else {
            send_two(to, bar, A[0], H[0]);
        }
    }
    __device__ __forceinline__ const float* receive(int it, int lane) {
        if (!lost) lost = !mbar_wait<true>(bars + (it & 1), (it >> 1) & 1, kPeerWaitNs);
        return sets + ((it & 1) * kMaxCluster * C + lane * CPL) * 2;
    }
};

// ---- the steps of a piece, shared by both kinds of staging ------------------------------------------------
// forward: results from zero and products of the a so far, for the warp's steps
template <class T, int CPL, int N>
__device__ __forceinline__ void run_forward(const T* sg, const T* sx, float2 (&h)[N], float2 (&a)[N], float (&A)[CPL], float (&H)[CPL]) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) { H[c] = 0.f; A[c] = 1.f; }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float2 at, zt;
        gates2(read_pair<T, CPL>(sg, i), at, zt);
        h[i] = run_pair<CPL>(at, mul2(zt, read_pair<T, CPL>(sx, i)), H);
        a[i] = scale_pair<CPL>(at, A);
    }
}
// After the barrier behind write_map: the state before the warp's first step (in), and the one before the next piece
// (carry), which a single block's last warp hands on through `next`, [2][C], and a cluster's warps all know.
template <int CPL>
__device__ __forceinline__ void join_forward(const float* map, float* next, int it, int W, int warp, int lane, float (&A)[CPL], float (&H)[CPL],
                                             float (&in)[CPL], float (&carry)[CPL], Peers<CPL>& peers) {
    constexpr int C = 32 * CPL;
    if (peers.split == 1) {
        if (it > 0) read_state<CPL>(next + (it & 1) * C, carry, CPL);
#pragma unroll
        for (int c = 0; c < CPL; ++c) in[c] = carry[c];
#pragma unroll 4
        for (int w = 0; w < warp; ++w) apply_map<CPL>(map + w * 2 * C, in);
        if (warp == W - 1) {
#pragma unroll
            for (int c = 0; c < CPL; ++c) next[(~it & 1) * C + c] = carry[c] = fmaf(A[c], in[c], H[c]);
        }
        return;
    }
    if (warp < peers.split) {                             // W >= split: see rec_launch
#pragma unroll
        for (int c = 0; c < CPL; ++c) { A[c] = 1.f; H[c] = 0.f; }
#pragma unroll 4
        for (int w = 0; w < W; ++w) join_map<CPL>(map + w * 2 * C, A, H);
        peers.send(it, warp, lane, A, H);
    }
    const float* set = peers.receive(it, lane);
#pragma unroll 4
    for (int j = 0; j < peers.rank; ++j) apply_map<CPL>(set + j * 2 * C, carry);
#pragma unroll
    for (int c = 0; c < CPL; ++c) in[c] = carry[c];
#pragma unroll 4
    for (int w = 0; w < warp; ++w) apply_map<CPL>(map + w * 2 * C, in);
#pragma unroll 4
    for (int j = peers.rank; j < peers.split; ++j) apply_map<CPL>(set + j * 2 * C, carry);
    peers.spoil(in, carry);
}

// backward: a, 1 - a and the maps of the warp's steps.  E, what e of zero becomes over the steps, is the sum of dy_t times
// the product of the a up to a_t.
template <class T, int CPL, int N>
__device__ __forceinline__ void run_backward(const T* sg, const T* sx, const T* sd, float2 (&a)[N], float2 (&z)[N], float (&A)[CPL],
                                             float (&H)[CPL], float (&E)[CPL]) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) { A[c] = 1.f; H[c] = E[c] = 0.f; }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        gates2(read_pair<T, CPL>(sg, i), a[i], z[i]);
        run_pair<CPL>(a[i], mul2(z[i], read_pair<T, CPL>(sx, i)), H);
        const float2 P = scale_pair<CPL>(a[i], A), u = read_pair<T, CPL>(sd, i);
        if constexpr (CPL == 2) {
            const float2 r = fma2(P, u, make_float2(E[0], E[1]));
            E[0] = r.x;
            E[1] = r.y;
        } else {
            E[0] = fmaf(P.y, u.y, fmaf(P.x, u.x, E[0]));
        }
    }
}
// The warps' A, H and E, [W][C] each.
template <int CPL>
struct Maps3 {
    static constexpr int C = 32 * CPL;
    float* at;                   // this lane's place
    int W;
    __device__ __forceinline__ void write(int warp, const float (&A)[CPL], const float (&H)[CPL], const float (&E)[CPL]) const {
        write_state<CPL>(at + warp * C, A, CPL);
        write_state<CPL>(at + (W + warp) * C, H, CPL);
        write_state<CPL>(at + (2 * W + warp) * C, E, CPL);
    }
    // v -> A v + H (which = 1) or A v + E (which = 2) of warp w
    __device__ __forceinline__ void apply(int w, int which, float (&v)[CPL]) const {
        const float *A = at + w * C, *B = at + (which * W + w) * C;
        if constexpr (CPL == 2) {
            const float2 r = fma2(*reinterpret_cast<const float2*>(A), make_float2(v[0], v[1]), *reinterpret_cast<const float2*>(B));
            v[0] = r.x;
            v[1] = r.y;
        } else {
            v[0] = fmaf(A[0], v[0], B[0]);
        }
    }
};
// After the barrier behind Maps3::write.  First what the other blocks wait for: the map of the whole piece.
template <int CPL>
__device__ __forceinline__ void send_backward(const Maps3<CPL>& maps, int k, int warp, int lane, Peers<CPL>& peers) {
    if (warp >= peers.split || peers.split == 1) return;
    float A[CPL], E[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) { A[c] = 1.f; E[c] = 0.f; }
#pragma unroll 4
    for (int w = maps.W - 1; w >= 0; --w) {
        maps.apply(w, 2, E);
#pragma unroll
        for (int c = 0; c < CPL; ++c) A[c] *= maps.at[w * maps.C + c];
    }
    peers.send(k, warp, lane, A, E);
}
// Then, while it is on its way, dgate's factor (h_{t-1} - x_t) a z of each step: the states run again from hb, the one
// before the piece.
template <class T, int CPL, int N>
__device__ __forceinline__ void factors_backward(const Maps3<CPL>& maps, int warp, const T* sx, const float2 (&a)[N], const float2 (&z)[N],
                                                 float (&hb)[CPL], float2 (&f)[N]) {
#pragma unroll 4
    for (int w = 0; w < warp; ++w) maps.apply(w, 1, hb);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 v = read_pair<T, CPL>(sx, i);
        float2 before;
        run_pair<CPL>(a[i], mul2(z[i], v), hb, &before);
        f[i] = mul2(fma2(v, make_float2(-1.f, -1.f), before), mul2(a[i], z[i]));
    }
}
// e from behind the warp's last step; A and E are the warp's own
template <int CPL>
__device__ __forceinline__ void join_backward(const Maps3<CPL>& maps, float* next, int k, int warp, int lane, const float (&A)[CPL],
                                              const float (&E)[CPL], float (&e)[CPL], float (&carry)[CPL], Peers<CPL>& peers) {
    constexpr int C = 32 * CPL;
    if (peers.split == 1) {
        if (k > 0) read_state<CPL>(next + (k & 1) * C, carry, CPL);
#pragma unroll
        for (int c = 0; c < CPL; ++c) e[c] = carry[c];
#pragma unroll 4
        for (int w = maps.W - 1; w > warp; --w) maps.apply(w, 2, e);
        if (warp == 0) {
#pragma unroll
            for (int c = 0; c < CPL; ++c) next[(~k & 1) * C + c] = carry[c] = fmaf(A[c], e[c], E[c]);
        }
        return;
    }
    const float* set = peers.receive(k, lane);
#pragma unroll 4
    for (int j = peers.split - 1; j > peers.rank; --j) apply_map<CPL>(set + j * 2 * C, carry);
#pragma unroll
    for (int c = 0; c < CPL; ++c) e[c] = carry[c];
#pragma unroll 4
    for (int w = maps.W - 1; w > warp; --w) maps.apply(w, 2, e);
#pragma unroll 4
    for (int j = peers.rank; j >= 0; --j) apply_map<CPL>(set + j * 2 * C, carry);
    peers.spoil(e, carry);
}
// dgate and dx of the warp's steps, put(i, dgate, dx) for every pair from the last one on
template <class T, int CPL, int N, class Put>
__device__ __forceinline__ void sweep_backward(const T* sd, const float2 (&a)[N], const float2 (&z)[N], const float2 (&f)[N], float (&e)[CPL], Put&& put) {
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {
        const float2 u = read_pair<T, CPL>(sd, i);
        float2 et;                                        // e of the pair's steps
        if constexpr (CPL == 2) {
            et = add2(make_float2(e[0], e[1]), u);
            const float2 r = mul2(et, a[i]);
            e[0] = r.x;
            e[1] = r.y;
        } else {
            et.y = e[0] + u.y;
            et.x = fmaf(et.y, a[i].y, u.x);
            e[0] = et.x * a[i].x;
        }
        put(i, mul2(et, f[i]), mul2(et, z[i]));
    }
}

// ---- staging by cp.async -----------------------------------------------------------------------------------
// [2 stages][tensors][rows][C], the warps' maps (the barrier at the top of a piece is behind their last reader), next, peers.
// For single steps (64 x 2048 bf16: 7 us a call, which is the host's time; 3.5 us in a replayed graph, of which an empty kernel
// takes 0.5), short sequences and strides that tiles do not take.
// 8 x 4096 steps of 2048 bf16 channels took 73 us with it, its gradient's 4 x 8192 steps of 1024 86 us: the staging's
// instructions are what tiles save.
template <class T, int CPL, int S, int ALIGN>
__global__ void __launch_bounds__(256, 2) rec_fwd(const RecArgs p) {
    constexpr int C = 32 * CPL, N = S * CPL / 2;
    extern __shared__ __align__(128) unsigned char smem[];
    const int W = blockDim.x >> 5, warp = warp_index(), lane = threadIdx.x & 31, rows = W * S;
    T* stage = reinterpret_cast<T*>(smem);
    float* map = reinterpret_cast<float*>(smem + 4 * (size_t)rows * C * sizeof(T));      // [W][C]{A, H}
    float* next = map + 2 * W * C;
    Peers<CPL> peers(next + 2 * C, p.split, blockIdx.x % p.split);
    const int group = blockIdx.x / p.split, b = group / p.groups, d0 = (group - b * p.groups) * C, d = d0 + lane * CPL, left = p.D - d;
    const T* gate = static_cast<const T*>(p.gate) + b * p.gate_b;
    const T* x = static_cast<const T*>(p.x) + b * p.x_b;
    T* y = static_cast<T*>(p.y) + (long long)b * p.T * p.D + d;
    const int n = (p.T + rows * p.split - 1) / (rows * p.split);
    const long long at_state = (long long)b * p.D + d;

    auto issue = [&](int it) {
        if (it < n) {
            T* s = stage + (it & 1) * 2 * rows * C;
            const int t0 = (it * p.split + peers.rank) * rows;
            stage_rows<T, CPL, ALIGN, S>(s, gate, p.gate_t, t0, rows, d0, p.T, p.D, __int_as_float(0x7f800000));
            stage_rows<T, CPL, ALIGN, S>(s + rows * C, x, p.x_t, t0, rows, d0, p.T, p.D, 0.f);
        }
        cp_commit();
    };
    issue(0);
    issue(1);
    float carry[CPL];                                     // the state before the cluster's next piece
    read_state<CPL>(p.h0 ? p.h0 + at_state : nullptr, carry, left);
    if (p.split > 1) peers.begin();
    for (int it = 0; it < n; ++it) {
        const int t0 = (it * p.split + peers.rank) * rows + warp * S;
        const T* sg = stage + (it & 1) * 2 * rows * C + warp * S * C + lane * CPL;
        cp_wait<1>();
        __syncthreads();
        float2 h[N], a[N];
        float H[CPL], A[CPL], in[CPL];
        run_forward<T, CPL, N>(sg, sg + rows * C, h, a, A, H);
        write_map<CPL>(map + (warp * C + lane * CPL) * 2, A, H);
        __syncthreads();
        issue(it + 2);                                    // every warp has read this stage
        join_forward<CPL>(map + lane * CPL * 2, next + lane * CPL, it, W, warp, lane, A, H, in, carry, peers);
        if (p.states && t0 < p.T && t0 % kSaved == 0)
            write_state<CPL>(p.states + ((long long)b * p.chunks + t0 / kSaved) * p.D + d, in, left);
        T* to = y + (long long)t0 * p.D;
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = fma2(a[i], both<CPL>(in), h[i]);
        if (p.T - t0 >= S) {
#pragma unroll
            for (int i = 0; i < N; ++i) write_pair<T, CPL, (ALIGN >= 4)>(to, p.D, i, h[i], S, left);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) write_pair<T, CPL, (ALIGN >= 4)>(to, p.D, i, h[i], p.T - t0, left);
        }
    }
    if (warp == W - 1 && peers.rank == 0) write_state<CPL>(p.last + at_state, carry, left);
    if (p.split > 1) cluster_sync();                      // no block ends while a peer may still write to it
}

template <class T, int CPL, int S, int ALIGN>
__global__ void __launch_bounds__(512, 1) rec_bwd(const RecArgs p) {
    constexpr int C = 32 * CPL, N = S * CPL / 2;
    extern __shared__ __align__(128) unsigned char smem[];
    const int W = blockDim.x >> 5, warp = warp_index(), lane = threadIdx.x & 31, rows = W * S;
    T* stage = reinterpret_cast<T*>(smem);
    float* base = reinterpret_cast<float*>(smem + 6 * (size_t)rows * C * sizeof(T));
    const Maps3<CPL> maps{base + lane * CPL, W};
    float* next = base + 3 * W * C;
    Peers<CPL> peers(next + 2 * C, p.split, blockIdx.x % p.split);
    const int group = blockIdx.x / p.split, b = group / p.groups, d0 = (group - b * p.groups) * C, d = d0 + lane * CPL, left = p.D - d;
    const T* gate = static_cast<const T*>(p.gate) + b * p.gate_b;
    const T* x = static_cast<const T*>(p.x) + b * p.x_b;
    const T* dy = static_cast<const T*>(p.dy) + b * p.dy_b;
    T* dgate = static_cast<T*>(p.dgate) + (long long)b * p.T * p.D + d;
    T* dx = static_cast<T*>(p.dx) + (long long)b * p.T * p.D + d;
    const int n = (p.T + rows * p.split - 1) / (rows * p.split);
    const long long at_state = (long long)b * p.D + d;

    auto issue = [&](int k) {                              // the k-th piece from the end
        if (k < n) {
            T* s = stage + (k & 1) * 3 * rows * C;
            const int t0 = ((n - 1 - k) * p.split + peers.rank) * rows;
            stage_rows<T, CPL, ALIGN, S>(s, gate, p.gate_t, t0, rows, d0, p.T, p.D, __int_as_float(0x7f800000));
            stage_rows<T, CPL, ALIGN, S>(s + rows * C, x, p.x_t, t0, rows, d0, p.T, p.D, 0.f);
            stage_rows<T, CPL, ALIGN, S>(s + 2 * rows * C, dy, p.dy_t, t0, rows, d0, p.T, p.D, 0.f);
        }
        cp_commit();
    };
    issue(0);
    float carry[CPL];                                     // a e of the step after the cluster's next piece
    read_state<CPL>(p.dlast ? p.dlast + at_state : nullptr, carry, left);
    if (p.split > 1) peers.begin();
    for (int k = 0; k < n; ++k) {
        const int first = ((n - 1 - k) * p.split + peers.rank) * rows, t0 = first + warp * S;
        const T* sg = stage + (k & 1) * 3 * rows * C + warp * S * C + lane * CPL;
        const T *sx = sg + rows * C, *sd = sx + rows * C;
        // a block's piece begins where the forward pass saved a state
        float hb[CPL];
        read_state<CPL>(first < p.T ? p.states + ((long long)b * p.chunks + first / kSaved) * p.D + d : nullptr, hb, left);
        cp_wait<0>();
        __syncthreads();                                  // the stage is there, and the other one has been read
        issue(k + 1);
        float2 a[N], z[N], f[N];
        float A[CPL], H[CPL], E[CPL], e[CPL];
        run_backward<T, CPL, N>(sg, sx, sd, a, z, A, H, E);
        maps.write(warp, A, H, E);
        __syncthreads();
        send_backward<CPL>(maps, k, warp, lane, peers);
        factors_backward<T, CPL, N>(maps, warp, sx, a, z, hb, f);
        join_backward<CPL>(maps, next + lane * CPL, k, warp, lane, A, E, e, carry, peers);
        T *to_g = dgate + (long long)t0 * p.D, *to_x = dx + (long long)t0 * p.D;
        auto sweep = [&](int steps) {
            sweep_backward<T, CPL, N>(sd, a, z, f, e, [&](int i, float2 dg, float2 dv) {
                write_pair<T, CPL, (ALIGN >= 4)>(to_g, p.D, i, dg, steps, left);
                write_pair<T, CPL, (ALIGN >= 4)>(to_x, p.D, i, dv, steps, left);
            });
        };
        if (p.T - t0 >= S) sweep(S);
        else sweep(p.T - t0);
    }
    if (warp == 0 && peers.rank == 0) write_state<CPL>(p.dh0 + at_state, carry, left);
    if (p.split > 1) cluster_sync();
}

// ---- staging by TMA tiles ----------------------------------------------------------------------------------
struct RecTiles {
    CUtensorMap gate, x, dy, out0, out1;                  // [B][T][D], a box of a piece's steps and 32 lanes' channels
};
__device__ __forceinline__ void load_tile(void* to, const CUtensorMap* m, int d, int t, int b, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                     smem_u32(to)),
                 "l"(m), "r"(d), "r"(t), "r"(b), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void store_tile(const CUtensorMap* m, const void* from, int d, int t, int b) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(m), "r"(smem_u32(from)), "r"(d),
                 "r"(t), "r"(b)
                 : "memory");
}
constexpr unsigned long long kTileWaitNs = 2000000000ull;
// The computing warps give up on tiles and on peers once each and then go on with NaN, so a piece's results are late by
// both waits at most; the warp that stores them waits longer, or results that are NaN would not be stored at all.
constexpr unsigned long long kWrittenWaitNs = kTileWaitNs + kPeerWaitNs + 1000000000ull;
constexpr int kFwdStages = 3, kBwdStages = 2;

// The warp beside the W computing ones: loads pieces ahead, stores a piece's results when all warps have written them
// (`written`, an mbarrier for each stage: a warp may be pieces ahead of another one, so a barrier that only counts
// arrivals would take one piece's for another's) and loads the next piece into their place when the copy has read them.
template <int STAGES, class Load, class Store>
__device__ __forceinline__ void move_tiles(int n, int lane, unsigned long long* written, Load&& load, Store&& store) {
    if (lane == 0) {
        for (int k = 0; k < STAGES && k < n; ++k) load(k);
        int stage = 0, parity = 0;
        for (int k = 0; k < n; ++k) {
            if (!mbar_wait(written + stage, parity, kWrittenWaitNs)) break;   // the others find no more tiles and give up
            store(k);
            bulk_commit();
            if (k + STAGES < n) {
                bulk_wait_read<0>();
                load(k + STAGES);
            }
            if (++stage == STAGES) {
                stage = 0;
                parity ^= 1;
            }
        }
        bulk_wait<0>();
    }
    __syncwarp();
}
// a computing warp's side of it
__device__ __forceinline__ void results_written(unsigned long long* written, int lane) {
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(written);
}
__device__ __forceinline__ void computing_sync(int threads) { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); }
// a pair into the place of the input it was made of
template <class T, int CPL>
__device__ __forceinline__ void put_pair(T* at, int i, float2 v) {
    constexpr int C = 32 * CPL;
    if constexpr (CPL == 2) {
        const float2 w[1] = {v};
        *reinterpret_cast<Pack<T, 2>*>(at + i * C) = pack_pairs<T, 2>(w);
    } else {
        at[2 * i * C] = from_f32<T>(v.x);
        at[(2 * i + 1) * C] = from_f32<T>(v.y);
    }
}
// A tile brings zeros for steps from T on; a gate of +infinity makes them leave the state as it is.  Each warp sees to its own.
template <class T, int CPL, int S>
__device__ __forceinline__ void hold_beyond(T* sg, int steps) {
    constexpr int C = 32 * CPL;
    for (int s = steps < 0 ? 0 : steps; s < S; ++s)
#pragma unroll
        for (int c = 0; c < CPL; ++c) sg[s * C + c] = from_f32<T>(__int_as_float(0x7f800000));
}

// Bound by memory: 8 x 4096 steps of 2048 bf16 channels in 71 us, 5.7 TB/s (issue slots are next: two blocks of 9 warps to an
// SM).  Few channels, 65537 steps of 768 floats by clusters of 8: 106 to 111 us, 5.5 TB/s.
template <class T, int CPL, int S>
__global__ void __launch_bounds__(kWarpsFwd * 32 + 32, 2) rec_fwd_tiles(const RecArgs p, const __grid_constant__ RecTiles m) {
    constexpr int C = 32 * CPL, N = S * CPL / 2, W = kWarpsFwd, rows = W * S, TILE = rows * C;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = warp_index(), lane = threadIdx.x & 31;
    T* stage = reinterpret_cast<T*>(smem);                                    // [stages][gate, x][rows][C]
    float* maps = reinterpret_cast<float*>(stage + kFwdStages * 2 * TILE);    // [2][W][C]{A, H}
    float* next = maps + 4 * W * C;
    unsigned long long* full = reinterpret_cast<unsigned long long*>(next + 2 * C);
    Peers<CPL> peers(reinterpret_cast<float*>(full + 2 * kFwdStages), p.split, blockIdx.x % p.split);
    const int group = blockIdx.x / p.split, b = group / p.groups, d0 = (group - b * p.groups) * C, d = d0 + lane * CPL, left = p.D - d;
    const int n = (p.T + rows * p.split - 1) / (rows * p.split);
    unsigned long long* written = full + kFwdStages;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kFwdStages; ++s) {
            mbar_init(full + s, 1);
            mbar_init(written + s, W);
        }
        fence_mbar_init();
    }
    if (p.split > 1) peers.begin();
    else __syncthreads();
    if (warp == W) {
        move_tiles<kFwdStages>(
            n, lane, written,
            [&](int it) {
                const int k = it % kFwdStages, t0 = (it * p.split + peers.rank) * rows;
                mbar_expect_tx(full + k, 2 * TILE * sizeof(T));
                load_tile(stage + 2 * k * TILE, &m.gate, d0, t0, b, full + k);
                load_tile(stage + (2 * k + 1) * TILE, &m.x, d0, t0, b, full + k);
            },
            [&](int it) {
                const int t0 = (it * p.split + peers.rank) * rows;
                if (t0 < p.T) store_tile(&m.out0, stage + (2 * (it % kFwdStages) + 1) * TILE, d0, t0, b);
            });
    } else {
        const long long at_state = (long long)b * p.D + d;
        float carry[CPL];
        read_state<CPL>(p.h0 ? p.h0 + at_state : nullptr, carry, left);
        bool there = true;
        int k = 0, parity = 0;
        for (int it = 0; it < n; ++it) {
            const int t0 = (it * p.split + peers.rank) * rows + warp * S;
            T* sg = stage + 2 * k * TILE + warp * S * C + lane * CPL;
            T* sx = sg + TILE;
            float* map = maps + (it & 1) * 2 * W * C;
            if (there) there = mbar_wait(full + k, parity, kTileWaitNs);
            if (p.T - t0 < S) hold_beyond<T, CPL, S>(sg, p.T - t0);
            float2 h[N], a[N];
            float H[CPL], A[CPL], in[CPL];
            run_forward<T, CPL, N>(sg, sx, h, a, A, H);
            write_map<CPL>(map + (warp * C + lane * CPL) * 2, A, H);
            computing_sync(W * 32);
            join_forward<CPL>(map + lane * CPL * 2, next + lane * CPL, it, W, warp, lane, A, H, in, carry, peers);
            if (!there) in[0] = in[CPL - 1] = carry[0] = carry[CPL - 1] = __int_as_float(0x7fc00000);
            if (p.states && t0 < p.T && t0 % kSaved == 0)
                write_state<CPL>(p.states + ((long long)b * p.chunks + t0 / kSaved) * p.D + d, in, left);
#pragma unroll
            for (int i = 0; i < N; ++i) put_pair<T, CPL>(sx, i, fma2(a[i], both<CPL>(in), h[i]));
            results_written(written + k, lane);
            if (++k == kFwdStages) {
                k = 0;
                parity ^= 1;
            }
        }
        if (warp == W - 1 && peers.rank == 0) write_state<CPL>(p.last + at_state, carry, left);
        __syncwarp();
    }
    if (p.split > 1) cluster_sync();                      // no block ends while a peer may still write to it
}

// The backward pass needs all registers that 16 warps leave each other, so no warp is left to move tiles: the last warp to
// finish a piece stores it, and loads another one into its place when it has gone through the first half of the next.
// Bound by issue slots: 4 x 8192 steps of 1024 bf16 channels in 76 us, 4.4 TB/s.
template <class T, int CPL, int S>
__global__ void __launch_bounds__(kWarpsBwd * 32, 1) rec_bwd_tiles(const RecArgs p, const __grid_constant__ RecTiles m) {
    constexpr int C = 32 * CPL, N = S * CPL / 2, W = kWarpsBwd, rows = W * S, TILE = rows * C;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned finished;                                             // warps, over all pieces
    const int warp = warp_index(), lane = threadIdx.x & 31;
    T* stage = reinterpret_cast<T*>(smem);                                    // [stages][gate, x, dy][rows][C]
    float* base = reinterpret_cast<float*>(stage + kBwdStages * 3 * TILE);    // [2][A, H, E][W][C]
    float* next = base + 6 * W * C;
    unsigned long long* full = reinterpret_cast<unsigned long long*>(next + 2 * C);
    Peers<CPL> peers(reinterpret_cast<float*>(full + kBwdStages), p.split, blockIdx.x % p.split);
    const int group = blockIdx.x / p.split, b = group / p.groups, d0 = (group - b * p.groups) * C, d = d0 + lane * CPL, left = p.D - d;
    const int n = (p.T + rows * p.split - 1) / (rows * p.split);
    const long long at_state = (long long)b * p.D + d;
    auto first_of = [&](int k) { return ((n - 1 - k) * p.split + peers.rank) * rows; };      // the k-th piece from the end
    auto load = [&](int k) {
        T* s = stage + 3 * (k & 1) * TILE;
        const int t0 = first_of(k);
        mbar_expect_tx(full + (k & 1), 3 * TILE * sizeof(T));
        load_tile(s, &m.gate, d0, t0, b, full + (k & 1));
        load_tile(s + TILE, &m.x, d0, t0, b, full + (k & 1));
        load_tile(s + 2 * TILE, &m.dy, d0, t0, b, full + (k & 1));
    };
    if (threadIdx.x == 0) {
        finished = 0;
        for (int s = 0; s < kBwdStages; ++s) mbar_init(full + s, 1);
        fence_mbar_init();
    }
    if (p.split > 1) peers.begin();
    else __syncthreads();
    if (threadIdx.x == 0)
        for (int k = 0; k < kBwdStages && k < n; ++k) load(k);
    float carry[CPL];
    read_state<CPL>(p.dlast ? p.dlast + at_state : nullptr, carry, left);
    bool there = true, stored = false;                    // stored: this lane has stored the last piece
    for (int k = 0; k < n; ++k) {
        const int first = first_of(k), t0 = first + warp * S;
        T* sg = stage + 3 * (k & 1) * TILE + warp * S * C + lane * CPL;
        T *sx = sg + TILE, *sd = sx + TILE;
        const Maps3<CPL> maps{base + (k & 1) * 3 * W * C + lane * CPL, W};
        float hb[CPL];
        read_state<CPL>(first < p.T ? p.states + ((long long)b * p.chunks + first / kSaved) * p.D + d : nullptr, hb, left);
        if (there) there = mbar_wait(full + (k & 1), (k >> 1) & 1, kTileWaitNs);
        if (p.T - t0 < S) hold_beyond<T, CPL, S>(sg, p.T - t0);
        float2 a[N], z[N], f[N];
        float A[CPL], H[CPL], E[CPL], e[CPL];
        run_backward<T, CPL, N>(sg, sx, sd, a, z, A, H, E);
        maps.write(warp, A, H, E);
        __syncthreads();
        send_backward<CPL>(maps, k, warp, lane, peers);
        if (stored) {
            bulk_wait_read<0>();
            if (k + 1 < n) load(k + 1);
            stored = false;
        }
        __syncwarp();
        factors_backward<T, CPL, N>(maps, warp, sx, a, z, hb, f);
        join_backward<CPL>(maps, next + lane * CPL, k, warp, lane, A, E, e, carry, peers);
        if (!there) e[0] = e[CPL - 1] = carry[0] = carry[CPL - 1] = __int_as_float(0x7fc00000);
        sweep_backward<T, CPL, N>(sd, a, z, f, e, [&](int i, float2 dg, float2 dv) {
            put_pair<T, CPL>(sg, i, dg);
            put_pair<T, CPL>(sx, i, dv);
        });
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
            __threadfence_block();
            // the pieces' counts do not mix: a warp counts the next piece only behind a barrier that all have reached
            stored = atomicAdd(&finished, 1u) % W == W - 1;
            if (stored) {
                __threadfence_block();
                if (first < p.T) {
                    store_tile(&m.out0, stage + 3 * (k & 1) * TILE, d0, first, b);
                    store_tile(&m.out1, stage + (3 * (k & 1) + 1) * TILE, d0, first, b);
                }
                bulk_commit();
            }
        }
        __syncwarp();
    }
    if (stored) bulk_wait<0>();
    if (warp == 0 && peers.rank == 0) write_state<CPL>(p.dh0 + at_state, carry, left);
    __syncwarp();
    if (p.split > 1) cluster_sync();
}

// ---- host ------------------------------------------------------------------------------------------------
bool rec_shape_ok(int64_t B, int64_t T, int D) { return B > 0 && T > 0 && D > 0; }
constexpr long long kMax32 = (1LL << 31) - 1;

template <class... KArgs, class... Args>
int launch_cluster(void (*kern)(KArgs...), int grid, int block, size_t smem, int cluster, cudaStream_t s, Args&&... args) {
    if (cluster == 1) return launch_kernel(kern, grid, block, smem, s, false, args...);
    allow_dynamic_smem((const void*)kern, smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...) != cudaSuccess) {
        (void)cudaGetLastError();
        return HFUSE_ERR_LAUNCH;
    }
    return check_launch();
}

// the largest of 16, 4 and the element size that divides every row's begin and the number of channels
int rec_align(int es, int D, std::initializer_list<const void*> ptrs, std::initializer_list<long long> strides) {
    uintptr_t all = (uintptr_t)D * es;
    for (const void* q : ptrs) all |= reinterpret_cast<uintptr_t>(q);
    for (long long s : strides) all |= (uintptr_t)(s * es);
    return (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : es;
}

// ---- TMA tiles ----
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}
// [B][T][D] with a box of `rows` steps and C channels; false where the strides do not nest (a shared gate, steps ahead of
// batch items in memory), which the other kernel takes
template <class T>
bool make_tiles(CUtensorMap& m, const void* at, long long stride_b, long long stride_t, const RecArgs& a, int rows, int C) {
    constexpr CUtensorMapDataType type = std::is_same_v<T, float>    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (a.B == 1) stride_b = a.T * stride_t;
    if (stride_t < a.D || stride_b / a.T < stride_t || stride_b * (long long)sizeof(T) >= 1LL << 40) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.T, (cuuint64_t)a.B};
    const cuuint64_t strides[2] = {(cuuint64_t)stride_t * sizeof(T), (cuuint64_t)stride_b * sizeof(T)};
    const cuuint32_t box[3] = {(cuuint32_t)C, (cuuint32_t)rows, 1}, step[3] = {1, 1, 1};
    return encode_tiled()(&m, type, 3, const_cast<void*>(at), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// From here on TMA tiles.  Times in a replayed graph, with tiles and by cp.async; the host needs about 1 us more for the maps.
// Forward they differ little: 8 x 512 steps of 2048 bf16 12.2 and 12.0 us, 768 15.5 and 16.2, 1024 19.3 and 20.6.  The gradient in
// 16 bits gains: 512 steps 24.0 and 26.0 us, 1024 40 and 51 (already 320 steps 20.6 and 23.0; 128 steps 13.0 and 7.6, since
// its tile is 256 steps).  In floats it loses up to here, and a little beyond: 8 x 384 steps of 1024 17.2 and 15.8, 1024 35.2 and 32.9.
constexpr int kTileSteps = 512;

template <class T, int CPL, int ALIGN, bool BWD>
int rec_launch(RecArgs a, cudaStream_t s) {
    constexpr int S = kSteps, MAXW = BWD ? kWarpsBwd : kWarpsFwd;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    const int C = 32 * CPL, W = a.T >= MAXW * S ? MAXW : (a.T + S - 1) / S;
    a.groups = (a.D + C - 1) / C;
    const long long groups = (long long)a.B * a.groups;
    const int pieces = (a.T + W * S - 1) / (W * S);
    // blocks that share a group: a power of two that the GPU has room for all at once and that all get work; a
    // sequence of several pieces has MAXW >= kMaxCluster warps in a block
    const long long room = (long long)f.sms * (BWD ? 1 : 2);
    int split = 1;
    while (2 * split <= kMaxCluster && 2 * split <= pieces && groups * 2 * split <= room) split *= 2;
    a.split = split;
    if (groups * split > kMax32) return HFUSE_ERR_TOO_LARGE;
    const size_t peers = split > 1 ? 2 * (size_t)kMaxCluster * C * 8 + 16 : 0;
    if constexpr (ALIGN == 16) {
        RecTiles m;
        const long long all = (long long)a.T * a.D;
        constexpr int rows = MAXW * S;
        bool ok = a.T >= kTileSteps && encode_tiled() && make_tiles<T>(m.gate, a.gate, a.gate_b, a.gate_t, a, rows, C) &&
                  make_tiles<T>(m.x, a.x, a.x_b, a.x_t, a, rows, C) && make_tiles<T>(m.out0, BWD ? a.dgate : a.y, all, a.D, a, rows, C);
        if (BWD)
            ok = ok && make_tiles<T>(m.dy, a.dy, a.dy_b, a.dy_t, a, rows, C) && make_tiles<T>(m.out1, a.dx, all, a.D, a, rows, C);
        else if (ok)
            m.dy = m.out1 = m.out0;
        if (ok) {
            const size_t smem = (size_t)(BWD ? kBwdStages * 3 : kFwdStages * 2) * rows * C * sizeof(T) + (BWD ? 6 : 4) * (size_t)MAXW * C * 4 +
                                2 * (size_t)C * 4 + (BWD ? kBwdStages * 8 : kFwdStages * 16) + peers;
            if constexpr (BWD) return launch_cluster(rec_bwd_tiles<T, CPL, S>, (int)(groups * split), MAXW * 32, smem, split, s, a, m);
            else return launch_cluster(rec_fwd_tiles<T, CPL, S>, (int)(groups * split), MAXW * 32 + 32, smem, split, s, a, m);
        }
    }
    const size_t smem = (size_t)(BWD ? 6 : 4) * W * S * C * sizeof(T) + (BWD ? 3 : 2) * (size_t)W * C * 4 + 2 * (size_t)C * 4 + peers;
    if constexpr (BWD) return launch_cluster(rec_bwd<T, CPL, S, ALIGN>, (int)(groups * split), W * 32, smem, split, s, a);
    else return launch_cluster(rec_fwd<T, CPL, S, ALIGN>, (int)(groups * split), W * 32, smem, split, s, a);
}

template <bool BWD>
int rec_dispatch(const RecArgs& a, int dtype, int align, cudaStream_t s) {
    return by_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        if constexpr (sizeof(T) == 4) {
            return align == 16 ? rec_launch<T, 1, 16, BWD>(a, s) : rec_launch<T, 1, 4, BWD>(a, s);
        } else {
            if (align == 16) return rec_launch<T, 2, 16, BWD>(a, s);
            if (align == 4) return rec_launch<T, 2, 4, BWD>(a, s);
            return rec_launch<T, 2, 2, BWD>(a, s);
        }
    });
}

}  // namespace

extern "C" {

int64_t hfuse_gated_recurrence_chunks(int64_t T) { return T > 0 ? (T + kSaved - 1) / kSaved : 0; }

int hfuse_gated_recurrence(const void* gate, int64_t gate_stride_b, int64_t gate_stride_t, const void* x, int64_t x_stride_b,
                           int64_t x_stride_t, int64_t B, int64_t T, int D, int dtype, const float* h0, void* out, float* h_last,
                           float* states, hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || !rec_shape_ok(B, T, D) || !gate || !x || !out || !h_last) return HFUSE_ERR_BAD_ARG;
    if (gate_stride_b < 0 || gate_stride_t < 0 || x_stride_b < 0 || x_stride_t < 0) return HFUSE_ERR_BAD_ARG;
    if (B > kMax32 || T > kMax32 - 65536 || B * D > kMax32 || D > kMaxWidth) return HFUSE_ERR_TOO_LARGE;
    const int es = lm_type_size(dtype);
    if (!aligned_to(gate, es) || !aligned_to(x, es) || !aligned_to(out, es) || !aligned_to(h0, 4) || !aligned_to(h_last, 4) ||
        !aligned_to(states, 4))
        return HFUSE_ERR_ALIGNMENT;
    RecArgs a{};
    a.gate = gate; a.x = x; a.h0 = h0; a.y = out; a.last = h_last; a.states = states;
    a.gate_b = gate_stride_b; a.gate_t = gate_stride_t; a.x_b = x_stride_b; a.x_t = x_stride_t;
    a.B = (int)B; a.T = (int)T; a.D = D; a.chunks = (int)hfuse_gated_recurrence_chunks(T);
    const int align = rec_align(es, D, {gate, x, out}, {gate_stride_b, gate_stride_t, x_stride_b, x_stride_t});
    return rec_dispatch<false>(a, dtype, align, static_cast<cudaStream_t>(stream));
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
    if (B > kMax32 || T > kMax32 - 65536 || B * D > kMax32 || D > kMaxWidth) return HFUSE_ERR_TOO_LARGE;
    const int es = lm_type_size(dtype);
    if (!aligned_to(gate, es) || !aligned_to(x, es) || !aligned_to(grad_out, es) || !aligned_to(grad_gate, es) ||
        !aligned_to(grad_x, es) || !aligned_to(states, 4) || !aligned_to(grad_h_last, 4) || !aligned_to(grad_h0, 4))
        return HFUSE_ERR_ALIGNMENT;
    RecArgs a{};
    a.gate = gate; a.x = x; a.dy = grad_out; a.dlast = grad_h_last; a.states = const_cast<float*>(states);
    a.dgate = grad_gate; a.dx = grad_x; a.dh0 = grad_h0;
    a.gate_b = gate_stride_b; a.gate_t = gate_stride_t; a.x_b = x_stride_b; a.x_t = x_stride_t;
    a.dy_b = grad_out_stride_b; a.dy_t = grad_out_stride_t;
    a.B = (int)B; a.T = (int)T; a.D = D; a.chunks = (int)hfuse_gated_recurrence_chunks(T);
    const int align = rec_align(es, D, {gate, x, grad_out, grad_gate, grad_x},
                                {gate_stride_b, gate_stride_t, x_stride_b, x_stride_t, grad_out_stride_b, grad_out_stride_t});
    return rec_dispatch<true>(a, dtype, align, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
