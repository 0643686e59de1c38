// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward   out[i] = scale table[ids[i]]
//   backward  grad_table[v] = scale sum over the tokens i with ids[i] = v, in ascending i, of grad_out[i]
//
// An id outside [0, rows) gives a row of zeros and no gradient; a padding id gives no gradient.
//
// The tokens are sorted by id with a stable radix sort (digits of up to 9 bits, at most 4 passes), so that the order
// of every sum, and with it every bit of the result, is fixed.  The sorted list is cut into chunks of kChunk tokens;
// each chunk is summed by one thread per group of columns, whatever ids it holds, so a frequent token costs no more than
// rare ones.  A token's run inside one chunk goes straight to the table; the parts of a run that crosses
// chunks go to the workspace and are added in order.
#include "launch.cuh"
#include "lm_common.cuh"

using namespace hfuse;

namespace {

constexpr int kChunk = 32;
constexpr int kTile = 2048;          // tokens a block ranks at a time
constexpr int kMaxTiles = 128;
constexpr int kMaxBins = 512;

struct EmbFwdArgs {
    const void *table, *ids;
    void* out;
    long long n, rows, items;
    int D, packs;
    float scale;
    FastDiv div;
};

template <class T, int EV, class I>
__global__ void __launch_bounds__(256) emb_fwd(const EmbFwdArgs a) {
    const T* table = static_cast<const T*>(a.table);
    T* out = static_cast<T*>(a.out);
    for (long long it = (long long)blockIdx.x * blockDim.x + threadIdx.x; it < a.items; it += (long long)gridDim.x * blockDim.x) {
        const long long i = it / a.packs;
        const int p = (int)(it - i * a.packs);
        const long long v = static_cast<const I*>(a.ids)[i];
        Pack<T, EV> r;
        if (v >= 0 && v < a.rows) {
            const Pack<T, EV> q = load_cached<T, EV>(table + v * a.D + p * EV);
            float2 f[(EV + 1) / 2];
#pragma unroll
            for (int k = 0; k < (EV + 1) / 2; ++k) f[k] = mul2(pair_of(q, k), make_float2(a.scale, a.scale));
            r = pack_pairs<T, EV>(f);
        } else {
            r = {};
        }
        store_stream<T, EV>(out + i * a.D + p * EV, r);
    }
}

// ---- sort ------------------------------------------------------------------------------------------
struct SortArgs {
    const void* ids;            // first pass only
    const unsigned *key, *pos;  // later passes
    unsigned *key_out, *pos_out;
    unsigned* count;            // [tiles][bins] of this pass
    long long rows, padding;
    int n, tile, tiles, shift, bits;
};

// ids that get no gradient become the key `rows`, which sorts behind all others
template <class I>
__device__ __forceinline__ unsigned token_key(const SortArgs& a, int i) {
    const long long v = static_cast<const I*>(a.ids)[i];
    return v < 0 || v >= a.rows || v == a.padding ? (unsigned)a.rows : (unsigned)v;
}
struct NoIds {};
template <class I>
__device__ __forceinline__ unsigned sort_key(const SortArgs& a, int i) {
    if constexpr (sizeof(I) >= 4) return token_key<I>(a, i);
    else return a.key[i];
}

template <class I>
__global__ void __launch_bounds__(256) emb_sort_count(const SortArgs a) {
    __shared__ unsigned bin[kMaxBins];
    const int bins = 1 << a.bits;
    for (int d = threadIdx.x; d < bins; d += 256) bin[d] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * a.tile, i1 = min(a.n, i0 + a.tile);
    for (int i = i0 + threadIdx.x; i < i1; i += 256) atomicAdd(&bin[(sort_key<I>(a, i) >> a.shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += 256) a.count[(size_t)blockIdx.x * bins + d] = bin[d];
}

template <class I>
__global__ void __launch_bounds__(256) emb_sort_scatter(const SortArgs a) {
    constexpr int WARPS = 8, ROUNDS = kTile / 256;
    __shared__ unsigned base[kMaxBins];               // where the tile's next key with this digit goes
    __shared__ unsigned cnt[WARPS][kMaxBins];         // a warp's keys with this digit
    __shared__ unsigned wsum[WARPS];
    const int bins = 1 << a.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // keys with a smaller digit, and those with the same digit in earlier tiles: two neighbouring digits per thread
    unsigned total[2] = {0, 0}, before[2] = {0, 0};
    for (int k = 0; k < 2; ++k) {
        const int d = 2 * threadIdx.x + k;
        if (d < bins)
            for (int t = 0; t < a.tiles; ++t) {
                const unsigned c = a.count[(size_t)t * bins + d];
                total[k] += c;
                before[k] += t < (int)blockIdx.x ? c : 0;
            }
    }
    unsigned s = total[0] + total[1], incl = s;
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    unsigned off = incl - s;
    for (int w = 0; w < warp; ++w) off += wsum[w];
    if (2 * threadIdx.x < bins) base[2 * threadIdx.x] = off + before[0];
    if (2 * threadIdx.x + 1 < bins) base[2 * threadIdx.x + 1] = off + total[0] + before[1];

    const int i0 = blockIdx.x * a.tile, i1 = min(a.n, i0 + a.tile);
    for (int at = i0; at < i1; at += kTile) {
        for (int d = lane; d < bins; d += 32) cnt[warp][d] = 0;
        __syncwarp();
        // each warp ranks its own stretch, 32 keys at a time
        unsigned key[ROUNDS], rank[ROUNDS];
        int pos[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int i = at + warp * (32 * ROUNDS) + r * 32 + lane;
            const bool in = i < i1;
            key[r] = in ? sort_key<I>(a, i) : 0u;
            if constexpr (sizeof(I) >= 4) pos[r] = i;
            else pos[r] = in ? (int)a.pos[i] : 0;
            const unsigned d = (key[r] >> a.shift) & (bins - 1);
            const unsigned same = __match_any_sync(0xffffffffu, in ? d : 0xffffffffu);
            rank[r] = in ? cnt[warp][d] + __popc(same & ((1u << lane) - 1)) : 0u;
            __syncwarp();
            if (in && (same >> lane) == 1u) cnt[warp][d] += __popc(same);      // the highest lane of each digit
            __syncwarp();
        }
        __syncthreads();
        for (int d = threadIdx.x; d < bins; d += 256) {     // each warp's first place for each digit
            unsigned b = base[d];
            for (int w = 0; w < WARPS; ++w) {
                const unsigned c = cnt[w][d];
                cnt[w][d] = b;
                b += c;
            }
            base[d] = b;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int i = at + warp * (32 * ROUNDS) + r * 32 + lane;
            if (i < i1) {
                const unsigned to = cnt[warp][(key[r] >> a.shift) & (bins - 1)] + rank[r];
                a.key_out[to] = key[r];
                a.pos_out[to] = (unsigned)pos[r];
            }
        }
        __syncthreads();
    }
}

// ---- sums ----------------------------------------------------------------------------------------------
struct EmbSumArgs {
    const void* dy;
    const unsigned *key, *pos;
    void* grad;
    float* part;                 // [chunks][2][D]: end of a run begun in an earlier chunk, begin of a run that goes on
    long long items;
    unsigned rows;
    int n, D, packs, chunks;
    float scale;
};

template <class T, int EV>
__device__ __forceinline__ void write_row(const EmbSumArgs& a, unsigned v, int p, const float2 (&acc)[(EV + 1) / 2]) {
    float2 r[(EV + 1) / 2];
#pragma unroll
    for (int k = 0; k < (EV + 1) / 2; ++k) r[k] = mul2(acc[k], make_float2(a.scale, a.scale));
    store_stream<T, EV>(static_cast<T*>(a.grad) + (long long)v * a.D + p * EV, pack_pairs<T, EV>(r));
}

template <class T, int EV>
__global__ void __launch_bounds__(256) emb_sum(const EmbSumArgs a) {
    for (long long it = (long long)blockIdx.x * 256 + threadIdx.x; it < a.items; it += (long long)gridDim.x * 256) {
        const int c = (int)(it / a.packs), p = (int)(it - (long long)c * a.packs);
        const int s = c * kChunk, e = min(a.n, s + kChunk);
        unsigned cur = a.key[s];
        if (cur >= a.rows) continue;
        bool begun = s > 0 && a.key[s - 1] == cur;          // the run began in an earlier chunk
        float2 acc[(EV + 1) / 2];
        auto clear = [&] {
#pragma unroll
            for (int k = 0; k < (EV + 1) / 2; ++k) acc[k] = make_float2(0.f, 0.f);
        };
        auto keep = [&](float* to) {
#pragma unroll
            for (int k = 0; k < EV; ++k) to[k] = k & 1 ? acc[k / 2].y : acc[k / 2].x;
        };
        clear();
        float* part = a.part + 2LL * c * a.D + p * EV;
        for (int i = s; i < e; ++i) {
            const unsigned v = a.key[i];
            if (v != cur) {
                if (begun) keep(part);
                else write_row<T, EV>(a, cur, p, acc);
                cur = v;
                begun = false;
                if (v >= a.rows) break;
                clear();
            }
            const Pack<T, EV> g = load_stream<T, EV>(static_cast<const T*>(a.dy) + (long long)a.pos[i] * a.D + p * EV);
#pragma unroll
            for (int k = 0; k < (EV + 1) / 2; ++k) acc[k] = add2(acc[k], pair_of(g, k));
        }
        if (cur >= a.rows) continue;
        if (begun) keep(part);
        else if (e < a.n && a.key[e] == cur) keep(part + a.D);
        else write_row<T, EV>(a, cur, p, acc);
    }
}

// runs that cross chunks: the thread of the chunk in which the run begins adds its parts in order
template <class T>
__global__ void __launch_bounds__(256) emb_join(const EmbSumArgs a) {
    for (long long it = (long long)blockIdx.x * 256 + threadIdx.x; it < (long long)a.chunks * a.D; it += (long long)gridDim.x * 256) {
        const int c = (int)(it / a.D), p = (int)(it - (long long)c * a.D);
        const int s = c * kChunk, e = s + kChunk;
        if (e >= a.n) continue;
        const unsigned v = a.key[e];
        if (v >= a.rows || a.key[e - 1] != v) continue;                          // nothing crosses this chunk's end
        if (s > 0 && a.key[s] == v && a.key[s - 1] == v) continue;               // the run began earlier
        float2 acc[1] = {make_float2(a.part[(2LL * c + 1) * a.D + p], 0.f)};
        for (int k = c + 1; k < a.chunks && a.key[k * kChunk] == v; ++k) acc[0].x += a.part[2LL * k * a.D + p];
        write_row<T, 1>(a, v, p, acc);
    }
}

struct EmbPlan {
    int tile, tiles, passes, bits, chunks;
    size_t key[2], pos[2], count, part, bytes;
};
EmbPlan emb_plan(long long n, long long rows, int D) {
    EmbPlan p{};
    const long long per = (n + (long long)kMaxTiles * kTile - 1) / ((long long)kMaxTiles * kTile);
    p.tile = (int)(kTile * (per < 1 ? 1 : per));
    p.tiles = (int)((n + p.tile - 1) / p.tile);
    int bits = 0;
    while (bits < 32 && (rows >> bits) != 0) ++bits;          // keys are 0 .. rows
    p.passes = (bits + 8) / 9;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.chunks = (int)((n + kChunk - 1) / kChunk);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) & ~(size_t)255;
        return r;
    };
    for (int k = 0; k < 2; ++k) {
        p.key[k] = take((size_t)n * 4);
        p.pos[k] = take((size_t)n * 4);
    }
    p.count = take((size_t)p.tiles * kMaxBins * 4);
    p.part = take((size_t)p.chunks * 2 * (size_t)D * 4);
    p.bytes = at;
    return p;
}

constexpr long long kMaxTokens = (1LL << 31) - 1 - (long long)kMaxTiles * kTile;
constexpr long long kMaxRows = (1LL << 31) - 1;

}  // namespace

extern "C" {

int hfuse_embedding(const void* table, int64_t rows, int D, int dtype, const void* ids, int64_t n, int id_bytes, float scale,
                    void* out, hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || rows <= 0 || D <= 0 || n < 0 || (id_bytes != 4 && id_bytes != 8)) return HFUSE_ERR_BAD_ARG;
    if (rows > kMaxRows || n > kMaxTokens) return HFUSE_ERR_TOO_LARGE;
    if (n == 0) return HFUSE_OK;
    if (!table || !ids || !out) return HFUSE_ERR_BAD_ARG;
    const size_t es = lm_type_size(dtype);
    if (!aligned_to(table, es) || !aligned_to(out, es) || !aligned_to(ids, id_bytes)) return HFUSE_ERR_ALIGNMENT;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    EmbFwdArgs a{};
    a.table = table; a.ids = ids; a.out = out;
    a.n = n; a.rows = rows; a.D = D; a.scale = scale;
    const bool wide = aligned_to(table, 16) && aligned_to(out, 16) && D * es % 16 == 0;
    return by_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        constexpr int EV = 16 / sizeof(T);
        a.packs = wide ? D / EV : D;
        a.items = (long long)n * a.packs;
        const long long want = (a.items + 255) / 256, most = f.sms * 8LL;
        const int grid = (int)(want < most ? want : most);
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (wide)
            return id_bytes == 8 ? launch_kernel(emb_fwd<T, EV, long long>, grid, 256, 0, s, false, a)
                                 : launch_kernel(emb_fwd<T, EV, int>, grid, 256, 0, s, false, a);
        return id_bytes == 8 ? launch_kernel(emb_fwd<T, 1, long long>, grid, 256, 0, s, false, a)
                             : launch_kernel(emb_fwd<T, 1, int>, grid, 256, 0, s, false, a);
    });
}

size_t hfuse_embedding_backward_workspace_bytes(int64_t n, int64_t rows, int D) {
    if (n <= 0 || rows <= 0 || D <= 0 || n > kMaxTokens || rows > kMaxRows) return 0;
    return emb_plan(n, rows, D).bytes;
}

int hfuse_embedding_backward(const void* grad_out, const void* ids, int64_t n, int id_bytes, int64_t rows, int D, int dtype,
                             float scale, int64_t padding_id, void* grad_table, void* workspace, size_t workspace_bytes,
                             hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || rows <= 0 || D <= 0 || n < 0 || (id_bytes != 4 && id_bytes != 8)) return HFUSE_ERR_BAD_ARG;
    if (rows > kMaxRows || n > kMaxTokens) return HFUSE_ERR_TOO_LARGE;
    if (!grad_table || (n > 0 && (!grad_out || !ids))) return HFUSE_ERR_BAD_ARG;
    const size_t es = lm_type_size(dtype);
    if (!aligned_to(grad_out, es) || !aligned_to(grad_table, es) || (n > 0 && !aligned_to(ids, id_bytes)) || !aligned_to(workspace, 16))
        return HFUSE_ERR_ALIGNMENT;
    const EmbPlan p = n > 0 ? emb_plan(n, rows, D) : EmbPlan{};
    if (n > 0 && (!workspace || workspace_bytes < p.bytes)) return HFUSE_ERR_WORKSPACE;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cudaMemsetAsync(grad_table, 0, (size_t)rows * D * es, s) != cudaSuccess) {
        (void)cudaGetLastError();
        return HFUSE_ERR_LAUNCH;
    }
    if (n == 0) return HFUSE_OK;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    auto at = [&](size_t off) { return reinterpret_cast<unsigned*>(ws + off); };
    SortArgs a{};
    a.ids = ids; a.rows = rows; a.padding = padding_id;
    a.n = (int)n; a.tile = p.tile; a.tiles = p.tiles; a.bits = p.bits; a.count = at(p.count);
    for (int k = 0; k < p.passes; ++k) {
        a.shift = k * p.bits;
        a.key = at(p.key[(k + 1) & 1]); a.pos = at(p.pos[(k + 1) & 1]);
        a.key_out = at(p.key[k & 1]); a.pos_out = at(p.pos[k & 1]);
        int rc;
        if (k > 0) {
            rc = launch_kernel(emb_sort_count<NoIds>, p.tiles, 256, 0, s, false, a);
            if (!rc) rc = launch_kernel(emb_sort_scatter<NoIds>, p.tiles, 256, 0, s, false, a);
        } else if (id_bytes == 8) {
            rc = launch_kernel(emb_sort_count<long long>, p.tiles, 256, 0, s, false, a);
            if (!rc) rc = launch_kernel(emb_sort_scatter<long long>, p.tiles, 256, 0, s, false, a);
        } else {
            rc = launch_kernel(emb_sort_count<int>, p.tiles, 256, 0, s, false, a);
            if (!rc) rc = launch_kernel(emb_sort_scatter<int>, p.tiles, 256, 0, s, false, a);
        }
        if (rc) return rc;
    }
    const int last = (p.passes - 1) & 1;
    EmbSumArgs b{};
    b.dy = grad_out; b.key = at(p.key[last]); b.pos = at(p.pos[last]); b.grad = grad_table;
    b.part = reinterpret_cast<float*>(ws + p.part);
    b.rows = (unsigned)rows; b.n = (int)n; b.D = D; b.chunks = p.chunks; b.scale = scale;
    const bool wide = aligned_to(grad_out, 16) && aligned_to(grad_table, 16) && D * es % 16 == 0;
    return by_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        constexpr int EV = 16 / sizeof(T);
        b.packs = wide ? D / EV : D;
        b.items = (long long)p.chunks * b.packs;
        const long long want = (b.items + 255) / 256, most = f.sms * 8LL;
        const int grid = (int)(want < most ? want : most);
        if (int rc = wide ? launch_kernel(emb_sum<T, EV>, grid, 256, 0, s, false, b) : launch_kernel(emb_sum<T, 1>, grid, 256, 0, s, false, b))
            return rc;
        const long long wantj = ((long long)p.chunks * D + 255) / 256;
        return launch_kernel(emb_join<T>, (int)(wantj < most ? wantj : most), 256, 0, s, false, b);
    });
}

}  // extern "C"
