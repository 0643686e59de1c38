// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward   out[i] = scale table[ids[i]]
//   backward  grad_table[v] = scale sum over the tokens i with ids[i] = v, in ascending i, of grad_out[i]
//
// An id outside [0, rows) gives a row of zeros and no gradient; a padding id gives no gradient.
//
// Memory-bound: the forward pass reads each row it needs and writes it; the backward pass reads grad_out once and
// writes every row of grad_table once.  The tokens are sorted by id with a stable radix sort (digits of up to 9 bits, at
// most 4 passes), so that the order of every sum, and with it every bit of the result, is fixed.  The sorted list is cut
// into chunks of 16 to 64 tokens; each chunk is summed by one thread per group of columns, whatever ids it holds, so a frequent
// token costs no more than rare ones.  A token's run inside one chunk goes straight to the table; the parts of a run that
// crosses chunks go to the workspace, and a last kernel adds them in order.
//
// Up to 256 tokens take one kernel: a block for each token that is the first with its id, which finds the others and
// adds them up, and blocks that write the rows that no token meets (a call of 8 tokens: 6.3 us of the host's time instead
// of 11.1 with the three kernels of a small sort).
// The kernels of a call with more tokens, each the programmatic dependent of the one before (its launch overlaps the other's end):
//   up to 8192 tokens and 262144 rows
//     sort_small  some warps of each block count, for a few tokens, how many come before them, while the others
//                 write the rows of the block's share that no token meets
//   otherwise
//     clear       the bitmap of the rows that are met and the counters
//     count       digit counts of each tile of tokens for the first pass; marks the rows that are met
//     scatter     one per pass: places the tile's tokens and counts the next pass's digits; blocks beside the sorting ones
//                 write rows that are not met until the tiles are done
//   sum           chunks, and the other rows that are not met
//   join          runs that cross chunks
// Rows that no token meets are often the larger part of all bytes, and sorting leaves the memory idle most of the time.
#include "launch.cuh"
#include "lm_common.cuh"

using namespace hfuse;

namespace {

// Tokens that a thread sums: few tokens need many threads, many tokens leave fewer parts to join with long chunks.  With 32 and
// with 64, into 32000 rows, in a replayed graph: 8193 tokens of 512 bf16 35 and 40 us, 32768 46 and 50, 40960 52 and 51,
// 65536 54 and 51; of 2048 bf16 8193 tokens 50 and 54, 32768 82 and 78, 65536 114 and 113, 131072 190 and 171.
constexpr int kChunk = 32, kSmallChunk = 16, kWideChunk = 64;
constexpr int kTile = 2048;          // tokens a block ranks at a time
constexpr int kMaxTiles = 128;
constexpr int kMaxBins = 512;
constexpr int kMaxPasses = 4;
constexpr int kSortThreads = 512;
constexpr int kSmallTokens = 8192;   // 13 bits beside the 19 of a key
constexpr long long kSmallRows = 262144;
constexpr int kRankWarps = 8;        // of 32 in the small sort; the others write zeros
constexpr int kLongRun = 33;         // parts from which a block, not a warp, adds them up

// counters in the workspace, set to zero by the first kernel of a call
struct Counters {
    unsigned short_runs, long_runs;      // runs that cross chunks
    unsigned zero_next;                  // batches of rows that sorting kernels have taken to write zeros into
    unsigned sorted[kMaxPasses];         // tiles that are done
};

__device__ __forceinline__ void after_predecessor() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

struct EmbFwdArgs {
    const void *table, *ids;
    void* out;
    long long n, rows;
    int D, packs, lanes;
    float scale;
};

// `lanes` threads to a token, kAhead accesses each, the block's second index over longer rows: all loads of a thread are
// under way together.  16384 tokens of 2048 floats from 50257 rows: 33 us, 5.5 TB/s; bound by memory.
constexpr int kAhead = 4;
template <class T, int EV, class I>
__global__ void __launch_bounds__(256) emb_fwd(const EmbFwdArgs a) {
    const int lanes = a.lanes, at = threadIdx.x & (lanes - 1);
    const long long i = (long long)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    if (i >= a.n) return;
    const long long v = __ldg(static_cast<const I*>(a.ids) + i);
    const bool in = v >= 0 && v < a.rows;
    const T* row = static_cast<const T*>(a.table) + (in ? v : 0) * a.D;
    T* out = static_cast<T*>(a.out) + i * a.D;
    for (int p0 = blockIdx.y * lanes * kAhead + at; p0 < a.packs; p0 += gridDim.y * lanes * kAhead) {
        Pack<T, EV> q[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            q[k] = {};
            if (in && p0 + k * lanes < a.packs) q[k] = load_cached<T, EV>(row + (p0 + k * lanes) * (long long)EV);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (p0 + k * lanes >= a.packs) continue;
            float2 f[(EV + 1) / 2];
#pragma unroll
            for (int j = 0; j < (EV + 1) / 2; ++j) f[j] = in ? mul2(pair_of(q[k], j), make_float2(a.scale, a.scale)) : make_float2(0.f, 0.f);
            store_stream<T, EV>(out + (p0 + k * lanes) * (long long)EV, pack_pairs<T, EV>(f));
        }
    }
}

// Rows of 16-bit elements that begin anywhere: what is written are whole accesses of the output's row, and up to 14 elements
// around them.  Such an access's elements lie in two neighbouring ones of the table's row, from which they are shifted together;
// the second of them is the next lane's first, so it comes from L1.  16384 tokens of 2047 bf16 take 29 us (of 2048: 20), as
// single elements 56; floats (1023 of them) 33 with it and 31 as single elements, so they stay that.
template <class T, class I>
__global__ void __launch_bounds__(256) emb_fwd_shifted(const EmbFwdArgs a) {
    constexpr int EV = 16 / sizeof(T);
    static_assert(EV == 8);
    const int lanes = a.lanes, at = threadIdx.x & (lanes - 1);
    const long long i = (long long)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    if (i >= a.n) return;
    const long long v = __ldg(static_cast<const I*>(a.ids) + i);
    const bool in = v >= 0 && v < a.rows;
    const T* row = static_cast<const T*>(a.table) + (in ? v : 0) * a.D;
    T* out = static_cast<T*>(a.out) + i * a.D;
    const int lead = (int)(-(reinterpret_cast<uintptr_t>(out) / sizeof(T)) & (EV - 1)), packs = (a.D - lead) / EV, edges = a.D - packs * EV;
    if (blockIdx.y == 0)
        for (int e = at; e < edges; e += lanes) {
            const int c = e < lead ? e : e + packs * EV;
            out[c] = from_f32<T>(in ? to_f32(row[c]) * a.scale : 0.f);
        }
    // the accesses of the table that hold the first elements, and how far into them they begin
    const int bytes = (int)(reinterpret_cast<uintptr_t>(row + lead) & 15), words = bytes >> 2, bits = (bytes & 3) * 8;
    const unsigned char* from = reinterpret_cast<const unsigned char*>(row + lead) - bytes;
    const unsigned char* const begin = static_cast<const unsigned char*>(a.table);
    const unsigned char* const end = begin + (size_t)a.rows * a.D * sizeof(T);
    for (int p0 = blockIdx.y * lanes * kAhead + at; p0 < packs; p0 += gridDim.y * lanes * kAhead) {
        unsigned w[kAhead][8];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int p = p0 + k * lanes;
            const unsigned char* q = from + 16LL * p;
#pragma unroll
            for (int j = 0; j < 8; ++j) w[k][j] = 0;
            if (!in || p >= packs) continue;
            if (q >= begin && q + 32 <= end) {
                const Pack<T, EV> lo = load_cached<T, EV>(reinterpret_cast<const T*>(q)), hi = load_cached<T, EV>(reinterpret_cast<const T*>(q + 16));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[k][j] = lo.w[j];
                    w[k][j + 4] = hi.w[j];
                }
            } else {                                       // the table's first and last elements
                const T* one = row + lead + p * EV;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // word j of the two accesses, as far as it is the row's
                    const unsigned short* h = reinterpret_cast<const unsigned short*>(one);
                    const int lo = (4 * j - bytes) / 2, hi = lo + 1;
                    if (4 * j >= bytes && lo < EV) w[k][j] = h[lo];
                    if (4 * j + 2 >= bytes && hi < EV) w[k][j] |= (unsigned)h[hi] << 16;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int p = p0 + k * lanes;
            if (p >= packs) continue;
            unsigned t[6], u[5];
#pragma unroll
            for (int j = 0; j < 6; ++j) t[j] = words & 2 ? w[k][j + 2] : w[k][j];
#pragma unroll
            for (int j = 0; j < 5; ++j) u[j] = words & 1 ? t[j + 1] : t[j];
            Pack<T, EV> q;
#pragma unroll
            for (int j = 0; j < 4; ++j) q.w[j] = __funnelshift_r(u[j], u[j + 1], bits);
            float2 f[EV / 2];
#pragma unroll
            for (int j = 0; j < EV / 2; ++j) f[j] = in ? mul2(pair_of(q, j), make_float2(a.scale, a.scale)) : make_float2(0.f, 0.f);
            store_stream<T, EV>(out + lead + p * EV, pack_pairs<T, EV>(f));
        }
    }
}

// ---- rows of the table that no token meets ---------------------------------------------------------------
struct ZeroArgs {
    unsigned char* grad;
    const unsigned* met;         // a bit for each row
    long long row_bytes, rows, batches;
    int per_warp;                // rows of a warp, a power of two up to 32
};
// zeros for the rows r0 + k of which bit k of `todo` is set
__device__ __forceinline__ void zero_marked(const ZeroArgs& z, long long r0, unsigned todo) {
    const int lane = threadIdx.x & 31;
    while (todo) {
        // neighbouring rows are written as one stretch
        const int k = __ffs(todo) - 1, run = __ffs(~(todo >> k)) - 1;
        const int count = run < 0 ? 32 - k : run;
        todo = k + count >= 32 ? 0 : todo & (~0u << (k + count));
        unsigned char* p = z.grad + (r0 + k) * z.row_bytes;
        unsigned char* const end = p + count * z.row_bytes;
        unsigned char* const a0 = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p) + 15) & ~(uintptr_t)15);
        unsigned char* const a1 = reinterpret_cast<unsigned char*>(reinterpret_cast<uintptr_t>(end) & ~(uintptr_t)15);
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        if (a0 >= a1) {
            for (unsigned char* q = p + 2 * lane; q < end; q += 64) *reinterpret_cast<unsigned short*>(q) = 0;
        } else {
            if (p + 2 * lane < a0) *reinterpret_cast<unsigned short*>(p + 2 * lane) = 0;
#pragma unroll 4
            for (unsigned char* q = a0 + 16 * lane; q < a1; q += 512) stg_stream4(reinterpret_cast<float*>(q), zero);
            if (a1 + 2 * lane < end) *reinterpret_cast<unsigned short*>(a1 + 2 * lane) = 0;
        }
    }
}
// the rows of a batch, 8 * per_warp of them (a block of 16 warps does two batches)
__device__ __forceinline__ void zero_batch(const ZeroArgs& z, long long batch) {
    const long long r0 = (batch * 8 + (threadIdx.x >> 5)) * z.per_warp;
    if (r0 >= z.rows) return;
    unsigned todo = ~(z.met[r0 >> 5] >> (r0 & 31));
    const int here = (int)min((long long)z.per_warp, z.rows - r0);
    if (here < 32) todo &= (1u << here) - 1;
    zero_marked(z, r0, todo);
}

// ---- sort ------------------------------------------------------------------------------------------
struct SortArgs {
    const void* ids;            // first pass and small sort
    const unsigned *key, *pos;  // later passes
    unsigned *key_out, *pos_out;
    unsigned *count, *next;     // [tiles][bins] of this pass and of the next one (or null)
    unsigned* met;
    Counters* counters;
    unsigned* clear;            // clear kernel: 4-byte words
    long long clear_words;
    long long rows, padding;
    int n, tile, tiles, shift, bits, pass, passes;
    ZeroArgs zero;
};

// ids that get no gradient become the key `rows`, which sorts behind all others
template <class I>
__device__ __forceinline__ unsigned token_key(const SortArgs& a, int i) {
    const long long v = __ldg(static_cast<const I*>(a.ids) + i);
    return v < 0 || v >= a.rows || v == a.padding ? (unsigned)a.rows : (unsigned)v;
}
struct NoIds {};
template <class I>
__device__ __forceinline__ unsigned sort_key(const SortArgs& a, int i) {
    if constexpr (sizeof(I) >= 4) return token_key<I>(a, i);
    else return a.key[i];
}

__global__ void __launch_bounds__(256) emb_clear(const SortArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.clear_words; i += (long long)gridDim.x * 256) a.clear[i] = 0;
}

template <class I>
__global__ void __launch_bounds__(kSortThreads) emb_sort_count(const SortArgs a) {
    __shared__ unsigned bin[kMaxBins];
    __shared__ unsigned seen[1024];                   // ids that the block has marked, one to a slot: frequent ones are marked once
    const int bins = 1 << a.bits;
    for (int d = threadIdx.x; d < bins; d += kSortThreads) bin[d] = 0;
    for (int d = threadIdx.x; d < 1024; d += kSortThreads) seen[d] = 0xffffffffu;
    __syncthreads();
    after_predecessor();
    const int i0 = blockIdx.x * a.tile, i1 = min(a.n, i0 + a.tile);
#pragma unroll 4
    for (int i = i0 + threadIdx.x; i < i1; i += kSortThreads) {
        const unsigned k = token_key<I>(a, i);
        atomicAdd(&bin[k & (bins - 1)], 1u);
        if (k < (unsigned)a.rows && *reinterpret_cast<volatile unsigned*>(&seen[k & 1023]) != k) {
            *reinterpret_cast<volatile unsigned*>(&seen[k & 1023]) = k;
            atomicOr(a.met + (k >> 5), 1u << (k & 31));
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) a.count[(size_t)blockIdx.x * bins + d] = bin[d];
}

// Ranks of a warp's keys among those with the same digit, 32 keys at a time in their order; cnt: the warp's counts so far.
// The lanes with the same digit are found with a vote for each of its bits: matching whole words at once
// (__match_any_sync) took four times as long.
template <class C>
__device__ __forceinline__ unsigned rank_digit(C* cnt, unsigned d, int bits, bool in, int lane) {
    unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
    for (int b = 0; b < 9; ++b)
        if (b < bits) {
            const bool set = d >> b & 1u;
            const unsigned votes = __ballot_sync(0xffffffffu, set);
            same &= set ? votes : ~votes;
        }
    const unsigned rank = in ? cnt[d] + __popc(same & ((1u << lane) - 1)) : 0u;
    __syncwarp();
    if (in && (same >> lane) == 1u) cnt[d] += (C)__popc(same);         // the highest lane of each digit
    __syncwarp();
    return rank;
}

template <class I>
__global__ void __launch_bounds__(kSortThreads) emb_sort_scatter(const SortArgs a) {
    constexpr int WARPS = kSortThreads / 32, ROUNDS = kTile / kSortThreads;
    __shared__ unsigned base[kMaxBins];               // where the tile's next key with this digit goes
    __shared__ unsigned sums[2][2][kMaxBins];         // two halves of the tiles: all keys with a digit, and those before this tile
    __shared__ unsigned short cnt[WARPS][kMaxBins];   // a warp's keys with this digit
    __shared__ unsigned wsum[WARPS];
    __shared__ unsigned batch;
    after_predecessor();
    if ((int)blockIdx.x >= a.tiles) {
        // nothing waits here: batches are taken until there are none, or the tiles are done
        for (;;) {
            __syncthreads();
            if (threadIdx.x == 0) {
                const unsigned done = *reinterpret_cast<volatile unsigned*>(&a.counters->sorted[a.pass]);
                batch = done == (unsigned)a.tiles ? 0xffffffffu : atomicAdd(&a.counters->zero_next, 2u);
            }
            __syncthreads();
            if (batch >= a.zero.batches) return;
            zero_batch(a.zero, batch);
        }
    }
    const int bins = 1 << a.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // keys with a smaller digit, and those with the same digit in earlier tiles: two neighbouring digits and every
    // second tile to a thread
    {
        const int pair = threadIdx.x & 255, half = threadIdx.x >> 8;
        unsigned total[2] = {0, 0}, before[2] = {0, 0};
        if (2 * pair < bins) {
#pragma unroll 16
            for (int t = half; t < a.tiles; t += 2) {
                const uint2 c = *reinterpret_cast<const uint2*>(a.count + (size_t)t * bins + 2 * pair);
                total[0] += c.x;
                total[1] += c.y;
                before[0] += t < (int)blockIdx.x ? c.x : 0;
                before[1] += t < (int)blockIdx.x ? c.y : 0;
            }
        }
        sums[half][0][2 * pair] = total[0];
        sums[half][0][2 * pair + 1] = total[1];
        sums[half][1][2 * pair] = before[0];
        sums[half][1][2 * pair + 1] = before[1];
    }
    __syncthreads();
    const int d0 = threadIdx.x;                       // one digit to a thread
    const unsigned mine = sums[0][0][d0] + sums[1][0][d0];
    unsigned incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    unsigned off = incl - mine;
    for (int w = 0; w < warp; ++w) off += wsum[w];
    base[d0] = off + sums[0][1][d0] + sums[1][1][d0];

    const int i0 = blockIdx.x * a.tile, i1 = min(a.n, i0 + a.tile);
    for (int at = i0; at < i1; at += kTile) {
        for (int d = lane; d < bins; d += 32) cnt[warp][d] = 0;
        // each warp ranks its own stretch
        unsigned key[ROUNDS], rank[ROUNDS];
        int pos[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int i = at + warp * (32 * ROUNDS) + r * 32 + lane;
            const bool in = i < i1;
            key[r] = in ? sort_key<I>(a, i) : 0u;
            if constexpr (sizeof(I) >= 4) pos[r] = i;
            else pos[r] = in ? (int)a.pos[i] : 0;
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            rank[r] = rank_digit(cnt[warp], (key[r] >> a.shift) & (bins - 1), a.bits, at + warp * (32 * ROUNDS) + r * 32 + lane < i1, lane);
        __syncthreads();
        if (d0 < bins) {                               // each warp's first place for each digit, relative to the tile's
            unsigned b = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const unsigned c = cnt[w][d0];
                cnt[w][d0] = (unsigned short)b;
                b += c;
            }
            sums[0][0][d0] = base[d0];
            base[d0] += b;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int i = at + warp * (32 * ROUNDS) + r * 32 + lane;
            if (i < i1) {
                const unsigned d = (key[r] >> a.shift) & (bins - 1), to = sums[0][0][d] + cnt[warp][d] + rank[r];
                a.key_out[to] = key[r];
                a.pos_out[to] = (unsigned)pos[r];
                if (a.next) atomicAdd(&a.next[(size_t)(to / (unsigned)a.tile) * bins + ((key[r] >> (a.shift + a.bits)) & (bins - 1))], 1u);
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) atomicAdd(&a.counters->sorted[a.pass], 1u);
}

// Up to 8192 tokens: key and position make one 32-bit number, all of them are in every block's shared memory, and a warp
// finds a token's place by counting the smaller ones.  The other warps write the zeros of the block's share of the rows,
// which begins at a multiple of 32 rows; its bits (32 KB at most, for all of kSmallRows) are in shared memory too.
// Counting keeps the arithmetic busy and zeros the memory, so the two hide each other: 18 us (by itself and cold, under ncu) for
// 4099 tokens and the 61 MB of rows that they do not meet in a table of 32000 x 1001 16-bit elements.
template <class I>
__global__ void __launch_bounds__(1024) emb_sort_small(const SortArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int blocks = gridDim.x, b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, padded = (a.n + 127) / 128 * 128;
    auto cut = [&](int k) { return min(a.rows, (a.rows + 31) / 32 * k / blocks * 32); };
    const long long first = cut(b), last = cut(b + 1);
    const int words = (int)((last - first + 31) / 32);
    unsigned* all = reinterpret_cast<unsigned*>(smem);
    unsigned* met = all + padded;
    for (int i = threadIdx.x; i < words; i += 1024) met[i] = 0;
    __syncthreads();
#pragma unroll 8
    for (int i = threadIdx.x; i < padded; i += 1024) {
        const long long k = i < a.n ? token_key<I>(a, i) : a.rows;
        all[i] = i < a.n ? (unsigned)k << 13 | (unsigned)i : 0xffffffffu;
        if (k >= first && k < last) atomicOr(met + (k - first) / 32, 1u << (k & 31));
    }
    if (b == 0 && threadIdx.x == 0) a.counters->short_runs = a.counters->long_runs = 0;
    __syncthreads();
    if (warp < kRankWarps) {
        for (int i = b * kRankWarps + warp; i < a.n; i += blocks * kRankWarps) {
            const unsigned mine = all[i];
            unsigned before = 0;
#pragma unroll 4
            for (int j = lane * 4; j < padded; j += 128) {
                const uint4 q = *reinterpret_cast<const uint4*>(all + j);
                before += (q.x < mine) + (q.y < mine) + (q.z < mine) + (q.w < mine);
            }
            for (int o = 16; o >= 1; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
            if (lane == 0) {
                a.key_out[before] = mine >> 13;
                a.pos_out[before] = mine & (kSmallTokens - 1);
            }
        }
    } else {
        for (long long r0 = first + (long long)(warp - kRankWarps) * a.zero.per_warp; r0 < last; r0 += (32LL - kRankWarps) * a.zero.per_warp) {
            const int at = (int)(r0 - first), here = (int)min((long long)a.zero.per_warp, last - r0);
            unsigned todo = ~(met[at >> 5] >> (at & 31));
            if (here < 32) todo &= (1u << here) - 1;
            zero_marked(a.zero, r0, todo);
        }
    }
}

// ---- sums ----------------------------------------------------------------------------------------------
struct EmbSumArgs {
    const void* dy;
    const unsigned *key, *pos;
    void* grad;
    float* part;                 // [chunks][2][D]: end of a run begun in an earlier chunk, begin of a run that goes on
    uint2* crossing;             // (chunk, id) in which a run begins that goes on, in any order: short runs from the front, long
    Counters* counters;          // ones from the back
    long long items;
    unsigned rows;
    int n, D, packs, chunks, chunk;
    float scale;
    ZeroArgs zero;
    long long blocks;
};

template <class T, int EV>
__device__ __forceinline__ void write_row(const EmbSumArgs& a, unsigned v, long long c, const float2 (&acc)[(EV + 1) / 2]) {
    float2 r[(EV + 1) / 2];
#pragma unroll
    for (int k = 0; k < (EV + 1) / 2; ++k) r[k] = mul2(acc[k], make_float2(a.scale, a.scale));
    store_stream<T, EV>(static_cast<T*>(a.grad) + (long long)v * a.D + c, pack_pairs<T, EV>(r));
}

// a run that begins in chunk c goes on in the next one
__device__ __forceinline__ void note_crossing(const EmbSumArgs& a, int c, unsigned id) {
    const bool is_long = c + kLongRun < a.chunks && a.key[(long long)(c + kLongRun) * a.chunk] == id;
    const unsigned k = atomicAdd(is_long ? &a.counters->long_runs : &a.counters->short_runs, 1u);
    a.crossing[is_long ? a.chunks - 1 - k : k] = make_uint2((unsigned)c, id);
}

// Chunks of the sorted tokens, EV columns to a thread; bound by memory: 96 us (under ncu) for 65536 tokens of 2048 bf16 and
// the part of the zeros of 128000 rows that the sort left.
template <class T, int EV>
__global__ void __launch_bounds__(256) emb_sum(const EmbSumArgs a) {
    constexpr int P = (EV + 1) / 2, U = 8;                // U rows of grad_out are under way together
    after_predecessor();
    // blocks that sum and blocks that write zeros take turns, so that reads and writes share the memory all the time
    const long long total = a.blocks + a.zero.batches, z0 = blockIdx.x * a.zero.batches / total, z1 = (blockIdx.x + 1) * a.zero.batches / total;
    if (z1 > z0) {
        zero_batch(a.zero, z0 + a.counters->zero_next);         // the batches before were written beside the sort
        return;
    }
    const long long it = (blockIdx.x - z0) * 256 + threadIdx.x;
    if (it >= a.items) return;
    const int c = (int)(it / a.packs), p = (int)(it - (long long)c * a.packs) * EV;
    const int s = c * a.chunk, e = min(a.n, s + a.chunk);
    unsigned cur = a.key[s];
    const unsigned before = s > 0 ? a.key[s - 1] : a.rows, after = e < a.n ? a.key[e] : a.rows;
    bool begun = before == cur;                           // the run began in an earlier chunk
    float2 acc[P];
#pragma unroll
    for (int k = 0; k < P; ++k) acc[k] = make_float2(0.f, 0.f);
    auto keep = [&](float* to) {
#pragma unroll
        for (int k = 0; k < EV; ++k) to[k] = k & 1 ? acc[k / 2].y : acc[k / 2].x;
    };
    float* part = a.part + 2LL * c * a.D + p;
    for (int i = s; i < e; i += U) {
        unsigned key[U], pos[U];
#pragma unroll
        for (int j = 0; j < U; j += 4) {                  // the lists are padded to whole chunks
            const uint4 k4 = *reinterpret_cast<const uint4*>(a.key + i + j), p4 = *reinterpret_cast<const uint4*>(a.pos + i + j);
            key[j] = k4.x; key[j + 1] = k4.y; key[j + 2] = k4.z; key[j + 3] = k4.w;
            pos[j] = p4.x; pos[j + 1] = p4.y; pos[j + 2] = p4.z; pos[j + 3] = p4.w;
        }
        Pack<T, EV> g[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (i + j >= e) key[j] = a.rows;
            if (key[j] < a.rows) g[j] = load_stream<T, EV>(static_cast<const T*>(a.dy) + (long long)pos[j] * a.D + p);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (i + j >= e) break;
            if (cur >= a.rows) return;
            if (key[j] != cur) {
                if (begun) keep(part);
                else write_row<T, EV>(a, cur, p, acc);
                begun = false;
                cur = key[j];
                if (cur >= a.rows) return;                // only keys that get no gradient follow
#pragma unroll
                for (int k = 0; k < P; ++k) acc[k] = make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int k = 0; k < P; ++k) acc[k] = add2(acc[k], pair_of(g[j], k));
        }
    }
    if (begun) {
        keep(part);
    } else if (after == cur) {
        keep(part + a.D);
        if (p == 0) note_crossing(a, c, cur);
    } else {
        write_row<T, EV>(a, cur, p, acc);
    }
}

// The same for rows that allow narrow accesses only (EV elements of 2 or 4 bytes): a warp takes a chunk and kCols
// accesses of each lane, a stretch of 32 apart; the chunk's keys and positions are in its lanes.  Bound by the number of
// accesses: 13 us (under ncu) for 4099 tokens of 1001 16-bit elements.
constexpr int kCols = 4;
template <class T, int EV>
__global__ void __launch_bounds__(256) emb_sum_narrow(const EmbSumArgs a) {
    constexpr int P = (EV + 1) / 2, U = 8;
    after_predecessor();
    const long long total = a.blocks + a.zero.batches, z0 = blockIdx.x * a.zero.batches / total, z1 = (blockIdx.x + 1) * a.zero.batches / total;
    if (z1 > z0) {
        zero_batch(a.zero, z0 + a.counters->zero_next);
        return;
    }
    const long long it = (blockIdx.x - z0) * 8 + (threadIdx.x >> 5);
    if (it >= a.items) return;
    const int tiles = (a.packs + 32 * kCols - 1) / (32 * kCols), lane = threadIdx.x & 31;
    const int c = (int)(it / tiles), first = (int)(it - (long long)c * tiles) * 32 * kCols + lane;
    const int s = c * a.chunk, count = min(a.n - s, a.chunk);
    const unsigned key = lane < count ? a.key[s + lane] : a.rows, pos = lane < count ? a.pos[s + lane] : 0;
    const unsigned before = s > 0 ? a.key[s - 1] : a.rows, after = s + count < a.n ? a.key[s + count] : a.rows;
    unsigned cur = __shfl_sync(0xffffffffu, key, 0);
    bool begun = before == cur;
    float2 acc[kCols][P];
    auto clear = [&] {
#pragma unroll
        for (int j = 0; j < kCols; ++j)
#pragma unroll
            for (int k = 0; k < P; ++k) acc[j][k] = make_float2(0.f, 0.f);
    };
    auto keep = [&](float* part) {
#pragma unroll
        for (int j = 0; j < kCols; ++j)
            if (first + 32 * j < a.packs) {
#pragma unroll
                for (int k = 0; k < EV; ++k) part[(first + 32 * j) * EV + k] = k & 1 ? acc[j][k / 2].y : acc[j][k / 2].x;
            }
    };
    auto finish = [&] {
#pragma unroll
        for (int j = 0; j < kCols; ++j)
            if (first + 32 * j < a.packs) write_row<T, EV>(a, cur, (long long)(first + 32 * j) * EV, acc[j]);
    };
    float* part = a.part + 2LL * c * a.D;
    clear();
    for (int i = 0; i < count; i += U) {
        Pack<T, EV> g[U][kCols];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned k = __shfl_sync(0xffffffffu, key, min(i + u, 31));
            const T* row = static_cast<const T*>(a.dy) + (long long)__shfl_sync(0xffffffffu, pos, min(i + u, 31)) * a.D;
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
                g[u][j] = {};
                if (i + u < count && k < a.rows && first + 32 * j < a.packs) g[u][j] = load_stream<T, EV>(row + (long long)(first + 32 * j) * EV);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= count || cur >= a.rows) break;
            const unsigned k = __shfl_sync(0xffffffffu, key, i + u);
            if (k != cur) {
                if (begun) keep(part);
                else finish();
                cur = k;
                begun = false;
                clear();
            }
#pragma unroll
            for (int j = 0; j < kCols; ++j)
#pragma unroll
                for (int q = 0; q < P; ++q) acc[j][q] = add2(acc[j][q], pair_of(g[u][j], q));
        }
    }
    if (cur >= a.rows) return;
    if (begun) {
        keep(part);
    } else if (after == cur) {
        keep(part + a.D);
        if (first == 0) note_crossing(a, c, cur);
    } else {
        finish();
    }
}

// Runs that cross chunks.  Up to kLongRun parts: a warp adds them for 32 accesses of COLS columns.  Longer ones: a block, 32
// columns, kRuns stretches of the run's parts, the stretches' sums added in order.  18 us (by itself and cold, under ncu)
// for 65536 tokens of 2048 bf16 with the frequencies of text.
constexpr int kRuns = 16;
template <class T, int COLS>
__global__ void __launch_bounds__(32 * kRuns) emb_join(const EmbSumArgs a) {
    __shared__ float sh[kRuns][32];
    __shared__ int other;
    after_predecessor();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int wide_tiles = (a.D + 32 * COLS - 1) / (32 * COLS);
    const long long work = (long long)a.counters->short_runs * wide_tiles;
    for (long long i = (long long)blockIdx.x * kRuns + ty; i < work; i += (long long)gridDim.x * kRuns) {
        const uint2 run = a.crossing[i / wide_tiles];
        const int c = (int)run.x, col = ((int)(i % wide_tiles) * 32 + tx) * COLS;
        const unsigned v = run.y;
        // the chunks that begin with the run's id follow each other
        const bool same = c + 1 + tx < a.chunks && a.key[(long long)(c + 1 + tx) * a.chunk] == v;
        const unsigned more = __ballot_sync(0xffffffffu, same);
        const int parts = 1 + (more == 0xffffffffu ? 32 : __ffs(~more) - 1);
        if (col >= a.D) continue;
        float2 acc[(COLS + 1) / 2];
#pragma unroll
        for (int j = 0; j < (COLS + 1) / 2; ++j) acc[j] = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < parts; ++k) {
            // written by the kernel before, which this one overlaps: no read-only load
            const float* q = a.part + (2LL * (c + k) + (k == 0 ? 1 : 0)) * a.D + col;
            if constexpr (COLS == 4) {
                const float4 v4 = __ldcg(reinterpret_cast<const float4*>(q));
                acc[0] = add2(acc[0], make_float2(v4.x, v4.y));
                acc[1] = add2(acc[1], make_float2(v4.z, v4.w));
            } else {
                acc[0].x += __ldcg(q);
            }
        }
        write_row<T, COLS>(a, v, col, acc);
    }
    const int tiles = (a.D + 31) / 32;
    const long long long_work = (long long)a.counters->long_runs * tiles;
    for (long long i = blockIdx.x; i < long_work; i += gridDim.x) {
        const uint2 run = a.crossing[a.chunks - 1 - i / tiles];
        const int c = (int)run.x, col = (int)(i % tiles) * 32 + tx;
        const unsigned v = run.y;
        int end = c + kLongRun;                            // the first chunk that begins with another id, or none
        for (bool found = false; !found; end += found ? 0 : 32 * kRuns) {
            if (threadIdx.x == 0) other = 0x7fffffff;
            __syncthreads();
            const int k = end + (int)threadIdx.x;
            if (k >= a.chunks || a.key[(long long)k * a.chunk] != v) atomicMin(&other, min(k, a.chunks));
            __syncthreads();
            found = other != 0x7fffffff;
            if (found) end = other;
            __syncthreads();
        }
        const int parts = end - c, per = (parts + kRuns - 1) / kRuns, k0 = ty * per, k1 = min(parts, k0 + per);
        float t = 0.f;
        if (col < a.D) {
#pragma unroll 8
            for (int k = k0; k < k1; ++k) t += a.part[(2LL * (c + k) + (k == 0 ? 1 : 0)) * a.D + col];
        }
        sh[ty][tx] = t;
        __syncthreads();
        if (ty == 0 && col < a.D) {
            const int runs = (parts + per - 1) / per;
            for (int k = 1; k < runs; ++k) t += sh[k][tx];
            const float2 acc[1] = {make_float2(t, 0.f)};
            write_row<T, 1>(a, v, col, acc);
        }
        __syncthreads();
    }
}

// ---- few tokens -------------------------------------------------------------------------------------------
constexpr int kFewTokens = 256;
struct FewArgs {
    SortArgs sort;               // ids, rows, padding, zeros
    const void* dy;
    void* grad;
    int D, packs;
    float scale;
};
template <class T, int EV, class I>
__global__ void __launch_bounds__(256) emb_few(const FewArgs a) {
    __shared__ unsigned key[kFewTokens], met[kSmallRows / 32];
    __shared__ unsigned short same[kFewTokens];
    __shared__ unsigned count[8];
    const int n = a.sort.n, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned k = (int)threadIdx.x < n ? token_key<I>(a.sort, threadIdx.x) : (unsigned)a.sort.rows;
    if ((int)blockIdx.x >= n) {
        // a share of the rows, from a multiple of 32 rows on
        const int blocks = gridDim.x - n, b = blockIdx.x - n;
        auto cut = [&](int j) { return min(a.sort.rows, (a.sort.rows + 31) / 32 * j / blocks * 32); };
        for (long long first = cut(b), last = cut(b + 1); first < last; first += kSmallRows) {
            const long long end = min(last, first + kSmallRows);
            const int words = (int)((end - first + 31) / 32);
            __syncthreads();
            for (int i = threadIdx.x; i < words; i += 256) met[i] = 0;
            __syncthreads();
            if (k >= first && k < end) atomicOr(met + (k - first) / 32, 1u << (k & 31));
            __syncthreads();
            for (long long r0 = first + (long long)warp * a.sort.zero.per_warp; r0 < end; r0 += 8LL * a.sort.zero.per_warp) {
                const int at = (int)(r0 - first), here = (int)min((long long)a.sort.zero.per_warp, end - r0);
                unsigned todo = ~(met[at >> 5] >> (at & 31));
                if (here < 32) todo &= (1u << here) - 1;
                zero_marked(a.sort.zero, r0, todo);
            }
        }
        return;
    }
    key[threadIdx.x] = k;
    __syncthreads();
    const unsigned mine = key[blockIdx.x];
    if (mine >= (unsigned)a.sort.rows) return;
    const unsigned votes = __ballot_sync(0xffffffffu, k == mine);
    if (lane == 0) count[warp] = __popc(votes);
    __syncthreads();
    unsigned place = __popc(votes & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < 8; ++w) {
        if (w < warp) place += count[w];
        total += count[w];
    }
    if (k == mine) same[place] = (unsigned short)threadIdx.x;
    __syncthreads();
    if (same[0] != blockIdx.x) return;                     // an earlier token has this id
    constexpr int P = (EV + 1) / 2, U = 8;
    for (int p = threadIdx.x; p < a.packs; p += 256) {
        float2 acc[P];
#pragma unroll
        for (int j = 0; j < P; ++j) acc[j] = make_float2(0.f, 0.f);
        for (unsigned i = 0; i < total; i += U) {
            Pack<T, EV> g[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                g[u] = {};
                if (i + u < total) g[u] = load_stream<T, EV>(static_cast<const T*>(a.dy) + (long long)same[i + u] * a.D + (long long)p * EV);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u < total) {
#pragma unroll
                    for (int j = 0; j < P; ++j) acc[j] = add2(acc[j], pair_of(g[u], j));
                }
        }
#pragma unroll
        for (int j = 0; j < P; ++j) acc[j] = mul2(acc[j], make_float2(a.scale, a.scale));
        store_stream<T, EV>(static_cast<T*>(a.grad) + (long long)mine * a.D + (long long)p * EV, pack_pairs<T, EV>(acc));
    }
}

struct EmbPlan {
    int tile, tiles, passes, bits, chunk, chunks;
    bool small;
    size_t key[2], pos[2], count[kMaxPasses], crossing, counters, met, clear, clear_end, part, bytes;
};
EmbPlan emb_plan(long long n, long long rows, int D) {
    EmbPlan p{};
    const long long per = (n + (long long)kMaxTiles * kTile - 1) / ((long long)kMaxTiles * kTile);
    p.tile = (int)(kTile * (per < 1 ? 1 : per));
    p.tiles = (int)((n + p.tile - 1) / p.tile);
    p.small = n <= kSmallTokens && rows <= kSmallRows;
    int bits = 0;
    while (bits < 32 && (rows >> bits) != 0) ++bits;          // keys are 0 .. rows
    p.passes = (bits + 8) / 9;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.chunk = p.small ? kSmallChunk : kChunk;
    p.chunks = (int)((n + p.chunk - 1) / p.chunk);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) & ~(size_t)255;
        return r;
    };
    for (int k = 0; k < 2; ++k) {
        p.key[k] = take((size_t)p.chunks * p.chunk * 4);
        p.pos[k] = take((size_t)p.chunks * p.chunk * 4);
    }
    p.crossing = take((size_t)p.chunks * sizeof(uint2));
    p.count[0] = take((size_t)p.tiles * kMaxBins * 4);
    p.clear = at;                                              // what is cleared first: from here ..
    for (int k = 1; k < p.passes; ++k) p.count[k] = take((size_t)p.tiles * kMaxBins * 4);
    p.counters = take(sizeof(Counters));
    p.met = take((size_t)((rows + 31) / 32) * 4);
    p.clear_end = at;                                          // .. to here
    p.part = take((size_t)p.chunks * 2 * (size_t)D * 4);
    p.bytes = at;
    return p;
}

constexpr long long kMaxTokens = (1LL << 31) - 1 - (long long)kMaxTiles * kTile;
constexpr long long kMaxRows = (1LL << 31) - 1;

// elements of an access: 16 bytes, or two 16-bit elements, or one
int emb_access(int es, int D, const void* a, const void* b) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (uintptr_t)D * es;
    return (all & 15) == 0 ? 16 / es : (all & 3) == 0 ? 4 / es : 1;
}

}  // namespace

extern "C" {

int hfuse_embedding(const void* table, int64_t rows, int D, int dtype, const void* ids, int64_t n, int id_bytes, float scale,
                    void* out, hfuse_stream_t stream) {
    if (!lm_type_ok(dtype) || rows <= 0 || D <= 0 || n < 0 || (id_bytes != 4 && id_bytes != 8)) return HFUSE_ERR_BAD_ARG;
    if (rows > kMaxRows || n > kMaxTokens || D > kMaxWidth) return HFUSE_ERR_TOO_LARGE;
    if (n == 0) return HFUSE_OK;
    if (!table || !ids || !out) return HFUSE_ERR_BAD_ARG;
    const size_t es = lm_type_size(dtype);
    if (!aligned_to(table, es) || !aligned_to(out, es) || !aligned_to(ids, id_bytes)) return HFUSE_ERR_ALIGNMENT;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    EmbFwdArgs a{};
    a.table = table; a.ids = ids; a.out = out;
    a.n = n; a.rows = rows; a.D = D; a.scale = scale;
    // whole accesses; shifted ones for 16-bit rows that have a few; single elements
    const bool aligned = aligned_to(table, 16) && aligned_to(out, 16) && D * es % 16 == 0, shifted = !aligned && es == 2 && D >= 32;
    a.packs = aligned || shifted ? (int)(D * es / 16) : D;
    a.lanes = 32;
    while (a.lanes > 1 && a.lanes / 2 * kAhead >= a.packs) a.lanes /= 2;
    const int per = 256 / a.lanes;
    const long long stretches = ((long long)a.packs + a.lanes * kAhead - 1) / (a.lanes * kAhead);
    const dim3 grid((unsigned)((n + per - 1) / per), (unsigned)(stretches < 65535 ? stretches : 65535));
    return by_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        constexpr int EV = 16 / sizeof(T);
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        auto go = [&](auto id) {
            using I = decltype(id);
            if constexpr (sizeof(T) == 2) {
                if (shifted) {
                    emb_fwd_shifted<T, I><<<grid, 256, 0, s>>>(a);
                    return check_launch();
                }
            }
            if (aligned) emb_fwd<T, EV, I><<<grid, 256, 0, s>>>(a);
            else emb_fwd<T, 1, I><<<grid, 256, 0, s>>>(a);
            return check_launch();
        };
        return id_bytes == 8 ? go((long long)0) : go((int)0);
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
    if (rows > kMaxRows || n > kMaxTokens || D > kMaxWidth) return HFUSE_ERR_TOO_LARGE;
    if (!grad_table || (n > 0 && (!grad_out || !ids))) return HFUSE_ERR_BAD_ARG;
    const size_t es = lm_type_size(dtype);
    if (!aligned_to(grad_out, es) || !aligned_to(grad_table, es) || (n > 0 && !aligned_to(ids, id_bytes)) || !aligned_to(workspace, 16))
        return HFUSE_ERR_ALIGNMENT;
    const EmbPlan p = n > 0 ? emb_plan(n, rows, D) : EmbPlan{};
    if (n > 0 && (!workspace || workspace_bytes < p.bytes)) return HFUSE_ERR_WORKSPACE;
    DeviceFacts f;
    if (int rc = device_facts(f)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (n == 0) {
        if (cudaMemsetAsync(grad_table, 0, (size_t)rows * D * es, s) == cudaSuccess) return HFUSE_OK;
        (void)cudaGetLastError();
        return HFUSE_ERR_LAUNCH;
    }
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    auto at = [&](size_t off) { return reinterpret_cast<unsigned*>(ws + off); };
    ZeroArgs z{};
    z.grad = static_cast<unsigned char*>(grad_table); z.met = at(p.met); z.row_bytes = (long long)D * es; z.rows = rows;
    const long long wanted = (16 << 10) / z.row_bytes;          // about 16 KB to a warp
    z.per_warp = 1;
    while (z.per_warp < 32 && 2 * z.per_warp <= wanted) z.per_warp *= 2;
    z.batches = (rows + 8LL * z.per_warp - 1) / (8LL * z.per_warp);
    SortArgs a{};
    a.ids = ids; a.rows = rows; a.padding = padding_id;
    a.n = (int)n; a.tile = p.tile; a.tiles = p.tiles; a.bits = p.bits; a.passes = p.passes; a.met = at(p.met);
    a.counters = reinterpret_cast<Counters*>(ws + p.counters);
    a.clear = at(p.clear); a.clear_words = (long long)((p.clear_end - p.clear) / 4);
    a.zero = z;
    int rc = HFUSE_OK;
    const int ev = emb_access((int)es, D, grad_out, grad_table);
    if (n <= kFewTokens) {
        FewArgs w{};
        w.sort = a; w.dy = grad_out; w.grad = grad_table; w.D = D; w.packs = D / ev; w.scale = scale;
        const long long shares = (z.batches < 4LL * f.sms ? z.batches : 4LL * f.sms);
        const int blocks = (int)(n + shares);
        return by_type(dtype, [&](auto t) {
            using T = typename decltype(t)::type;
            constexpr int EV = 16 / sizeof(T), EV4 = 4 / sizeof(T);
            auto go = [&](auto id) {
                using I = decltype(id);
                return ev == EV    ? launch_kernel(emb_few<T, EV, I>, blocks, 256, 0, s, false, w)
                       : ev == EV4 ? launch_kernel(emb_few<T, EV4, I>, blocks, 256, 0, s, false, w)
                                   : launch_kernel(emb_few<T, 1, I>, blocks, 256, 0, s, false, w);
            };
            return id_bytes == 8 ? go((long long)0) : go((int)0);
        });
    }
    const int last = p.small ? 0 : (p.passes - 1) & 1;
    if (p.small) {
        a.key_out = at(p.key[0]); a.pos_out = at(p.pos[0]);
        const size_t smem = (size_t)(n + 127) / 128 * 512 + (size_t)(rows + 31) / 32 * 4 + 16;      // a share's bits are a part of all
        rc = id_bytes == 8 ? launch_kernel(emb_sort_small<long long>, f.sms, 1024, smem, s, false, a)
                           : launch_kernel(emb_sort_small<int>, f.sms, 1024, smem, s, false, a);
        if (rc) return rc;
        z.batches = 0;                                          // nothing is left for the next kernel
    } else {
        if ((rc = launch_kernel(emb_clear, f.sms, 256, 0, s, false, a))) return rc;
        for (int k = 0; k < p.passes; ++k) {
            a.pass = k;
            a.shift = k * p.bits;
            a.key = at(p.key[(k + 1) & 1]); a.pos = at(p.pos[(k + 1) & 1]);
            a.key_out = at(p.key[k & 1]); a.pos_out = at(p.pos[k & 1]);
            a.count = at(p.count[k]); a.next = k + 1 < p.passes ? at(p.count[k + 1]) : nullptr;
            const int blocks = p.tiles + 3 * f.sms;
            if (k > 0) {
                rc = launch_kernel(emb_sort_scatter<NoIds>, blocks, kSortThreads, 0, s, true, a);
            } else if (id_bytes == 8) {
                rc = launch_kernel(emb_sort_count<long long>, p.tiles, kSortThreads, 0, s, true, a);
                if (!rc) rc = launch_kernel(emb_sort_scatter<long long>, blocks, kSortThreads, 0, s, true, a);
            } else {
                rc = launch_kernel(emb_sort_count<int>, p.tiles, kSortThreads, 0, s, true, a);
                if (!rc) rc = launch_kernel(emb_sort_scatter<int>, blocks, kSortThreads, 0, s, true, a);
            }
            if (rc) return rc;
        }
    }
    EmbSumArgs b{};
    b.dy = grad_out; b.key = at(p.key[last]); b.pos = at(p.pos[last]); b.grad = grad_table;
    b.part = reinterpret_cast<float*>(ws + p.part); b.crossing = reinterpret_cast<uint2*>(ws + p.crossing); b.counters = a.counters;
    b.rows = (unsigned)rows; b.n = (int)n; b.D = D; b.scale = scale;
    const bool narrow = ev * es < 16;
    b.chunk = p.small || narrow || n <= 32768 ? p.chunk : kWideChunk;      // the workspace is for the shorter ones
    b.chunks = (int)((n + b.chunk - 1) / b.chunk);
    b.zero = z;
    b.packs = D / ev;
    b.items = (long long)b.chunks * (narrow ? (b.packs + 32 * kCols - 1) / (32 * kCols) : b.packs);      // of warps, of threads
    b.blocks = narrow ? (b.items + 7) / 8 : (b.items + 255) / 256;
    const long long grid = b.blocks + z.batches;
    if (grid > kMaxRows) return HFUSE_ERR_TOO_LARGE;
    return by_type(dtype, [&](auto t) {
        using T = typename decltype(t)::type;
        constexpr int EV = 16 / sizeof(T), EV4 = 4 / sizeof(T);
        rc = ev == EV    ? launch_kernel(emb_sum<T, EV>, (int)grid, 256, 0, s, true, b)
             : ev == EV4 ? launch_kernel(emb_sum_narrow<T, EV4>, (int)grid, 256, 0, s, true, b)
                         : launch_kernel(emb_sum_narrow<T, 1>, (int)grid, 256, 0, s, true, b);
        if (rc) return rc;
        return ev == EV ? launch_kernel(emb_join<T, 4>, 4 * f.sms, 32 * kRuns, 0, s, true, b)
                        : launch_kernel(emb_join<T, 1>, 4 * f.sms, 32 * kRuns, 0, s, true, b);
    });
}

}  // extern "C"
