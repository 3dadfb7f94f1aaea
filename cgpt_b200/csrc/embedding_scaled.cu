// Scaled embedding lookup with dropout, and its gradient, for sm_100a.
//
//   forward    out[t] = dropout(scale * W[ids[t]])             (an id outside the table gives a zero row)
//   backward   dW[v] (+)= scale * sum_{t: ids[t] = v} drop(dout[t])     ids equal to padding_id or outside the table are skipped
//
// Backward. Token ids follow word frequencies: one id can hold a twentieth of all tokens (or, in a padded batch, most of
// them), so one owner per table row would leave one CTA adding thousands of rows. Here the tokens are sorted by id (stable
// radix sort, this file) and the SORTED list is cut into chunks of kChunk tokens, one group of threads each: a group adds its
// tokens' rows run by run, several rows in flight. A run inside a chunk is written to the table at once; runs that cross chunks
// are joined in shared memory within a CTA, and a run that crosses CTAs leaves fp32 partial rows that a last kernel adds. Every
// sum is taken in an order that follows from the ids alone, so results repeat bit for bit, and no group has more rows than others.
// Table rows without a token are zeroed by the same launch (their owners look the row up in the sorted list), so the table
// is written once.
//
// Memory-bound: backward reads dout once and writes the table once; the sort moves 16 bytes per token and pass.
#include <cooperative_groups.h>

#include "philox.cuh"
#include "launch_counter.h"

namespace cgpt {
namespace {

constexpr int kThreads = 128;        // lookup; threads per row at most
constexpr int kSumThreads = 512;
constexpr int kChunk = 16;           // sorted tokens per group of threads
constexpr int kInFlight = 8;         // rows a group loads before it adds them
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kKeysPerThread = 8;
constexpr int kSortTile = kSortThreads * kKeysPerThread;
constexpr int kMaxDigitBits = 9;
constexpr int kClusterThreads = 1024;
constexpr int kMaxCluster = 16;

// kLookups consecutive tokens per group of threads and trip: their ids, then their rows, are loaded together, and the decisions
// (about 10 instructions an element, most of the kernel's work) are made while the rows are on their way.
constexpr int kLookups = 4;
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
scaled_embedding_forward_kernel(T* __restrict__ out, const std::uint32_t* __restrict__ ids, const T* __restrict__ weight,
                                long long tokens, std::uint32_t vocab, int hidden, float scale, int group, const DropoutArgs args) {
    using Raw = typename RawVec<sizeof(T) * VEC>::type;
    const HoistedPhilox gen(args);
    const int lane = threadIdx.x % group;
    const long long step = static_cast<long long>(gridDim.x) * (kThreads / group) * kLookups;
    for (long long t0 = (static_cast<long long>(blockIdx.x) * (kThreads / group) + threadIdx.x / group) * kLookups; t0 < tokens; t0 += step) {
        std::uint32_t id[kLookups];
#pragma unroll
        for (int k = 0; k < kLookups; ++k) id[k] = t0 + k < tokens ? ids[t0 + k] : 0xffffffffu;
        for (int c = lane * VEC; c < hidden; c += group * VEC) {
            Pack<T, VEC> row[kLookups];
#pragma unroll
            for (int k = 0; k < kLookups; ++k)
                if (id[k] < vocab) *reinterpret_cast<Raw*>(&row[k]) = *reinterpret_cast<const Raw*>(weight + static_cast<long long>(id[k]) * hidden + c);
#pragma unroll
            for (int k = 0; k < kLookups; ++k) {
                if (t0 + k < tokens) {
                    const long long e = (t0 + k) * hidden + c;
                    float v[VEC];
                    if (id[k] < vocab) {
                        unpack_pack(v, row[k]);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) v[i] *= scale;
                        if (args.threshold != 0) drop_vec<VEC>(v, gen, e, args);
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) v[i] = 0.f;
                    }
                    store_vec<T, VEC>(out + e, v);
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------- radix sort
// Least significant digit first, `bits` (at most kMaxDigitBits) per pass: digit counts per tile of kSortTile keys, their
// prefix over tiles, then every tile scatters its keys to (keys of smaller digits) + (this digit in earlier tiles) + (rank
// in the tile). The rank counts equal digits in key order, which makes the sort stable.
struct SortPass {
    const std::uint32_t* keys_in;    // first pass: the token ids as given
    const std::uint32_t* vals_in;    // first pass: null (the value is the token's index)
    std::uint32_t* keys_out;
    std::uint32_t* vals_out;
    std::uint32_t* counts;           // [1 << bits][tiles]
    std::uint32_t* totals;           // [1 << bits]
    std::uint32_t* crossing;         // [0]: number of runs that cross a chunk border; cleared by the first pass
    long long n;
    std::uint32_t vocab, skip_id;    // ids >= vocab and skip_id sort behind the table as key `vocab`
    int shift, bits, tiles;
};

__device__ __forceinline__ std::uint32_t sort_key(const SortPass& p, long long i) {
    const std::uint32_t k = p.keys_in[i];
    return p.vals_in == nullptr && (k >= p.vocab || k == p.skip_id) ? p.vocab : k;
}

__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const SortPass p) {
    __shared__ std::uint32_t bins[1 << kMaxDigitBits];
    const int radix = 1 << p.bits;
    for (int d = threadIdx.x; d < radix; d += kSortThreads) bins[d] = 0;
    if (p.vals_in == nullptr && blockIdx.x == 0 && threadIdx.x == 0) *p.crossing = 0;
    __syncthreads();
    const long long base = static_cast<long long>(blockIdx.x) * kSortTile;
#pragma unroll
    for (int j = 0; j < kKeysPerThread; ++j) {
        const long long i = base + j * kSortThreads + threadIdx.x;
        if (i < p.n) atomicAdd(&bins[(sort_key(p, i) >> p.shift) & (radix - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < radix; d += kSortThreads) p.counts[static_cast<long long>(d) * p.tiles + blockIdx.x] = bins[d];
}

// One CTA per digit: exclusive prefix of its counts over the tiles, in place, and their total.
__global__ void __launch_bounds__(kSortThreads)
sort_prefix_kernel(const SortPass p) {
    __shared__ std::uint32_t warp_total[kSortWarps];
    std::uint32_t* row = p.counts + static_cast<long long>(blockIdx.x) * p.tiles;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    std::uint32_t carry = 0;
    for (int t0 = 0; t0 < p.tiles; t0 += kSortThreads) {
        const int t = t0 + threadIdx.x;
        const std::uint32_t v = t < p.tiles ? row[t] : 0;
        std::uint32_t inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const std::uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        std::uint32_t before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            if (w < warp) before += warp_total[w];
            all += warp_total[w];
        }
        if (t < p.tiles) row[t] = before + inc - v;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) p.totals[blockIdx.x] = carry;
}

__global__ void __launch_bounds__(kSortThreads)
sort_scatter_kernel(const SortPass p) {
    __shared__ std::uint32_t seen[kSortWarps][1 << kMaxDigitBits];   // keys of a digit met so far by each warp, then its base
    __shared__ std::uint32_t warp_total[kSortWarps];
    const int radix = 1 << p.bits;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int d = threadIdx.x; d < kSortWarps << kMaxDigitBits; d += kSortThreads) (&seen[0][0])[d] = 0;
    __syncthreads();
    // Order of the keys: (tile, warp, j, lane).
    const long long base = static_cast<long long>(blockIdx.x) * kSortTile + warp * (32 * kKeysPerThread) + lane;
    std::uint32_t key[kKeysPerThread], rank[kKeysPerThread];
#pragma unroll
    for (int j = 0; j < kKeysPerThread; ++j) {
        const long long i = base + j * 32;
        const bool in = i < p.n;
        key[j] = in ? sort_key(p, i) : 0u;
        // keys past the end get a digit of their own, which nobody counts
        const std::uint32_t digit = in ? (key[j] >> p.shift) & (radix - 1) : 0xffffffffu;
        const unsigned peers = __match_any_sync(0xffffffffu, digit);
        const unsigned below = __popc(peers & ((1u << lane) - 1u));
        const std::uint32_t so_far = in ? seen[warp][digit] : 0u;
        rank[j] = so_far + below;
        __syncwarp();
        if (in && below == 0) seen[warp][digit] = so_far + __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    // Digit d: keys of smaller digits (scan of the totals) + earlier tiles, then the warps one after the other.
    std::uint32_t carry = 0;
    for (int d0 = 0; d0 < radix; d0 += kSortThreads) {
        const int d = d0 + threadIdx.x;
        const std::uint32_t v = d < radix ? p.totals[d] : 0;
        std::uint32_t inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const std::uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        std::uint32_t before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            if (w < warp) before += warp_total[w];
            all += warp_total[w];
        }
        carry += all;
        if (d < radix) {
            std::uint32_t at = before + inc - v + p.counts[static_cast<long long>(d) * p.tiles + blockIdx.x];
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                const std::uint32_t here = seen[w][d];
                seen[w][d] = at;
                at += here;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kKeysPerThread; ++j) {
        const long long i = base + j * 32;
        if (i < p.n) {
            const std::uint32_t to = seen[warp][(key[j] >> p.shift) & (radix - 1)] + rank[j];
            p.keys_out[to] = key[j];
            p.vals_out[to] = p.vals_in == nullptr ? static_cast<std::uint32_t>(i) : p.vals_in[i];
        }
    }
}

// The whole sort in one launch, for up to kMaxCluster * kClusterThreads * KEYS tokens: one cluster holds all keys in registers,
// digit counts go round in distributed shared memory, keys of a pass through global memory (L2). A pass is then two cluster
// barriers instead of three launches.
struct ClusterSort {
    const std::uint32_t* ids;
    std::uint32_t *keys[2], *vals[2];   // pass i writes [i & 1]
    std::uint32_t* crossing;
    int n, bits, passes;
    std::uint32_t vocab, skip_id;
};

template <int KEYS>
__global__ void __launch_bounds__(kClusterThreads)
sort_cluster_kernel(const ClusterSort p) {
    constexpr int kWarps = kClusterThreads / 32;
    __shared__ unsigned short seen[kWarps][1 << kMaxDigitBits];   // keys of a digit met so far by each warp, then those of earlier warps
    __shared__ std::uint32_t mine[1 << kMaxDigitBits];            // the CTA's keys of each digit; read by the whole cluster
    __shared__ std::uint32_t base[1 << kMaxDigitBits];
    __shared__ std::uint32_t warp_total[kWarps];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks()), cta = static_cast<int>(cluster.block_rank());
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int radix = 1 << p.bits;
    const int first = (cta * kWarps + warp) * (32 * KEYS) + lane;  // order of the keys: (CTA, warp, j, lane)
    if (cta == 0 && threadIdx.x == 0) *p.crossing = 0;
    std::uint32_t key[KEYS], val[KEYS], rank[KEYS];
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
        const int i = first + j * 32;
        const std::uint32_t k = i < p.n ? p.ids[i] : 0u;
        key[j] = k >= p.vocab || k == p.skip_id ? p.vocab : k;
        val[j] = i;
    }
    for (int pass = 0; pass < p.passes; ++pass) {
        const int shift = pass * p.bits;
        if (pass > 0) {
#pragma unroll
            for (int j = 0; j < KEYS; ++j) {
                const int i = first + j * 32;
                key[j] = i < p.n ? __ldcg(p.keys[(pass - 1) & 1] + i) : 0u;
                val[j] = i < p.n ? __ldcg(p.vals[(pass - 1) & 1] + i) : 0u;
            }
        }
        for (int d = lane; d < radix; d += 32) seen[warp][d] = 0;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
            const bool in = first + j * 32 < p.n;
            // keys past the end get a digit of their own, which nobody counts
            const std::uint32_t digit = in ? (key[j] >> shift) & (radix - 1) : 0xffffffffu;
            const unsigned peers = __match_any_sync(0xffffffffu, digit);
            const unsigned below = __popc(peers & ((1u << lane) - 1u));
            const std::uint32_t so_far = in ? seen[warp][digit] : 0u;
            rank[j] = so_far + below;
            __syncwarp();
            if (in && below == 0) seen[warp][digit] = static_cast<unsigned short>(so_far + __popc(peers));
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < radix) {
            std::uint32_t before = 0;
#pragma unroll 8
            for (int w = 0; w < kWarps; ++w) {
                const std::uint32_t here = seen[w][threadIdx.x];
                seen[w][threadIdx.x] = static_cast<unsigned short>(before);
                before += here;
            }
            mine[threadIdx.x] = before;
        }
        cluster.sync();
        // Digit d of this CTA starts behind all smaller digits and behind digit d of the CTAs before it.
        std::uint32_t all = 0, earlier = 0;
        if (threadIdx.x < radix) {
            for (int c = 0; c < ctas; ++c) {
                const std::uint32_t v = cluster.map_shared_rank(mine, c)[threadIdx.x];
                all += v;
                if (c < cta) earlier += v;
            }
        }
        std::uint32_t inc = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const std::uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        if (threadIdx.x < radix) {
            std::uint32_t smaller = 0;
            for (int w = 0; w < warp; ++w) smaller += warp_total[w];
            base[threadIdx.x] = smaller + inc - all + earlier;
        }
        __syncthreads();
        std::uint32_t *keys_out = p.keys[pass & 1], *vals_out = p.vals[pass & 1];
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
            if (first + j * 32 < p.n) {
                const std::uint32_t digit = (key[j] >> shift) & (radix - 1), to = base[digit] + seen[warp][digit] + rank[j];
                keys_out[to] = key[j];
                vals_out[to] = val[j];
            }
        }
        cluster.sync();   // keys of this pass are written, counts of this pass read
    }
}

// -------------------------------------------------------------------------------------------------------- run sums
struct GradArgs {
    const std::uint32_t* ids;        // sorted; `vocab` marks skipped tokens
    const std::uint32_t* tokens;     // the token of each sorted position
    float* partial;                  // [CTAs][2][hidden]: a run's part that began in an earlier CTA, or goes on in the next one
    std::uint32_t* crossing;         // [0]: count, [1..]: CTAs in which a run starts that goes on in the next CTA
    long long n, hidden;
    std::uint32_t vocab;
    int ctas, accumulate;            // CTAs of the sum launch that hold tokens
    int group, groups;               // threads per row, groups per CTA
    float scale;
};

template <typename T, int VEC>
__device__ __forceinline__ void write_row(T* dst, const float (&acc)[VEC], float scale, int accumulate) {
    float out[VEC];
    if (accumulate) {
        load_vec<T, VEC>(out, dst);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = fmaf(acc[i], scale, out[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = acc[i] * scale;
    }
    store_vec<T, VEC>(dst, out);
}

// fp32 vectors of VEC values, 16 bytes at a time.
template <int VEC>
__device__ __forceinline__ void put_floats(float* to, const float (&v)[VEC]) {
    constexpr int N = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int i = 0; i < VEC; i += N) store_vec<float, N>(to + i, *reinterpret_cast<const float(*)[N]>(&v[i]));
}
template <int VEC>
__device__ __forceinline__ void add_floats(float (&v)[VEC], const float* from) {
    constexpr int N = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int i = 0; i < VEC; i += N) {
        float t[N];
        load_vec<float, N>(t, from + i);
#pragma unroll
        for (int k = 0; k < N; ++k) v[i + k] += t[k];
    }
}

// First position of the sorted list whose id is not below `id`.
__device__ __forceinline__ long long lower_bound(const std::uint32_t* ids, long long n, std::uint32_t id) {
    long long lo = 0, hi = n;
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (ids[mid] < id) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// CTAs [0, g.ctas): g.groups chunks each. The others zero the table rows that no token has, 32 rows per warp.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads, 2)
scaled_embedding_sum_kernel(T* dw, const T* __restrict__ dout, const GradArgs g, const DropoutArgs args) {
    extern __shared__ __align__(16) float parts[];           // [groups][2][group * VEC]: what a chunk's first and last run leave
    __shared__ std::uint32_t ids[kSumThreads * kChunk / 8 + 2], tokens[kSumThreads * kChunk / 8];
    const int lane = threadIdx.x % g.group, group = threadIdx.x / g.group;
    if (blockIdx.x >= static_cast<unsigned>(g.ctas)) {
        const int wl = threadIdx.x & 31;
        const long long first = (static_cast<long long>(blockIdx.x - g.ctas) * (blockDim.x / 32) + (threadIdx.x >> 5)) * 32;
        const long long row = first + wl;
        bool empty = false;
        if (row < g.vocab) {
            const long long at = lower_bound(g.ids, g.n, static_cast<std::uint32_t>(row));
            empty = at == g.n || g.ids[at] != static_cast<std::uint32_t>(row);
        }
        unsigned todo = __ballot_sync(0xffffffffu, empty);
        const float zero[VEC] = {};
        while (todo != 0) {
            const int r = __ffs(todo) - 1;
            todo &= todo - 1;
            for (long long c = static_cast<long long>(wl) * VEC; c < g.hidden; c += 32 * VEC) store_vec<T, VEC>(dw + (first + r) * g.hidden + c, zero);
        }
        return;
    }
    const HoistedPhilox gen(args);
    // The CTA's tokens, with one id before and one behind them; no neighbour: an id that no token has (vocab marks skipped ones).
    const int span = g.groups * kChunk;
    const long long lo = static_cast<long long>(blockIdx.x) * span;
    const int count = g.n - lo < span ? static_cast<int>(g.n - lo) : span;
    constexpr std::uint32_t kNone = 0xffffffffu;
    for (int i = threadIdx.x; i < count + 2; i += blockDim.x) {
        const long long at = lo + i - 1;
        ids[i] = at >= 0 && at < g.n ? g.ids[at] : kNone;
        if (i < count) tokens[i] = g.tokens[lo + i];
    }
    __syncthreads();
    const std::uint32_t* id_at = ids + 1;                     // id_at[-1] .. id_at[count]
    const bool first_from_before = id_at[-1] == id_at[0], last_goes_on = id_at[count] == id_at[count - 1];
    const bool single = id_at[0] == id_at[count - 1];         // all of the CTA's tokens have one id
    if (threadIdx.x == 0 && last_goes_on && id_at[count - 1] < g.vocab && !(single && first_from_before))
        g.crossing[1 + atomicAdd(g.crossing, 1u)] = blockIdx.x;   // their order changes no result
    float* before = g.partial + static_cast<long long>(blockIdx.x) * 2 * g.hidden;
    float* after = before + g.hidden;
    const int width = g.group * VEC;
    float* head = parts + group * 2 * width + lane * VEC;
    float* tail = head + width;
    const int begin = group * kChunk, end = begin + kChunk < count ? begin + kChunk : count;
    for (long long c0 = 0; c0 < g.hidden; c0 += width) {
        const long long c = c0 + lane * VEC;
        if (c < g.hidden && begin < end) {
            float acc[VEC] = {};
            std::uint32_t id = id_at[begin];
            bool open = id_at[begin - 1] == id;               // the run began in an earlier chunk
            for (int p0 = begin; p0 < end; p0 += kInFlight) {
                Pack<T, VEC> rows[kInFlight];
                using Raw = typename RawVec<sizeof(T) * VEC>::type;
#pragma unroll
                for (int u = 0; u < kInFlight; ++u)
                    if (p0 + u < end && id_at[p0 + u] < g.vocab)
                        *reinterpret_cast<Raw*>(&rows[u]) = __ldcs(reinterpret_cast<const Raw*>(dout + static_cast<long long>(tokens[p0 + u]) * g.hidden + c));
#pragma unroll
                for (int u = 0; u < kInFlight; ++u) {
                    if (p0 + u < end) {
                        const std::uint32_t next = id_at[p0 + u];
                        if (next != id) {
                            if (open) put_floats<VEC>(head, acc);
                            else write_row<T, VEC>(dw + static_cast<long long>(id) * g.hidden + c, acc, g.scale, g.accumulate);
#pragma unroll
                            for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
                            id = next;
                            open = false;
                        }
                        if (next < g.vocab) {
                            float v[VEC];
                            unpack_pack(v, rows[u]);
                            if (args.threshold != 0) drop_vec<VEC>(v, gen, static_cast<long long>(tokens[p0 + u]) * g.hidden + c, args);
#pragma unroll
                            for (int i = 0; i < VEC; ++i) acc[i] += v[i];
                        }
                    }
                }
            }
            if (id < g.vocab) {
                if (open) put_floats<VEC>(head, acc);         // also where the whole chunk is one run that goes on
                else if (id_at[end] == id) put_floats<VEC>(tail, acc);
                else write_row<T, VEC>(dw + static_cast<long long>(id) * g.hidden + c, acc, g.scale, g.accumulate);
            }
        }
        __syncthreads();
        // Runs that cross chunks: the threads of group 0 (more, where a group has few) walk over the CTA's chunks in order.
        for (int k = threadIdx.x; k < g.group; k += blockDim.x) {
            const long long col = c0 + k * VEC;
            if (col >= g.hidden) continue;
            float acc[VEC] = {};
            bool carried = false, from_before = false;
            for (int q = 0; q * kChunk < count; ++q) {
                const int b = q * kChunk, e = b + kChunk < count ? b + kChunk : count;
                const std::uint32_t id0 = id_at[b], id1 = id_at[e - 1];
                if (id0 >= g.vocab) break;
                const float* part = parts + q * 2 * width + k * VEC;
                if (id_at[b - 1] == id0) {
                    if (q == 0) { carried = true; from_before = true; }
                    add_floats<VEC>(acc, part);
                    if (id_at[e] != id0 || id1 != id0) {      // the run ends in this chunk
                        if (from_before) put_floats<VEC>(before + col, acc);
                        else write_row<T, VEC>(dw + static_cast<long long>(id0) * g.hidden + col, acc, g.scale, g.accumulate);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
                        carried = from_before = false;
                    }
                }
                if (id1 < g.vocab && id_at[e] == id1 && !(id1 == id0 && id_at[b - 1] == id0)) {
                    add_floats<VEC>(acc, part + width);
                    carried = true;
                }
            }
            if (carried) put_floats<VEC>((from_before ? before : after) + col, acc);
        }
        __syncthreads();
    }
}

// Runs that cross CTAs: the part of the CTA they start in and those of all later CTAs they reach, eight part lanes of 32 x VEC
// columns; a (run, column tile) pair per trip.
constexpr int kJoinThreads = 256;
template <typename T, int VEC>
__global__ void __launch_bounds__(kJoinThreads)
scaled_embedding_join_kernel(T* dw, const GradArgs g) {
    __shared__ float tile[kJoinThreads / 32][32 * VEC];
    const int lane = threadIdx.x & 31, pl = threadIdx.x >> 5;
    const unsigned column_tiles = static_cast<unsigned>((g.hidden + 32 * VEC - 1) / (32 * VEC)), runs = *g.crossing;
    const int span = g.groups * kChunk;
    for (unsigned run = blockIdx.x / column_tiles; run < runs; run += gridDim.x / column_tiles) {
        const long long cta = g.crossing[1 + run];
        const long long col = (static_cast<long long>(blockIdx.x % column_tiles) * 32 + lane) * VEC;
        const std::uint32_t id = g.ids[cta * span + span - 1];
        // last CTA whose first token belongs to the run
        long long lo = cta + 1, hi = g.ctas - 1;
        for (long long reach = 1; lo + reach <= hi && g.ids[(lo + reach) * span] == id; reach *= 2) lo += reach;   // most runs are short
        if (lo + 1 < hi + 1) {
            long long top = hi;
            while (lo < top) {
                const long long mid = (lo + top + 1) >> 1;
                if (g.ids[mid * span] == id) lo = mid;
                else top = mid - 1;
            }
        }
        float acc[VEC] = {};
        if (col < g.hidden)
            for (long long k = cta + pl; k <= lo; k += kJoinThreads / 32) add_floats<VEC>(acc, g.partial + (k * 2 + (k == cta ? 1 : 0)) * g.hidden + col);
        __syncthreads();
        put_floats<VEC>(&tile[pl][lane * VEC], acc);
        __syncthreads();
        if (pl == 0 && col < g.hidden) {
            float t[VEC] = {};
#pragma unroll
            for (int r = 0; r < kJoinThreads / 32; ++r) add_floats<VEC>(t, &tile[r][lane * VEC]);
            write_row<T, VEC>(dw + static_cast<long long>(id) * g.hidden + col, t, g.scale, g.accumulate);
        }
    }
}

int bit_length(std::uint64_t v) {
    int b = 0;
    while (v) { ++b; v >>= 1; }
    return b;
}

// Threads per row: enough for the row's vectors, at most kThreads.
int group_for(std::size_t hidden, int vec) {
    int g = 1;
    while (g < kThreads && static_cast<std::size_t>(g) * vec < hidden) g *= 2;
    return g;
}

// Layout of the run sums: threads per row, groups per CTA, CTAs.
struct SumPlan {
    int group, groups, ctas;
    SumPlan(std::size_t tokens, std::size_t hidden, int vec) {
        group = group_for(hidden, vec);
        // As many groups as threads (and the staged ids) allow, fewer when there are few tokens: then every SM gets some.
        const std::size_t chunks = (tokens + kChunk - 1) / kChunk, share = (chunks + 2 * kNumSMs - 1) / (2 * kNumSMs);
        std::size_t n = kSumThreads / (group < 8 ? 8 : group);
        const std::size_t whole_warps = group < 32 ? 32 / group : 1;
        if (n > share) n = share;
        n = n < whole_warps ? whole_warps : n / whole_warps * whole_warps;
        groups = static_cast<int>(n);
        ctas = static_cast<int>((chunks + n - 1) / n);
    }
};

// Byte offsets of the workspace's parts, enough for every type and alignment.
struct Layout {
    std::size_t keys[2], vals[2], counts, totals, crossing, partial, bytes;
    int tiles;
    Layout(std::size_t tokens, std::size_t hidden) {
        tiles = static_cast<int>((tokens + kSortTile - 1) / kSortTile);
        std::size_t ctas = 0;
        for (int vec : {1, 4, 8}) {
            const SumPlan p(tokens, hidden, vec);
            if (static_cast<std::size_t>(p.ctas) > ctas) ctas = p.ctas;
        }
        bytes = 0;
        auto take = [&](std::size_t n) {
            const std::size_t at = bytes;
            bytes += (n + 255) & ~std::size_t{255};
            return at;
        };
        for (int i = 0; i < 2; ++i) { keys[i] = take(tokens * 4); vals[i] = take(tokens * 4); }
        counts = take((std::size_t{4} << kMaxDigitBits) * tiles);
        totals = take(std::size_t{4} << kMaxDigitBits);
        crossing = take(4 * (ctas + 1));
        partial = take(ctas * 2 * hidden * sizeof(float));
    }
};

bool valid_sizes(std::size_t tokens, std::size_t vocab, std::size_t hidden) {
    return tokens != 0 && vocab != 0 && hidden != 0 && tokens <= 0x7fffffffull && vocab <= 0x7ffffffeull && hidden <= 0x7fffffffull &&
           tokens <= (1ull << 46) / hidden && vocab <= (1ull << 46) / hidden;
}

template <typename T, int VEC>
int launch_sum(void* dw, const void* dout, GradArgs g, const DropoutArgs& args, cudaStream_t s) {
    const SumPlan p(static_cast<std::size_t>(g.n), static_cast<std::size_t>(g.hidden), VEC);
    g.group = p.group;
    g.groups = p.groups;
    g.ctas = p.ctas;
    const int threads = g.groups * g.group;
    const unsigned zero_ctas = g.accumulate ? 0 : static_cast<unsigned>((g.vocab + threads - 1ull) / threads);
    const std::size_t smem = static_cast<std::size_t>(g.groups) * 2 * g.group * VEC * sizeof(float);
    scaled_embedding_sum_kernel<T, VEC><<<g.ctas + zero_ctas, threads, smem, s>>>(static_cast<T*>(dw), static_cast<const T*>(dout), g, args);
    count_launch();
    CGPT_LAUNCH_CHECK();
    if (g.ctas == 1) return CGPT_OK;
    constexpr int JV = VEC < 4 ? 1 : 4;
    const unsigned column_tiles = static_cast<unsigned>((g.hidden + 32 * JV - 1) / (32 * JV));
    const unsigned runs = g.ctas - 1, lanes = column_tiles < kNumSMs * 8u ? kNumSMs * 8u / column_tiles : 1;   // runs at a time
    scaled_embedding_join_kernel<T, JV><<<column_tiles * (runs < lanes ? runs : lanes), kJoinThreads, 0, s>>>(static_cast<T*>(dw), g);
    count_launch();
    CGPT_LAUNCH_CHECK();
    return CGPT_OK;
}

constexpr std::size_t kClusterTokens = std::size_t{8} * kMaxCluster * kClusterThreads;

// One launch of one cluster, up to kClusterTokens tokens.
int launch_cluster_sort(const ClusterSort& p, cudaStream_t s) {
    int ctas = 1;
    while (ctas < kMaxCluster && ctas * kClusterThreads < p.n) ctas *= 2;
    const int keys = (p.n + ctas * kClusterThreads - 1) / (ctas * kClusterThreads);
    auto kernel = keys == 1 ? sort_cluster_kernel<1> : keys == 2 ? sort_cluster_kernel<2> : keys <= 4 ? sort_cluster_kernel<4> : sort_cluster_kernel<8>;
    static PerDeviceOnce once[4];
    PerDeviceOnce& o = once[keys == 1 ? 0 : keys == 2 ? 1 : keys <= 4 ? 2 : 3];
    if (o.needed()) {
        CGPT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        o.done();
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(ctas);
    config.blockDim = dim3(kClusterThreads);
    config.stream = s;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = ctas;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    CGPT_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, p));
    count_launch();
    return CGPT_OK;
}

}  // namespace
}  // namespace cgpt

using namespace cgpt;

extern "C" int cgpt_scaled_embedding_forward(void* out, const uint32_t* ids, const void* weight, size_t tokens, size_t vocab,
                                             size_t hidden, float scale, float probability, const uint64_t* state, uint32_t site,
                                             int dtype, cgpt_stream_t stream) {
    if (!out || !ids || !weight) return CGPT_ERR_NULL;
    if (!valid_float_dtype(dtype)) return CGPT_ERR_DTYPE;
    if (!valid_sizes(tokens, vocab, hidden)) return CGPT_ERR_SHAPE;
    if (!std::isfinite(scale)) return CGPT_ERR_OPTION;
    if (!element_aligned(dtype, {out, weight}) || !element_aligned(CGPT_DTYPE_F32, {ids})) return CGPT_ERR_ALIGN;
    DropoutArgs args;
    CGPT_TRY(dropout_args(&args, probability, state, site, tokens * hidden));
    auto s = static_cast<cudaStream_t>(stream);
    CGPT_DISPATCH_DTYPE(dtype, T, {
        constexpr int V = 16 / sizeof(T);
        const bool vector = hidden % V == 0 && aligned16(out) && aligned16(weight);
        auto kernel = vector ? scaled_embedding_forward_kernel<T, V> : scaled_embedding_forward_kernel<T, 1>;
        const int group = group_for(hidden, vector ? V : 1);
        const std::size_t per_cta = static_cast<std::size_t>(kThreads / group) * kLookups, need = (tokens + per_cta - 1) / per_cta;
        kernel<<<static_cast<unsigned>(need), kThreads, 0, s>>>(
            static_cast<T*>(out), ids, static_cast<const T*>(weight), static_cast<long long>(tokens), static_cast<std::uint32_t>(vocab),
            static_cast<int>(hidden), scale, group, args);
        count_launch();
        CGPT_LAUNCH_CHECK();
    });
    return CGPT_OK;
}

extern "C" size_t cgpt_scaled_embedding_backward_workspace_bytes(size_t tokens, size_t hidden) {
    return valid_sizes(tokens, 1, hidden) ? Layout(tokens, hidden).bytes : 0;
}

extern "C" int cgpt_scaled_embedding_backward(void* grad_weight, const void* grad_output, const uint32_t* ids, void* workspace,
                                              size_t workspace_size, size_t tokens, size_t vocab, size_t hidden, float scale,
                                              uint32_t padding_id, float probability, const uint64_t* state, uint32_t site,
                                              int accumulate, int dtype, cgpt_stream_t stream) {
    if (!grad_weight || !grad_output || !ids || !workspace) return CGPT_ERR_NULL;
    if (!valid_float_dtype(dtype)) return CGPT_ERR_DTYPE;
    if (!valid_sizes(tokens, vocab, hidden)) return CGPT_ERR_SHAPE;
    const Layout at(tokens, hidden);
    if (workspace_size < at.bytes) return CGPT_ERR_SHAPE;
    if (!std::isfinite(scale) || grad_weight == grad_output) return CGPT_ERR_OPTION;
    if (!element_aligned(dtype, {grad_weight, grad_output}) || !element_aligned(CGPT_DTYPE_F32, {ids}) || !aligned16(workspace)) return CGPT_ERR_ALIGN;
    DropoutArgs args;
    CGPT_TRY(dropout_args(&args, probability, state, site, tokens * hidden));
    auto s = static_cast<cudaStream_t>(stream);
    auto* base = static_cast<unsigned char*>(workspace);
    auto words = [&](std::size_t offset) { return reinterpret_cast<std::uint32_t*>(base + offset); };

    const int bits = bit_length(vocab);   // keys are in [0, vocab]
    const int passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    const int digit_bits = (bits + passes - 1) / passes;
    ClusterSort c{ids, {words(at.keys[0]), words(at.keys[1])}, {words(at.vals[0]), words(at.vals[1])}, words(at.crossing),
                  static_cast<int>(tokens), digit_bits, passes, static_cast<std::uint32_t>(vocab), padding_id};
    if (tokens <= kClusterTokens) {
        CGPT_TRY(launch_cluster_sort(c, s));
    } else {
        SortPass p{};
        p.counts = words(at.counts);
        p.totals = words(at.totals);
        p.crossing = c.crossing;
        p.n = static_cast<long long>(tokens);
        p.vocab = c.vocab;
        p.skip_id = padding_id;
        p.bits = digit_bits;
        p.tiles = at.tiles;
        p.keys_in = ids;
        for (int i = 0; i < passes; ++i) {
            p.shift = i * p.bits;
            p.keys_out = c.keys[i & 1];
            p.vals_out = c.vals[i & 1];
            sort_count_kernel<<<at.tiles, kSortThreads, 0, s>>>(p);
            CGPT_LAUNCH_CHECK();
            sort_prefix_kernel<<<1 << p.bits, kSortThreads, 0, s>>>(p);
            CGPT_LAUNCH_CHECK();
            sort_scatter_kernel<<<at.tiles, kSortThreads, 0, s>>>(p);
            CGPT_LAUNCH_CHECK();
            count_launch(3);
            p.keys_in = p.keys_out;
            p.vals_in = p.vals_out;
        }
    }
    const int last = (passes - 1) & 1;
    const GradArgs g{c.keys[last], c.vals[last], reinterpret_cast<float*>(base + at.partial), c.crossing, static_cast<long long>(tokens),
                     static_cast<long long>(hidden), c.vocab, 0, accumulate, 0, 0, scale};
    CGPT_DISPATCH_DTYPE(dtype, T, {
        constexpr int V = 16 / sizeof(T);
        if (hidden % V == 0 && aligned16(grad_weight) && aligned16(grad_output)) return (launch_sum<T, V>(grad_weight, grad_output, g, args, s));
        return (launch_sum<T, 1>(grad_weight, grad_output, g, args, s));
    });
    return CGPT_OK;
}
