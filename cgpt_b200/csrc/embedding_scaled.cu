// Scaled embedding lookup with dropout, and its gradient, for sm_100a.
//
//   forward    out[t] = dropout(scale * W[ids[t]])             (an id outside the table gives a zero row)
//   backward   dW[v] (+)= scale * sum_{t: ids[t] = v} drop(dout[t])     ids equal to padding_id or outside the table are skipped
//
// Backward. Token ids follow word frequencies: one id can hold a twentieth of all tokens (or, in a padded batch, most of
// them), so one owner per table row would leave one CTA adding thousands of rows. Here the tokens are sorted by id (stable
// radix sort, this file) and the SORTED list is cut into chunks of kChunk tokens, one group of threads each: a chunk adds its
// tokens' rows run by run; a run inside the chunk is written to the table at once, a run that crosses a chunk border leaves an
// fp32 partial row, and a second kernel adds the partial rows of such runs. Every sum is taken in an order that follows from
// the ids alone, so results repeat bit for bit, and no run is longer than kChunk rows for any one group.
// Table rows without a token are zeroed by the same launch (their owners look the row up in the sorted list), so the table
// is written once.
//
// Memory-bound: backward reads dout once and writes the table once; the sort moves 16 bytes per token and pass.
#include "philox.cuh"
#include "launch_counter.h"

namespace cgpt {
namespace {

constexpr int kThreads = 128;        // lookup and chunk sums
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kKeysPerThread = 8;
constexpr int kSortTile = kSortThreads * kKeysPerThread;
constexpr int kMaxDigitBits = 9;
constexpr int kChunk = 32;           // sorted tokens per chunk

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
scaled_embedding_forward_kernel(T* __restrict__ out, const std::uint32_t* __restrict__ ids, const T* __restrict__ weight,
                                long long tokens, std::uint32_t vocab, long long hidden, float scale, int group,
                                const DropoutArgs args) {
    const Philox gen(args);
    const int lane = threadIdx.x % group;
    const long long groups = static_cast<long long>(gridDim.x) * (kThreads / group);
    for (long long t = static_cast<long long>(blockIdx.x) * (kThreads / group) + threadIdx.x / group; t < tokens; t += groups) {
        const std::uint32_t id = ids[t];
        for (long long c = static_cast<long long>(lane) * VEC; c < hidden; c += static_cast<long long>(group) * VEC) {
            float v[VEC];
            if (id < vocab) {
                load_vec<T, VEC>(v, weight + static_cast<long long>(id) * hidden + c);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] *= scale;
                if (args.threshold != 0) drop_vec<VEC>(v, gen, t * hidden + c, args);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] = 0.f;
            }
            store_vec<T, VEC>(out + t * hidden + c, v);
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

// ------------------------------------------------------------------------------------------------- chunk sums
struct GradArgs {
    const std::uint32_t* ids;        // sorted; `vocab` marks skipped tokens
    const std::uint32_t* tokens;     // the token of each sorted position
    float* partial;                  // [chunks][2][hidden]: a run's part that began in an earlier chunk, or goes on in the next one
    std::uint32_t* crossing;         // [0]: count, [1..]: chunks in which a run starts that goes on in the next chunk
    long long n, hidden;
    std::uint32_t vocab;
    int chunks, accumulate;
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

// CTAs [0, chunk_ctas): `kThreads / group` chunks each. The others zero the table rows that no token has, 32 rows per warp.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
scaled_embedding_sum_kernel(T* dw, const T* __restrict__ dout, const GradArgs g, int group, unsigned chunk_ctas, const DropoutArgs args) {
    if (blockIdx.x >= chunk_ctas) {
        const int lane = threadIdx.x & 31;
        const long long first = (static_cast<long long>(blockIdx.x - chunk_ctas) * (kThreads / 32) + (threadIdx.x >> 5)) * 32;
        const long long row = first + lane;
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
            for (long long c = static_cast<long long>(lane) * VEC; c < g.hidden; c += 32 * VEC) store_vec<T, VEC>(dw + (first + r) * g.hidden + c, zero);
        }
        return;
    }
    const Philox gen(args);
    const int lane = threadIdx.x % group;
    const long long chunk = static_cast<long long>(blockIdx.x) * (kThreads / group) + threadIdx.x / group;
    if (chunk >= g.chunks) return;
    const long long lo = chunk * kChunk, hi = lo + kChunk < g.n ? lo + kChunk : g.n;
    const std::uint32_t first_id = g.ids[lo], last_id = g.ids[hi - 1];
    const bool from_before = lo > 0 && g.ids[lo - 1] == first_id;
    const bool goes_on = hi < g.n && g.ids[hi] == last_id;
    if (lane == 0 && goes_on && last_id < g.vocab && !(from_before && first_id == last_id))
        g.crossing[1 + atomicAdd(g.crossing, 1u)] = static_cast<std::uint32_t>(chunk);   // their order changes no result
    for (long long c = static_cast<long long>(lane) * VEC; c < g.hidden; c += static_cast<long long>(group) * VEC) {
        float acc[VEC] = {};
        std::uint32_t id = first_id;
        bool before = from_before;
        for (long long p = lo; p < hi; ++p) {
            const std::uint32_t next = g.ids[p];
            if (next >= g.vocab) break;               // skipped tokens are last
            if (next != id) {
                if (before) store_vec<float, VEC>(g.partial + (chunk * 2) * g.hidden + c, acc);
                else write_row<T, VEC>(dw + static_cast<long long>(id) * g.hidden + c, acc, g.scale, g.accumulate);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
                id = next;
                before = false;
            }
            const long long e = static_cast<long long>(g.tokens[p]) * g.hidden + c;
            float v[VEC];
            load_vec_stream<T, VEC>(v, dout + e);
            if (args.threshold != 0) drop_vec<VEC>(v, gen, e, args);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += v[i];
        }
        if (id >= g.vocab) continue;
        if (before) store_vec<float, VEC>(g.partial + (chunk * 2) * g.hidden + c, acc);
        else if (goes_on && id == last_id) store_vec<float, VEC>(g.partial + (chunk * 2 + 1) * g.hidden + c, acc);
        else write_row<T, VEC>(dw + static_cast<long long>(id) * g.hidden + c, acc, g.scale, g.accumulate);
    }
}

// Runs that cross chunk borders: the part of the chunk they start in and those of all later chunks they reach, 32 columns
// and 32 part lanes per CTA; a (run, column tile) pair per trip.
template <typename T>
__global__ void __launch_bounds__(1024)
scaled_embedding_join_kernel(T* dw, const GradArgs g) {
    __shared__ float tile[32][33];
    const int lane = threadIdx.x & 31, pl = threadIdx.x >> 5;
    const long long column_tiles = (g.hidden + 31) / 32;
    const long long items = *g.crossing * column_tiles;
    for (long long it = blockIdx.x; it < items; it += gridDim.x) {
        const long long chunk = g.crossing[1 + it / column_tiles];
        const long long col = (it % column_tiles) * 32 + lane;
        const std::uint32_t id = g.ids[chunk * kChunk + kChunk - 1];
        // last chunk whose first token belongs to the run
        long long lo = chunk + 1, hi = g.chunks - 1;
        while (lo < hi) {
            const long long mid = (lo + hi + 1) >> 1;
            if (g.ids[mid * kChunk] == id) lo = mid;
            else hi = mid - 1;
        }
        float acc = 0.f;
        if (col < g.hidden)
            for (long long k = chunk + pl; k <= lo; k += 32) acc += g.partial[(k * 2 + (k == chunk ? 1 : 0)) * g.hidden + col];
        tile[pl][lane] = acc;
        __syncthreads();
        if (pl == 0 && col < g.hidden) {
            float t[1] = {0.f};
#pragma unroll
            for (int r = 0; r < 32; ++r) t[0] += tile[r][lane];
            write_row<T, 1>(dw + static_cast<long long>(id) * g.hidden + col, t, g.scale, g.accumulate);
        }
        __syncthreads();
    }
}

int bit_length(std::uint64_t v) {
    int b = 0;
    while (v) { ++b; v >>= 1; }
    return b;
}

// Byte offsets of the workspace's parts.
struct Layout {
    std::size_t keys[2], vals[2], counts, totals, crossing, partial, bytes;
    int tiles, chunks;
    Layout(std::size_t tokens, std::size_t hidden) {
        tiles = static_cast<int>((tokens + kSortTile - 1) / kSortTile);
        chunks = static_cast<int>((tokens + kChunk - 1) / kChunk);
        bytes = 0;
        auto take = [&](std::size_t n) {
            const std::size_t at = bytes;
            bytes += (n + 255) & ~std::size_t{255};
            return at;
        };
        for (int i = 0; i < 2; ++i) { keys[i] = take(tokens * 4); vals[i] = take(tokens * 4); }
        counts = take((std::size_t{4} << kMaxDigitBits) * tiles);
        totals = take(std::size_t{4} << kMaxDigitBits);
        crossing = take(4 * (static_cast<std::size_t>(chunks) + 1));
        partial = take(static_cast<std::size_t>(chunks) * 2 * hidden * sizeof(float));
    }
};

// Threads per row: enough for the row's vectors, at most a CTA.
int group_for(std::size_t hidden, int vec) {
    int g = 1;
    while (g < kThreads && static_cast<std::size_t>(g) * vec < hidden) g *= 2;
    return g;
}

bool valid_sizes(std::size_t tokens, std::size_t vocab, std::size_t hidden) {
    return tokens != 0 && vocab != 0 && hidden != 0 && tokens <= 0x7fffffffull && vocab <= 0x7ffffffeull && hidden <= 0x7fffffffull &&
           tokens <= (1ull << 46) / hidden && vocab <= (1ull << 46) / hidden;
}

template <typename T, int VEC>
int launch_sum(void* dw, const void* dout, const GradArgs& g, const DropoutArgs& args, cudaStream_t s) {
    const int group = group_for(static_cast<std::size_t>(g.hidden), VEC);
    const unsigned per_cta = kThreads / group;
    const unsigned chunk_ctas = (g.chunks + per_cta - 1) / per_cta;
    const unsigned zero_ctas = g.accumulate ? 0 : static_cast<unsigned>((g.vocab + kThreads - 1ull) / kThreads);
    scaled_embedding_sum_kernel<T, VEC><<<chunk_ctas + zero_ctas, kThreads, 0, s>>>(static_cast<T*>(dw), static_cast<const T*>(dout), g, group,
                                                                                   chunk_ctas, args);
    count_launch();
    CGPT_LAUNCH_CHECK();
    const unsigned cap = static_cast<unsigned>(kNumSMs) * 2;
    const unsigned long long most = static_cast<unsigned long long>(g.chunks) * ((g.hidden + 31) / 32);
    scaled_embedding_join_kernel<T><<<static_cast<unsigned>(most < cap ? most : cap), 1024, 0, s>>>(static_cast<T*>(dw), g);
    count_launch();
    CGPT_LAUNCH_CHECK();
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
        const std::size_t per_cta = kThreads / group, need = (tokens + per_cta - 1) / per_cta;
        const std::size_t cap = static_cast<std::size_t>(kNumSMs) * resident_ctas_per_sm(reinterpret_cast<const void*>(kernel), kThreads, 0);
        kernel<<<static_cast<unsigned>(need < cap ? need : cap), kThreads, 0, s>>>(
            static_cast<T*>(out), ids, static_cast<const T*>(weight), static_cast<long long>(tokens), static_cast<std::uint32_t>(vocab),
            static_cast<long long>(hidden), scale, group, args);
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
    SortPass p{};
    p.counts = words(at.counts);
    p.totals = words(at.totals);
    p.crossing = words(at.crossing);
    p.n = static_cast<long long>(tokens);
    p.vocab = static_cast<std::uint32_t>(vocab);
    p.skip_id = padding_id;
    p.bits = (bits + passes - 1) / passes;
    p.tiles = at.tiles;
    p.keys_in = ids;
    for (int i = 0; i < passes; ++i) {
        p.shift = i * p.bits;
        p.keys_out = words(at.keys[i & 1]);
        p.vals_out = words(at.vals[i & 1]);
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
    const GradArgs g{p.keys_in, p.vals_in, reinterpret_cast<float*>(base + at.partial), p.crossing, p.n, static_cast<long long>(hidden),
                     p.vocab, at.chunks, accumulate, scale};
    CGPT_DISPATCH_DTYPE(dtype, T, {
        constexpr int V = 16 / sizeof(T);
        if (hidden % V == 0 && aligned16(grad_weight) && aligned16(grad_output)) return (launch_sum<T, V>(grad_weight, grad_output, g, args, s));
        return (launch_sum<T, 1>(grad_weight, grad_output, g, args, s));
    });
    return CGPT_OK;
}
