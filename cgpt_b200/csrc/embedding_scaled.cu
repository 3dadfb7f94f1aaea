// Scaled embedding lookup with dropout, and its gradient, for sm_100a.
//
//   forward    out[t] = dropout(scale * W[ids[t]])             (an id outside the table gives a zero row)
//   backward   dW[v] (+)= scale * sum_{t: ids[t] = v} drop(dout[t])     ids equal to padding_id or outside the table are skipped
//
// Backward. Token ids follow word frequencies: one id can hold a twentieth of all tokens (or, in a padded batch, most of
// them), so one owner per table row would leave one CTA adding thousands of rows. Here the tokens are sorted by id (stable
// radix sort, this file) and the SORTED list is cut into chunks of as many tokens, one group of threads each: a group adds its
// tokens' rows run by run, several rows in flight. A run inside a chunk is written to the table at once; runs that cross chunks
// are joined in shared memory within a CTA, and a run that crosses CTAs leaves fp32 partial rows that a last kernel adds. Every
// sum is taken in an order that follows from the ids alone, so results repeat bit for bit, and no group has more rows than others.
// The sort takes one cluster of at most 16 SMs and is all latency; the others clear the table meanwhile (65 MB take 20 us, memory
// takes 3.5 TB/s of writes alone). Rows with tokens are then written twice. Zeroing only the other rows, from a bitmap that the
// sort fills, while gradient rows are read, was measured slower (51 against 48 us at 32768 tokens, 32000 x 1024 bf16: the hot
// words of the bitmap cost the sort more than it saves).
//
// Backward reads dout once and writes the table once; the sort moves 16 bytes per token and pass.
// 32768 tokens, 32000 x 1024 bf16: 47 us, with dropout 58: sort and clearing 20, the rest the sums, in which the decisions make the
// difference. Added to the table 45 and 57 (nothing is cleared, rows are read). 131072 tokens, sorted by launches per digit: 160 us.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "dependent_launch.cuh"
#include "philox.cuh"
#include "launch_counter.h"

namespace cgpt {
namespace {

constexpr int kThreads = 128;        // lookup; threads per row at most
constexpr int kSumThreads = 512;
constexpr int kMostChunk = 32;       // sorted tokens per group of threads at most
constexpr int kMostGroups = 8;       // groups per CTA at most
constexpr int kInFlight = 4;         // rows a group loads before it adds them
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kKeysPerThread = 8;
constexpr int kSortTile = kSortThreads * kKeysPerThread;
constexpr int kMaxDigitBits = 9;
constexpr int kClusterThreads = 1024;
constexpr int kMaxCluster = 16;
constexpr int kMostKeys = 4;         // keys per thread of the cluster sort

// kLookups consecutive tokens per group of 2^shift threads and trip: their ids, then their rows, are loaded together. 32768 tokens of
// 32000 x 1024 bf16 take 27.2 us, 3.1 TB/s of what has to move; 18.4 without dropout. No unit is full (integer pipe 61 %, 0.60
// instructions per scheduler and cycle): ids, rows, the decisions (15 instructions an element) and stores of a trip follow one another.
constexpr int kLookups = 4;
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
scaled_embedding_forward_kernel(T* __restrict__ out, const std::uint32_t* __restrict__ ids, const T* __restrict__ weight,
                                long long tokens, std::uint32_t vocab, int hidden, float scale, int shift, const DropoutArgs args) {
    using Raw = typename RawVec<sizeof(T) * VEC>::type;
    const HoistedPhilox gen(args);
    const float factor = scale * args.scale;
    const int group = 1 << shift, lane = threadIdx.x & (group - 1);
    const long long step = static_cast<long long>(gridDim.x) * (kThreads >> shift) * kLookups;
    // trips are uniform over a warp: its lanes share their decisions where a vector is one element
    const long long first = (static_cast<long long>(blockIdx.x) * (kThreads >> shift) + (threadIdx.x >> shift)) * kLookups;
    const long long warp_first = (static_cast<long long>(blockIdx.x) * (kThreads >> shift) + ((threadIdx.x & ~31u) >> shift)) * kLookups;
    for (long long w0 = warp_first, t0 = first; w0 < tokens; w0 += step, t0 += step) {
        std::uint32_t id[kLookups];
#pragma unroll
        for (int k = 0; k < kLookups; ++k) id[k] = t0 + k < tokens ? ids[t0 + k] : 0xffffffffu;
        for (int c0 = 0; c0 < hidden; c0 += group * VEC) {
            const int c = c0 + lane * VEC;
            const bool in = c < hidden;
            Raw row[kLookups];
#pragma unroll
            for (int k = 0; k < kLookups; ++k) {
                row[k] = Raw{};                               // an id outside the table gives zeros
                if (in && id[k] < vocab) row[k] = *reinterpret_cast<const Raw*>(weight + static_cast<long long>(id[k]) * hidden + c);
            }
            T* to = out + t0 * hidden + c;
            if constexpr (VEC > 1) {
#pragma unroll
                for (int k = 0; k < kLookups; ++k) {
                    if (in && t0 + k < tokens) {
                        Pair v[VEC / 2];
                        to_pairs<T>(v, row[k]);
                        if (args.threshold != 0) drop_pairs<VEC / 2, false>(v, gen, (t0 + k) * hidden + c, args);
#pragma unroll
                        for (int i = 0; i < VEC / 2; ++i) v[i] = mul2(v[i], pair(factor));
                        *reinterpret_cast<uint4*>(to + static_cast<long long>(k) * hidden) = to_raw<T>(v);
                    }
                }
            } else {
                std::uint32_t kept = 15u;
                if (args.threshold != 0 && shift >= 5) {
                    long long start[kLookups];
#pragma unroll
                    for (int k = 0; k < kLookups; ++k) start[k] = (t0 + k) * hidden + c - static_cast<int>(threadIdx.x & 31);
                    kept = keep_four_runs(start, gen, args.threshold);
                }
#pragma unroll
                for (int k = 0; k < kLookups; ++k) {
                    if (in && t0 + k < tokens) {
                        float v = to_f32<T>(*reinterpret_cast<const T*>(&row[k])) * factor;
                        if (args.threshold != 0) v = shift >= 5 ? ((kept >> k) & 1u ? v : 0.f) : apply_one<false>(v, gen, (t0 + k) * hidden + c, args);
                        to[static_cast<long long>(k) * hidden] = from_f32<T>(v);
                    }
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
    std::uint32_t* crossing;         // [0]: number of runs that cross a CTA border; cleared by the first pass
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

// Lanes of the warp that are `in` and have this lane's digit: one vote per bit of the digit, whatever the digits are (a match
// instruction takes as long as there are different values in the warp, six times as long for the low digit of token ids).
__device__ __forceinline__ unsigned same_digit(std::uint32_t digit, bool in, int bits) {
    unsigned peers = __ballot_sync(0xffffffffu, in);
#pragma unroll
    for (int b = 0; b < kMaxDigitBits; ++b) {
        const unsigned set = __ballot_sync(0xffffffffu, (digit >> b) & 1u);
        if (b < bits) peers &= (digit >> b) & 1u ? set : ~set;
    }
    return peers;
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
        const std::uint32_t digit = (key[j] >> p.shift) & (radix - 1);
        const unsigned peers = same_digit(digit, in, p.bits);
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

// The whole sort in one launch, for up to kMaxCluster * kClusterThreads * KEYS tokens: the CTAs of one cluster hold a share of the
// keys each. Digit counts and, between passes, keys go round in distributed shared memory; only the last pass writes to global
// memory. A pass is then two cluster barriers instead of three launches. The other clusters of the launch clear memory. (Four keys a
// thread spill 32 bytes.)
struct ClusterSort {
    uint4* clear;                       // memory that the other clusters set to zero
    long long clear_vectors;            // 16-byte vectors of it; `clear_tail` bytes more behind them
    int clear_tail;
    const std::uint32_t* ids;
    std::uint32_t *keys, *vals, *crossing;
    int n, bits, passes;
    std::uint32_t vocab, skip_id;
};

template <int KEYS>
struct alignas(16) ClusterSmem {
    static constexpr int kWarps = kClusterThreads / 32, kShare = kClusterThreads * KEYS;   // keys per CTA
    std::uint32_t key[kShare], val[kShare];                  // the CTA's share in the order of the last pass; written by the whole cluster
    std::uint32_t mine[1 << kMaxDigitBits];                  // the CTA's keys of each digit; read by the whole cluster
    std::uint32_t base[1 << kMaxDigitBits];
    std::uint32_t warp_total[kWarps];
    alignas(16) unsigned short seen[kWarps][1 << kMaxDigitBits];   // keys of a digit met so far by each warp, then those of earlier warps
    unsigned short sums[kClusterThreads];                    // [share of the warps][digit]
};

template <int KEYS>
__global__ void __launch_bounds__(kClusterThreads)
sort_cluster_kernel(const ClusterSort p) {
    extern __shared__ __align__(16) unsigned char cluster_smem[];
    using Smem = ClusterSmem<KEYS>;
    Smem& sm = *reinterpret_cast<Smem*>(cluster_smem);
    constexpr int kWarps = Smem::kWarps;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    launch_dependents();
    if (blockIdx.x >= cluster.num_blocks()) {
        const long long workers = static_cast<long long>(gridDim.x - cluster.num_blocks()) * kClusterThreads;
        long long i = static_cast<long long>(blockIdx.x - cluster.num_blocks()) * kClusterThreads + threadIdx.x;
        if (i < p.clear_tail) reinterpret_cast<unsigned char*>(p.clear + p.clear_vectors)[i] = 0;
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        for (; i + 7 * workers < p.clear_vectors; i += 8 * workers) {
#pragma unroll
            for (int k = 0; k < 8; ++k) p.clear[i + k * workers] = zero;
        }
        for (; i < p.clear_vectors; i += workers) p.clear[i] = zero;
        return;
    }
    const int ctas = static_cast<int>(cluster.num_blocks()), cta = static_cast<int>(cluster.block_rank());
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int radix = 1 << p.bits;
    const int local = warp * (32 * KEYS) + lane, first = cta * Smem::kShare + local;   // order of the keys: (CTA, warp, j, lane)
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
        for (int d = lane; d < radix / 8; d += 32) reinterpret_cast<uint4*>(sm.seen[warp])[d] = make_uint4(0u, 0u, 0u, 0u);
        if (radix < 8 && lane < radix) sm.seen[warp][lane] = 0;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
            const bool in = first + j * 32 < p.n;
            const std::uint32_t digit = (key[j] >> shift) & (radix - 1);
            const unsigned peers = same_digit(digit, in, p.bits);
            const unsigned below = __popc(peers & ((1u << lane) - 1u));
            const std::uint32_t so_far = in ? sm.seen[warp][digit] : 0u;
            rank[j] = so_far + below;
            __syncwarp();
            if (in && below == 0) sm.seen[warp][digit] = static_cast<unsigned short>(so_far + __popc(peers));
            __syncwarp();
        }
        __syncthreads();
        // Counts of the warps before each warp: kClusterThreads / radix threads per digit take a share of the warps each.
        const int digit_of = threadIdx.x & (radix - 1), part = threadIdx.x >> p.bits, parts = kClusterThreads >> p.bits;
        const int share = parts < kWarps ? kWarps / parts : 1;
        if (part < kWarps) {
            std::uint32_t before = 0;
            for (int w = part * share; w < (part + 1) * share; ++w) {
                const std::uint32_t here = sm.seen[w][digit_of];
                sm.seen[w][digit_of] = static_cast<unsigned short>(before);
                before += here;
            }
            sm.sums[part * radix + digit_of] = static_cast<unsigned short>(before);
        }
        __syncthreads();
        if (part < kWarps) {
            std::uint32_t before = 0;
            for (int k = 0; k < part; ++k) before += sm.sums[k * radix + digit_of];
            if (before != 0)
                for (int w = part * share; w < (part + 1) * share; ++w) sm.seen[w][digit_of] = static_cast<unsigned short>(sm.seen[w][digit_of] + before);
            if (part == (parts < kWarps ? parts : kWarps) - 1) sm.mine[digit_of] = before + sm.sums[part * radix + digit_of];
        }
        cluster.sync();
        // Digit d of this CTA starts behind all smaller digits and behind digit d of the CTAs before it.
        std::uint32_t all = 0, earlier = 0;
        if (threadIdx.x < radix) {
#pragma unroll
            for (int c = 0; c < kMaxCluster; ++c) {           // unrolled: the remote reads are on their way together
                const std::uint32_t v = c < ctas ? cluster.map_shared_rank(sm.mine, c)[threadIdx.x] : 0u;
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
        if (lane == 31) sm.warp_total[warp] = inc;
        __syncthreads();
        if (threadIdx.x < radix) {
            std::uint32_t smaller = 0;
            for (int w = 0; w < warp; ++w) smaller += sm.warp_total[w];
            sm.base[threadIdx.x] = smaller + inc - all + earlier;
        }
        __syncthreads();
        const bool last = pass + 1 == p.passes;
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
            if (first + j * 32 < p.n) {
                const std::uint32_t digit = (key[j] >> shift) & (radix - 1), to = sm.base[digit] + sm.seen[warp][digit] + rank[j];
                if (last) {
                    p.keys[to] = key[j];
                    p.vals[to] = val[j];
                } else {
                    Smem* there = cluster.map_shared_rank(&sm, to / Smem::kShare);
                    there->key[to % Smem::kShare] = key[j];
                    there->val[to % Smem::kShare] = val[j];
                }
            }
        }
        // The keys of this pass have arrived, the counts have been read; after the last pass nobody is still being read from.
        cluster.sync();
        if (!last) {
#pragma unroll
            for (int j = 0; j < KEYS; ++j) {
                key[j] = sm.key[local + j * 32];
                val[j] = sm.val[local + j * 32];
            }
        }
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
    int ctas, accumulate;
    int shift, groups, chunk;        // 2^shift threads per row, groups per CTA, tokens per group
    float scale;                     // of the lookup times that of kept elements
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

// g.groups chunks of g.chunk sorted tokens per CTA. Two CTAs per SM leave 64 registers, of which the round keys take 16: 16-bit vectors
// spill 48 bytes a thread.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads, 2)
scaled_embedding_sum_kernel(T* dw, const T* __restrict__ dout, const GradArgs g, const DropoutArgs args) {
    extern __shared__ __align__(16) float parts[];           // [threads / per_row][2][per_row * VEC]: what a chunk's first and last run leave
    const int per_row = 1 << g.shift, lane = threadIdx.x & (per_row - 1), group = threadIdx.x >> g.shift;
    const int span = g.groups * g.chunk;
    std::uint32_t* ids = reinterpret_cast<std::uint32_t*>(parts + 2 * VEC * blockDim.x);   // [4 + span + 4]
    std::uint32_t* tokens = ids + span + 8;                                                 // [span]
    const HoistedPhilox gen(args);
    launch_dependents();
    wait_for_previous();
    // The CTA's ids and the ones before and behind them; what is not there counts as skipped (id `vocab`, token 0).
    const long long lo = static_cast<long long>(blockIdx.x) * span;
    const int count = g.n - lo < span ? static_cast<int>(g.n - lo) : span;
    for (int i = static_cast<int>(threadIdx.x) - 1; i < span + 1; i += blockDim.x) {
        const long long at = lo + i;
        ids[4 + i] = at >= 0 && at < g.n ? g.ids[at] : g.vocab;
        if (i >= 0 && i < span) tokens[i] = at < g.n ? g.tokens[at] : 0u;
    }
    __syncthreads();
    const std::uint32_t* id_at = ids + 4;                     // id_at[-1] .. id_at[span]
    const bool first_from_before = id_at[-1] == id_at[0], last_goes_on = id_at[count] == id_at[count - 1];
    const bool single = id_at[0] == id_at[count - 1];         // all of the CTA's tokens have one id
    if (threadIdx.x == 0 && last_goes_on && id_at[count - 1] < g.vocab && !(single && first_from_before))
        g.crossing[1 + atomicAdd(g.crossing, 1u)] = blockIdx.x;   // their order changes no result
    float* before = g.partial + static_cast<long long>(blockIdx.x) * 2 * g.hidden;
    float* after = before + g.hidden;
    const int width = per_row * VEC;
    float* head = parts + group * 2 * width + lane * VEC;
    float* tail = head + width;
    const int begin = group * g.chunk, end = begin + g.chunk;
    for (long long c0 = 0; c0 < g.hidden; c0 += width) {
        const long long c = c0 + lane * VEC;
        const bool in = c < g.hidden;
        float acc[VEC] = {};
        const bool works = begin < span;                      // threads beyond the groups only join in with the warp
        std::uint32_t id = works ? id_at[begin] : g.vocab;
        bool open = works && id_at[begin - 1] == id;          // the run began in an earlier chunk
        for (int p0 = begin; p0 < begin + g.chunk; p0 += kInFlight) {
            using Raw = typename RawVec<sizeof(T) * VEC>::type;
            const uint4 at4 = works ? *reinterpret_cast<const uint4*>(id_at + p0) : make_uint4(g.vocab, g.vocab, g.vocab, g.vocab);
            const uint4 token4 = works ? *reinterpret_cast<const uint4*>(tokens + p0) : make_uint4(0u, 0u, 0u, 0u);
            const std::uint32_t at[kInFlight] = {at4.x, at4.y, at4.z, at4.w}, token[kInFlight] = {token4.x, token4.y, token4.z, token4.w};
            Raw rows[kInFlight];
#pragma unroll
            for (int u = 0; u < kInFlight; ++u)               // without conditions: token 0 stands in past the end
                rows[u] = __ldcs(reinterpret_cast<const Raw*>(dout + static_cast<long long>(token[u]) * g.hidden + (in ? c : 0)));
            std::uint32_t kept = 15u;
            if constexpr (VEC == 1) {
                if (args.threshold != 0 && g.shift >= 5) {
                    long long start[kInFlight];
#pragma unroll
                    for (int u = 0; u < kInFlight; ++u) start[u] = static_cast<long long>(token[u]) * g.hidden + c - static_cast<int>(threadIdx.x & 31);
                    kept = keep_four_runs(start, gen, args.threshold);
                }
            }
#pragma unroll
            for (int u = 0; u < kInFlight; ++u) {
                if (at[u] != id) {                            // never from a skipped token: they are last
                    if (in && open) put_floats<VEC>(head, acc);
                    else if (in) write_row<T, VEC>(dw + static_cast<long long>(id) * g.hidden + c, acc, g.scale, g.accumulate);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
                    id = at[u];
                    open = false;
                }
                {                                             // skipped tokens are added to a sum that nobody writes
                    const long long e = static_cast<long long>(token[u]) * g.hidden + c;
                    if constexpr (VEC > 1) {
                        Pair v[VEC / 2];
                        to_pairs<T>(v, rows[u]);
                        if (args.threshold != 0) drop_pairs<VEC / 2, false>(v, gen, e, args);
#pragma unroll
                        for (int i = 0; i < VEC / 2; ++i) {
                            const float2 s = both(add2(pair(acc[2 * i], acc[2 * i + 1]), v[i]));
                            acc[2 * i] = s.x;
                            acc[2 * i + 1] = s.y;
                        }
                    } else {
                        float v = to_f32<T>(*reinterpret_cast<const T*>(&rows[u]));
                        if (args.threshold != 0) v = g.shift >= 5 ? ((kept >> u) & 1u ? v : 0.f) : apply_one<false>(v, gen, e, args);
                        acc[0] += v;
                    }
                }
            }
        }
        if (in && id < g.vocab) {
            if (open) put_floats<VEC>(head, acc);             // also where the whole chunk is one run that goes on
            else if (id_at[end] == id) put_floats<VEC>(tail, acc);
            else write_row<T, VEC>(dw + static_cast<long long>(id) * g.hidden + c, acc, g.scale, g.accumulate);
        }
        __syncthreads();
        // Runs that cross chunks: the threads of group 0 (more, where a group has few) walk over the CTA's chunks in order.
        for (int k = threadIdx.x; k < per_row; k += blockDim.x) {
            const long long col = c0 + k * VEC;
            if (col >= g.hidden) continue;
            float acc[VEC] = {};
            bool carried = false, from_before = false;
            for (int q = 0; q < g.groups; ++q) {
                const int b = q * g.chunk, e = b + g.chunk;
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
    __shared__ __align__(16) float tile[kJoinThreads / 32][32 * VEC];
    const int lane = threadIdx.x & 31, pl = threadIdx.x >> 5;
    wait_for_previous();
    const unsigned column_tiles = static_cast<unsigned>((g.hidden + 32 * VEC - 1) / (32 * VEC)), runs = *g.crossing;
    const long long span = static_cast<long long>(g.groups) * g.chunk;
    for (unsigned run = blockIdx.x / column_tiles; run < runs; run += gridDim.x / column_tiles) {
        const long long cta = g.crossing[1 + run];
        const long long col = (static_cast<long long>(blockIdx.x % column_tiles) * 32 + lane) * VEC;
        const std::uint32_t id = g.ids[cta * span + span - 1];
        // last CTA whose first token belongs to the run, looked for 32 CTAs at a time
        long long lo = cta;
        unsigned alike = 0xffffffffu;
        while (alike == 0xffffffffu) {
            alike = __ballot_sync(0xffffffffu, lo + 1 + lane < g.ctas && g.ids[(lo + 1 + lane) * span] == id);
            lo += alike == 0xffffffffu ? 32 : __ffs(~alike) - 1;
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

// ------------------------------------------------------------------------------------------------- few tokens
// One launch for few tokens and a small table: sort, sums and joins would be three, of a few microseconds of latency each. A
// CTA owns every gridDim.x-th row of the table (frequent ids are often neighbours) and a tile of columns. It picks the tokens of
// its rows out of all ids, in token order, zeroes its rows that have none, and adds up the others, a warp per row; rows with
// more than kFewOfRow tokens are shared out to all warps afterwards, each taking a part of the list (16 against 32: 11.7 | 13.4
// us for 777 tokens of 1000 x 250 f32, 14.8 | 17.0 for 512 of 1024 x 1024 bf16; 8 gives 12.4 and 14.8). The order of every sum
// follows from the ids alone.
// The rule (takes_few) by what was measured on both sides, us for one launch against the sort's three, dropout 0.1:
// vectors, 4 MB table: 1 token f32 1024 wide 8 | 12; 128 tokens f32 256 wide 10 | 14; 512 tokens bf16 1024 wide 17 | 19, f32
// 768 wide 16 | 21; 1024 tokens 22 | 18; 512 tokens and 8 MB 20 | 19; 32 MB 34 | 21 (rows cleared one by one).
// Single elements, 513 wide: 1024 tokens f32 4 MB 23 | 33, bf16 16 MB 27 | 33; 1 token, 16 MB 12 | 16. Vectors do best with
// a warp's width of columns per CTA (four: 33 instead of 27 for 1024 wide), single elements with four. The rule is by the table's size
// also where the gradient is added and nothing is cleared. Single elements of 16 bits spill 32 bytes a thread.
constexpr int kFewTokens = 1024, kFewOfRow = 16, kFewThreads = 512, kFewWarps = kFewThreads / 32;
constexpr unsigned kFewRows = 16384;     // rows of a CTA at most (a bit each)
static_assert(kFewOfRow <= 32, "a warp lists 32 tokens at a time");

struct FewArgs {
    const std::uint32_t* ids;
    int tokens, hidden, tile, accumulate;        // tile: columns per CTA
    std::uint32_t vocab, skip_id;
    float scale;
};

// Adds the rows of `count` listed tokens to acc, kInFlight at a time. Every lane of the warp takes part, whether it has columns
// (`in`) or not: single elements share their decisions.
template <typename T, int VEC, typename Generator>
__device__ __forceinline__ void add_rows(float (&acc)[VEC], const T* dout, const std::uint32_t* list, int count, int hidden, int c, bool in, const Generator& gen,
                                         const DropoutArgs& args) {
    using Raw = typename RawVec<sizeof(T) * VEC>::type;
    for (int k = 0; k < count; k += kInFlight) {
        Raw rows[kInFlight];
        long long e[kInFlight];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            e[u] = static_cast<long long>(list[k + u < count ? k + u : k]) * hidden + c;      // past the end: the first one again, not added
            rows[u] = *reinterpret_cast<const Raw*>(dout + (in ? e[u] : 0));
        }
        std::uint32_t kept = 15u;
        if constexpr (VEC == 1) {
            if (args.threshold != 0) {
                long long start[kInFlight];
#pragma unroll
                for (int u = 0; u < kInFlight; ++u) start[u] = e[u] - static_cast<int>(threadIdx.x & 31);
                kept = keep_four_runs(start, gen, args.threshold);
            }
        }
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            if (k + u < count) {
                if constexpr (VEC > 1) {
                    Pair v[VEC / 2];
                    to_pairs<T>(v, rows[u]);
                    if (args.threshold != 0) drop_pairs<VEC / 2, false>(v, gen, e[u], args);
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) {
                        const float2 f = both(v[i]);
                        acc[2 * i] += f.x;
                        acc[2 * i + 1] += f.y;
                    }
                } else if ((kept >> u) & 1u) {
                    acc[0] += to_f32<T>(*reinterpret_cast<const T*>(&rows[u]));
                }
            }
        }
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kFewThreads)
scaled_embedding_few_kernel(T* dw, const T* __restrict__ dout, const FewArgs f, const DropoutArgs args) {
    __shared__ std::uint32_t token[kFewTokens], row_of[kFewTokens];      // the tokens of this CTA's rows, in token order
    __shared__ std::uint32_t present[kFewRows / 32];
    __shared__ std::uint32_t heads[kFewTokens];                         // list positions at which a row is met first
    __shared__ std::uint32_t few[kFewWarps][32];                         // per warp: the tokens it adds up
    __shared__ int in_warp[kFewWarps], rows_listed;
    __shared__ __align__(16) float part[kFewWarps][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const std::uint32_t shares = gridDim.x, rows = (f.vocab - blockIdx.x + shares - 1) / shares;     // row r of the CTA: r * shares + blockIdx.x
    const int c_begin = blockIdx.y * f.tile, c_end = c_begin + f.tile < f.hidden ? c_begin + f.tile : f.hidden;
    const HoistedPhilox gen(args);
    for (unsigned i = threadIdx.x; i < (rows + 31) / 32; i += kFewThreads) present[i] = 0;
    if (threadIdx.x == 0) rows_listed = 0;
    __syncthreads();
    int so_far = 0;
    for (int t0 = 0; t0 < f.tokens; t0 += kFewThreads) {
        const int t = t0 + threadIdx.x;
        const std::uint32_t id = t < f.tokens ? f.ids[t] : 0xffffffffu;
        const std::uint32_t row = id / shares;
        const bool mine = t < f.tokens && id < f.vocab && id != f.skip_id && id - row * shares == blockIdx.x;
        const unsigned votes = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) in_warp[warp] = __popc(votes);
        __syncthreads();
        int at = so_far + __popc(votes & ((1u << lane) - 1u)), all = 0;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            at += w < warp ? in_warp[w] : 0;
            all += in_warp[w];
        }
        if (mine) {
            token[at] = t;
            row_of[at] = row;
            atomicOr(&present[row >> 5], 1u << (row & 31));
        }
        so_far += all;
        __syncthreads();
    }
    const int n = so_far;
    if (!f.accumulate) {
        const float zero[VEC] = {};
        for (unsigned word = warp; word < (rows + 31) / 32; word += kFewWarps) {
            unsigned todo = ~present[word];
            if (rows - word * 32 < 32) todo &= (1u << (rows - word * 32)) - 1u;
            while (todo != 0) {
                T* to = dw + (static_cast<long long>(word * 32 + __ffs(todo) - 1) * shares + blockIdx.x) * f.hidden;
                todo &= todo - 1;
                for (int c = c_begin + lane * VEC; c < c_end; c += 32 * VEC) store_vec<T, VEC>(to + c, zero);
            }
        }
    }
    for (int i = threadIdx.x; i < n; i += kFewThreads) {
        bool first = true;
        for (int j = 0; j < i && first; ++j) first = row_of[j] != row_of[i];
        if (first) heads[atomicAdd(&rows_listed, 1)] = i;                // their order changes no result
    }
    __syncthreads();
    for (int h = warp; h < rows_listed; h += kFewWarps) {                // a warp per row of up to kFewOfRow tokens
        const int first = heads[h];
        const std::uint32_t row = row_of[first];
        int count = 0;
        for (int i0 = first; i0 < n; i0 += 32) {
            const bool same = i0 + lane < n && row_of[i0 + lane] == row;
            const unsigned votes = __ballot_sync(0xffffffffu, same);
            const int at = count + __popc(votes & ((1u << lane) - 1u));
            if (same && at < kFewOfRow) few[warp][at] = token[i0 + lane];
            count += __popc(votes);
        }
        __syncwarp();
        if (count <= kFewOfRow) {
            for (int c0 = c_begin; c0 < c_end; c0 += 32 * VEC) {
                const int c = c0 + lane * VEC;
                float acc[VEC] = {};
                add_rows<T, VEC>(acc, dout, few[warp], count, f.hidden, c, c < c_end, gen, args);
                if (c < c_end) write_row<T, VEC>(dw + (static_cast<long long>(row) * shares + blockIdx.x) * f.hidden + c, acc, f.scale, f.accumulate);
            }
        }
        __syncwarp();
    }
    if (n <= kFewOfRow) return;
    // Rows of more tokens: every warp adds those in its part of the list, then the parts are added in order.
    const int share = (n + kFewWarps - 1) / kFewWarps, begin = warp * share, end = begin + share < n ? begin + share : n;
    for (int h = 0; h < rows_listed; ++h) {
        const int first = heads[h];
        const std::uint32_t row = row_of[first];
        int count = 0;
        for (int i = first + threadIdx.x; i < n; i += kFewThreads) count += row_of[i] == row;
        if (__syncthreads_count(count != 0) <= kFewOfRow) {              // at most one token a thread is counted: look closer
            int total = 0;
            for (int i0 = first; i0 < n; i0 += 32) total += __popc(__ballot_sync(0xffffffffu, i0 + lane < n && row_of[i0 + lane] == row));
            if (total <= kFewOfRow) continue;                            // the same in every warp
        }
        for (int c0 = c_begin; c0 < c_end; c0 += 32 * VEC) {
            const int c = c0 + lane * VEC;
            float acc[VEC] = {};
            for (int i0 = begin; i0 < end; i0 += 32) {
                const bool same = i0 + lane < end && row_of[i0 + lane] == row;
                const unsigned votes = __ballot_sync(0xffffffffu, same);
                __syncwarp();
                if (same) few[warp][__popc(votes & ((1u << lane) - 1u))] = token[i0 + lane];
                __syncwarp();
                add_rows<T, VEC>(acc, dout, few[warp], __popc(votes), f.hidden, c, c < c_end, gen, args);
            }
            put_floats<VEC>(&part[warp][lane * VEC], acc);
            __syncthreads();
            if (warp == 0 && c < c_end) {
                float total[VEC] = {};
                for (int w = 0; w < kFewWarps; ++w) add_floats<VEC>(total, &part[w][lane * VEC]);
                write_row<T, VEC>(dw + (static_cast<long long>(row) * shares + blockIdx.x) * f.hidden + c, total, f.scale, f.accumulate);
            }
            __syncthreads();
        }
    }
}

int bit_length(std::uint64_t v) {
    int b = 0;
    while (v) { ++b; v >>= 1; }
    return b;
}

// Threads per row, as a power of two: enough for the row's vectors, at most kThreads.
int group_shift(std::size_t hidden, int vec) {
    int s = 0;
    while ((1 << s) < kThreads && (std::size_t{1} << s) * vec < hidden) ++s;
    return s;
}

std::size_t at_most(std::size_t n, std::size_t limit) { return n < limit ? n : limit; }

// Layout of the run sums: threads per row (2^shift), groups per CTA, CTAs.
struct SumPlan {
    static constexpr std::size_t kSlots = 2 * kNumSMs;       // CTAs that run at once
    int shift, groups, chunk, ctas;
    SumPlan(std::size_t tokens, std::size_t hidden, int vec) {
        shift = group_shift(hidden, vec);
        // As many groups as threads allow (and kMostGroups, whose runs are joined one after the other), fewer when there are few
        // tokens: then every SM gets some. Chunks as long as lets all CTAs run at once (two per SM), up to kMostChunk.
        std::size_t n = at_most(most_groups(shift), (tokens + kSlots * kInFlight - 1) / (kSlots * kInFlight));
        groups = static_cast<int>(n);
        const std::size_t even = (tokens + kSlots * n - 1) / (kSlots * n);
        chunk = static_cast<int>(even < kMostChunk ? (even + kInFlight - 1) / kInFlight * kInFlight : kMostChunk);
        ctas = static_cast<int>((tokens + n * chunk - 1) / (n * chunk));
    }
    static std::size_t most_groups(int shift) { return at_most(kSumThreads >> shift, kMostGroups); }
    // The most CTAs of a plan for up to `tokens` tokens. (`ctas` itself falls where CTAs get another group.) A CTA has kInFlight
    // tokens at least. Shorter chunks than kMostChunk are as long as lets all CTAs run at once; a plan that needs the longest has
    // all groups by then: it takes more than 31 kSlots tokens a group, and kInFlight kSlots tokens make a group.
    static std::size_t most_ctas(std::size_t tokens, std::size_t hidden, int vec) {
        const std::size_t span = most_groups(group_shift(hidden, vec)) * kMostChunk;
        return std::max(at_most((tokens + kInFlight - 1) / kInFlight, kSlots), (tokens + span - 1) / span);
    }
};

// Byte offsets of the workspace's parts, enough for every type and alignment.
struct Layout {
    std::size_t keys[2], vals[2], counts, totals, crossing, partial, bytes;
    int tiles;
    Layout(std::size_t tokens, std::size_t hidden) {
        tiles = static_cast<int>((tokens + kSortTile - 1) / kSortTile);
        std::size_t ctas = 0;
        for (int vec : {1, 4, 8}) ctas = std::max(ctas, SumPlan::most_ctas(tokens, hidden, vec));
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
    return tokens != 0 && vocab != 0 && hidden != 0 && tokens <= 0x7fffffffull && vocab <= 0x7ffffffeull && hidden <= (1ull << 30) &&
           tokens <= (1ull << 46) / hidden && vocab <= (1ull << 46) / hidden;
}

template <typename T, int VEC>
int launch_sum(void* dw, const void* dout, GradArgs g, const DropoutArgs& args, cudaStream_t s) {
    const SumPlan p(static_cast<std::size_t>(g.n), static_cast<std::size_t>(g.hidden), VEC);
    g.shift = p.shift;
    g.groups = p.groups;
    g.chunk = p.chunk;
    g.ctas = p.ctas;
    const int threads = g.groups << g.shift < 32 ? 32 : g.groups << g.shift;
    const std::size_t smem = static_cast<std::size_t>(threads) * 2 * VEC * sizeof(float) + (2 * static_cast<std::size_t>(g.groups) * g.chunk + 8) * 4;
    static PerDeviceOnce once;
    if (once.needed()) {
        CGPT_CUDA_TRY(cudaFuncSetAttribute(scaled_embedding_sum_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024));
        once.done();
    }
    CGPT_CUDA_TRY(launch_after_previous(scaled_embedding_sum_kernel<T, VEC>, dim3(g.ctas), threads, smem, s, static_cast<T*>(dw), static_cast<const T*>(dout), g, args));
    count_launch();
    if (g.ctas == 1) return CGPT_OK;
    constexpr int JV = VEC < 4 ? 1 : 4;
    const unsigned column_tiles = static_cast<unsigned>((g.hidden + 32 * JV - 1) / (32 * JV));
    const unsigned runs = g.ctas - 1, lanes = column_tiles < kNumSMs * 32u ? kNumSMs * 32u / column_tiles : 1;   // runs at a time
    CGPT_CUDA_TRY(launch_after_previous(scaled_embedding_join_kernel<T, JV>, dim3(column_tiles * (runs < lanes ? runs : lanes)), kJoinThreads, 0, s,
                                        static_cast<T*>(dw), g));
    count_launch();
    return CGPT_OK;
}

bool takes_few(std::size_t tokens, std::size_t vocab, std::size_t hidden, std::size_t elem, bool vectors) {
    return tokens <= (vectors ? kFewTokens / 2 : kFewTokens) && hidden <= (1u << 20) &&      // a grid has 65535 tiles at most
           vocab <= (vectors ? (4u << 20) : (16u << 20)) / (hidden * elem);
}

// Row shares and column tiles of the few-tokens launch: about two CTAs per SM.
template <typename T, int VEC>
int launch_few(void* dw, const void* dout, FewArgs f, const DropoutArgs& args, cudaStream_t s) {
    const int chunk = 32 * VEC;                                          // columns of a warp
    const int most = f.hidden > (VEC > 1 ? 1 : 4) * chunk ? (VEC > 1 ? 1 : 4) * chunk : f.hidden;
    const unsigned tiles = static_cast<unsigned>((f.hidden + most - 1) / most);
    f.tile = most;
    const unsigned want = tiles < 2 * kNumSMs ? 2 * kNumSMs / tiles : 1, least = (f.vocab + kFewRows - 1) / kFewRows;
    unsigned shares = want > least ? want : least;
    if (shares > f.vocab) shares = f.vocab;
    scaled_embedding_few_kernel<T, VEC><<<dim3(shares, tiles), kFewThreads, 0, s>>>(static_cast<T*>(dw), static_cast<const T*>(dout), f, args);
    count_launch();
    CGPT_LAUNCH_CHECK();
    return CGPT_OK;
}

// Clusters of the sort by keys per thread (1, 2, kMostKeys).
void (*const kClusterKernels[3])(ClusterSort) = {sort_cluster_kernel<1>, sort_cluster_kernel<2>, sort_cluster_kernel<kMostKeys>};
constexpr std::size_t kClusterSmem[3] = {sizeof(ClusterSmem<1>), sizeof(ClusterSmem<2>), sizeof(ClusterSmem<kMostKeys>)};

int cluster_config(cudaLaunchConfig_t* config, cudaLaunchAttribute* attribute, int size, int ctas, cudaStream_t s) {
    static PerDeviceOnce once[3];
    if (once[size].needed()) {
        CGPT_CUDA_TRY(cudaFuncSetAttribute(kClusterKernels[size], cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        CGPT_CUDA_TRY(cudaFuncSetAttribute(kClusterKernels[size], cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kClusterSmem[size])));
        once[size].done();
    }
    *config = cudaLaunchConfig_t{};
    config->gridDim = dim3(ctas);
    config->blockDim = dim3(kClusterThreads);
    config->dynamicSmemBytes = kClusterSmem[size];
    config->stream = s;
    attribute->id = cudaLaunchAttributeClusterDimension;
    attribute->val.clusterDim.x = ctas;
    attribute->val.clusterDim.y = attribute->val.clusterDim.z = 1;
    config->attrs = attribute;
    config->numAttrs = 1;
    return CGPT_OK;
}

// CTAs of the largest cluster that the current device places: 16, or the 8 that every device has to, where a part of the GPU is
// not ours. Asked once per device.
int most_cluster_ctas(int* ctas) {
    static std::atomic<int> known[64];
    int device = 0;
    CGPT_CUDA_TRY(cudaGetDevice(&device));
    if (device < 0 || device >= 64) return CGPT_ERR_UNSUPPORTED;
    *ctas = known[device].load(std::memory_order_relaxed);
    if (*ctas == 0) {
        cudaLaunchConfig_t config;
        cudaLaunchAttribute attribute;
        CGPT_TRY(cluster_config(&config, &attribute, 2, kMaxCluster, nullptr));
        int n = 0;
        const bool asked = cudaOccupancyMaxActiveClusters(&n, kClusterKernels[2], &config) == cudaSuccess, fits = asked && n > 0;
        if (!asked) cudaGetLastError();       // its own error only: an earlier one is the caller's to read
        *ctas = fits ? kMaxCluster : 8;
        known[device].store(*ctas, std::memory_order_relaxed);
    }
    return CGPT_OK;
}

// One launch: a cluster that sorts, others that clear. p.n <= most * kClusterThreads * kMostKeys.
int launch_cluster_sort(const ClusterSort& p, int most, cudaStream_t s) {
    int ctas = 1;
    while (ctas < most && ctas * kClusterThreads < p.n) ctas *= 2;
    const int keys = (p.n + ctas * kClusterThreads - 1) / (ctas * kClusterThreads), size = keys == 1 ? 0 : keys == 2 ? 1 : 2;
    cudaLaunchConfig_t config;
    cudaLaunchAttribute attribute;
    CGPT_TRY(cluster_config(&config, &attribute, size, ctas, s));
    if (p.clear != nullptr) config.gridDim = dim3(128 / ctas * ctas);   // clusters of 16 that fit on the SMs at a time: 8
    CGPT_CUDA_TRY(cudaLaunchKernelEx(&config, kClusterKernels[size], p));
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
    if (!element_aligned(dtype, {out, weight}) || !element_aligned(CGPT_DTYPE_F32, {ids})) return CGPT_ERR_ALIGN;
    DropoutArgs args;
    CGPT_TRY(dropout_args(&args, probability, state, site, tokens * hidden));
    if (!std::isfinite(scale * args.scale)) return CGPT_ERR_OPTION;      // what kept elements are multiplied by
    auto s = static_cast<cudaStream_t>(stream);
    CGPT_DISPATCH_DTYPE(dtype, T, {
        constexpr int V = 16 / sizeof(T);
        const bool vector = hidden % V == 0 && aligned16(out) && aligned16(weight);
        auto kernel = vector ? scaled_embedding_forward_kernel<T, V> : scaled_embedding_forward_kernel<T, 1>;
        const int shift = group_shift(hidden, vector ? V : 1);
        const std::size_t per_cta = static_cast<std::size_t>(kThreads >> shift) * kLookups, need = (tokens + per_cta - 1) / per_cta;
        const std::size_t cap = static_cast<std::size_t>(kNumSMs) * resident_ctas_per_sm(reinterpret_cast<const void*>(kernel), kThreads, 0);
        kernel<<<static_cast<unsigned>(need < cap ? need : cap), kThreads, 0, s>>>(
            static_cast<T*>(out), ids, static_cast<const T*>(weight), static_cast<long long>(tokens), static_cast<std::uint32_t>(vocab),
            static_cast<int>(hidden), scale, shift, args);
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
    if (grad_weight == grad_output) return CGPT_ERR_OPTION;
    if (!element_aligned(dtype, {grad_weight, grad_output}) || !element_aligned(CGPT_DTYPE_F32, {ids}) || !aligned16(workspace)) return CGPT_ERR_ALIGN;
    DropoutArgs args;
    CGPT_TRY(dropout_args(&args, probability, state, site, tokens * hidden));
    if (!std::isfinite(scale * args.scale)) return CGPT_ERR_OPTION;
    auto s = static_cast<cudaStream_t>(stream);
    auto* base = static_cast<unsigned char*>(workspace);
    auto words = [&](std::size_t offset) { return reinterpret_cast<std::uint32_t*>(base + offset); };

    const bool vectors = hidden % (16 / dtype_size(dtype)) == 0 && aligned16(grad_weight) && aligned16(grad_output);
    if (takes_few(tokens, vocab, hidden, dtype_size(dtype), vectors)) {
        const FewArgs f{ids, static_cast<int>(tokens), static_cast<int>(hidden), 0, accumulate, static_cast<std::uint32_t>(vocab), padding_id, scale * args.scale};
        CGPT_DISPATCH_DTYPE(dtype, T, {
            if (vectors) return (launch_few<T, 16 / sizeof(T)>(grad_weight, grad_output, f, args, s));
            return (launch_few<T, 1>(grad_weight, grad_output, f, args, s));
        });
    }
    const int bits = bit_length(vocab);   // keys are in [0, vocab]
    const int passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    const int digit_bits = (bits + passes - 1) / passes;
    int most = 0;
    CGPT_TRY(most_cluster_ctas(&most));
    const bool one_cluster = tokens <= static_cast<std::size_t>(most) * kClusterThreads * kMostKeys;
    const std::size_t table_bytes = vocab * hidden * dtype_size(dtype);
    ClusterSort c{};
    // The table starts on an element, the vectors that clear it on 16 bytes: the few bytes before go with a small memset.
    const std::size_t lead = std::min<std::size_t>((16 - (reinterpret_cast<std::uintptr_t>(grad_weight) & 15)) & 15, table_bytes);
    if (!accumulate) {
        if (lead != 0 || !one_cluster) CGPT_CUDA_TRY(cudaMemsetAsync(grad_weight, 0, one_cluster ? lead : table_bytes, s));
        c.clear = reinterpret_cast<uint4*>(static_cast<unsigned char*>(grad_weight) + lead);
        c.clear_vectors = static_cast<long long>((table_bytes - lead) / 16);
        c.clear_tail = static_cast<int>((table_bytes - lead) % 16);
    }
    c.ids = ids;
    const int last = one_cluster ? 0 : (passes - 1) & 1;   // which buffers the sorted tokens end up in
    c.keys = words(at.keys[last]);
    c.vals = words(at.vals[last]);
    c.crossing = words(at.crossing);
    c.n = static_cast<int>(tokens);
    c.bits = digit_bits;
    c.passes = passes;
    c.vocab = static_cast<std::uint32_t>(vocab);
    c.skip_id = padding_id;
    if (one_cluster) {
        CGPT_TRY(launch_cluster_sort(c, most, s));
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
    }
    const GradArgs g{c.keys, c.vals, reinterpret_cast<float*>(base + at.partial), c.crossing, static_cast<long long>(tokens),
                     static_cast<long long>(hidden), c.vocab, 0, accumulate, 0, 0, 0, scale * args.scale};
    CGPT_DISPATCH_DTYPE(dtype, T, {
        if (vectors) return (launch_sum<T, 16 / sizeof(T)>(grad_weight, grad_output, g, args, s));
        return (launch_sum<T, 1>(grad_weight, grad_output, g, args, s));
    });
    return CGPT_OK;
}
