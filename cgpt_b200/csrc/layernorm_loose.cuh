// Layer norm of rows that no 16-byte vector fits (odd lengths, unaligned tensors). Included by layernorm.cu only.
//
// Element by element from global memory these rows are slow for want of loads in flight (2-byte loads, 64 bytes a warp). So they
// come through the same rings as whole-vector rows: consecutive rows are one contiguous range of bytes, of which the part on the
// 16-byte grid is fetched by a bulk copy, rounded OUTWARD to the grid where that stays inside the tensor. Only the first and last
// rows of a tensor can have up to 15 bytes on either side that the grid cuts off; the threads that use those rows load them.
// Lanes then take consecutive elements from shared memory, so that their stores to global memory are consecutive too. All is done
// an element at a time (a warp moves 64 bytes of a 16-bit type per access), by few warps: 0.65 instructions per scheduler and cycle,
// one warp eligible. Measured at 32768 x 1001 bf16: forward 57 us (2.3 TB/s), backward with a residual 87 (3.0 TB/s), the fused
// forward 128 (2.1 TB/s) and backward 147 (2.2 TB/s); 3000 x 6001 fp16 backward 72.
#pragma once

namespace loose_kernels {

using ring_kernels::kMaxStages;
constexpr int kForwardThreads = 1024;    // one CTA per SM
constexpr int kBackwardThreads = 512;    // per SM: two CTAs of 256 or one of 512
constexpr int kMostColumns = 16;         // columns per thread of the backward
constexpr int kMaxTileRows = 64;
constexpr std::size_t kStatsBytes = 2 * kMaxTileRows * 16;   // static shared memory of the backward
constexpr unsigned kSlack = 32;          // bytes of a stage beside the rows: both ends rounded to the grid

// Rows row0 .. row0 + n of a tensor: which bytes of it a bulk copy brings, and where a stage has them.
struct Span {
    const unsigned char* from;     // first byte of the copy
    unsigned bytes;                // of the copy, a multiple of 16
    unsigned at;                   // where in the stage it goes
    unsigned first;                // where in the stage element (row0, 0) is
    unsigned head, tail;           // elements before and behind the copy, which are loaded one by one
};
template <typename T>
__host__ __device__ __forceinline__ Span span_of(const T* tensor, long long row0, unsigned n, long long rows, int hidden) {
    const std::uintptr_t begin = reinterpret_cast<std::uintptr_t>(tensor + row0 * hidden), end = begin + static_cast<std::uintptr_t>(n) * hidden * sizeof(T);
    const std::uintptr_t all = reinterpret_cast<std::uintptr_t>(tensor), all_end = reinterpret_cast<std::uintptr_t>(tensor + rows * hidden);
    const std::uintptr_t grid = begin & ~std::uintptr_t{15};
    std::uintptr_t lo = grid < all ? grid + 16 : grid, hi = (end + 15) & ~std::uintptr_t{15};
    if (hi > all_end) hi -= 16;
    if (hi < lo) hi = lo;
    Span s;
    s.from = reinterpret_cast<const unsigned char*>(lo);
    s.bytes = static_cast<unsigned>(hi - lo);
    s.at = static_cast<unsigned>(lo - grid);
    s.first = static_cast<unsigned>(begin - grid);
    s.head = lo > begin ? static_cast<unsigned>(((lo < end ? lo : end) - begin) / sizeof(T)) : 0u;
    const std::uintptr_t done = hi > begin ? hi : begin;     // everything before it is copied or in the head
    s.tail = lo <= end && done < end ? static_cast<unsigned>((end - done) / sizeof(T)) : 0u;
    return s;
}

// Ring of stages of consecutive rows of up to three tensors, each where its span has it.
struct Ring : BulkRing {
    template <typename T>
    __device__ __forceinline__ void fill(int s, const T* a, const T* b, const T* c, long long row0, int step_rows, long long rows, int hidden) const {
        if (row0 >= rows) return;
        const unsigned n = static_cast<unsigned>(rows - row0 < step_rows ? rows - row0 : step_rows);
        const Span sa = span_of(a, row0, n, rows, hidden), sb = b != nullptr ? span_of(b, row0, n, rows, hidden) : Span{},
                   sc = c != nullptr ? span_of(c, row0, n, rows, hidden) : Span{};
        unsigned char* to = data + s * stage_bytes;
        sm100::mbar_expect_tx(&full[s], sa.bytes + sb.bytes + sc.bytes);
        if (sa.bytes != 0) sm100::bulk_load_1d(to + sa.at, sa.from, sa.bytes, &full[s]);
        if (sb.bytes != 0) sm100::bulk_load_1d(to + tensor_bytes + sb.at, sb.from, sb.bytes, &full[s]);
        if (sc.bytes != 0) sm100::bulk_load_1d(to + 2 * tensor_bytes + sc.at, sc.from, sc.bytes, &full[s]);
    }
};

// Orders this thread's stores to a stage before the copies that refill it after the next barrier.
__device__ __forceinline__ void stores_before_copies() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The rows of a tensor in a stage. The elements that the copy left out are loaded by `threads` threads; returns whether there
// were any (then the threads have to meet before they read).
template <typename T>
__device__ __forceinline__ bool complete(T*& rows_at, unsigned char* stage, const T* tensor, long long row0, unsigned n, long long rows, int hidden, int thread,
                                         int threads) {
    const Span s = span_of(tensor, row0, n, rows, hidden);
    rows_at = reinterpret_cast<T*>(stage + s.first);
    const unsigned all = n * hidden;
    const T* from = tensor + row0 * hidden;
    for (unsigned i = thread; i < s.head; i += threads) rows_at[i] = from[i];
    for (unsigned i = thread; i < s.tail; i += threads) rows_at[all - s.tail + i] = from[all - s.tail + i];
    if (s.head + s.tail != 0) stores_before_copies();
    return s.head + s.tail != 0;
}

struct LooseArgs {
    unsigned int* status;
    int warps_per_row, step_rows, groups, stages;
    unsigned tensor_bytes, data_offset;
};

__device__ __forceinline__ void meet(int warps, int barrier) {
    if (warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
}

// Shared memory: [barriers][sums of multi-warp rows][w][b][rings], as ring_kernels.
constexpr int kMaxGroups = kForwardThreads / 32;
constexpr unsigned kSumsOffset = kMaxGroups * kMaxStages * 8, kVectorsOffset = kSumsOffset + kMaxGroups / 2 * 64 * 4;

template <typename T>
__device__ __forceinline__ void stage_vector(float* to, const T* from, int hidden) {
    for (int i = threadIdx.x; i < hidden; i += blockDim.x) to[i] = from != nullptr ? to_f32<T>(from[i]) : 0.f;
}

// Calls f(c) for the columns c = begin + lane, begin + lane + 32, ... below end; eight at a time, so that a column's addresses
// are constants beside the first one's.
template <typename F>
__device__ __forceinline__ void each_column(int begin, int end, int lane, const F& f) {
    int c0 = begin;
    for (; c0 + 256 <= end; c0 += 256) {
#pragma unroll
        for (int u = 0; u < 8; ++u) f(c0 + lane + u * 32);
    }
    for (int c = c0 + lane; c < end; c += 32) f(c);
}

// A group of warps per row, row after row of a stage; a warp has a contiguous part of the row.
template <typename T, bool FUSED>
__global__ void __launch_bounds__(kForwardThreads, 1)
layernorm_forward_loose_kernel(T* __restrict__ y, T* sum, const T* x, const T* residual, const T* __restrict__ w, const T* __restrict__ b,
                               long long rows, int hidden, float epsilon, const LooseArgs la, const DropoutArgs args) {
    extern __shared__ __align__(128) unsigned char shared[];
    float* ws = reinterpret_cast<float*>(shared + kVectorsOffset);
    float* bs = ws + hidden;
    const int lanes = la.warps_per_row * 32, group = threadIdx.x / lanes, tid = threadIdx.x - group * lanes;
    const int warp_in_row = tid >> 5, lane = tid & 31, part = (hidden + la.warps_per_row - 1) / la.warps_per_row;
    const int begin = warp_in_row * part, end = begin + part < hidden ? begin + part : hidden;
    float* red = reinterpret_cast<float*>(shared + kSumsOffset) + group * 64;
    const long long step = static_cast<long long>(gridDim.x) * la.groups * la.step_rows;
    const long long first = (static_cast<long long>(blockIdx.x) * la.groups + group) * la.step_rows;
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    bool leader = tid == 0;
    Ring ring{};
    ring.tensor_bytes = la.tensor_bytes;
    ring.stage_bytes = FUSED ? 2 * la.tensor_bytes : la.tensor_bytes;
    ring.stages = la.stages;
    ring.full = reinterpret_cast<std::uint64_t*>(shared) + group * kMaxStages;
    ring.data = shared + la.data_offset + static_cast<std::size_t>(group) * la.stages * ring.stage_bytes;
    ring.status = la.status;
    const T *second = FUSED ? residual : nullptr, *none = nullptr;
    if (leader) {
        ring.init();
        for (int s = 0; s < la.stages; ++s) ring.fill(s, x, second, none, first + s * step, la.step_rows, rows, hidden);
    }
    stage_vector(ws, w, hidden);
    stage_vector(bs, b, hidden);
    const KeptPhilox gen(args);
    __syncthreads();

    for (long long row0 = first; row0 < rows; row0 += step) {
        unsigned char* stage = ring.wait(&leader);
        const unsigned n = static_cast<unsigned>(rows - row0 < la.step_rows ? rows - row0 : la.step_rows);
        T *xs, *rs = nullptr;
        bool loaded = complete(xs, stage, x, row0, n, rows, hidden, tid, lanes);
        if constexpr (FUSED) loaded |= complete(rs, stage + ring.tensor_bytes, residual, row0, n, rows, hidden, tid, lanes);
        if (loaded) meet(la.warps_per_row, group + 1);
        for (unsigned r = 0; r < n; ++r) {
            T* row = xs + static_cast<std::size_t>(r) * hidden;
            const long long e0 = (row0 + r) * hidden;
            float s[1] = {0.f};
            if constexpr (FUSED) {
                const T* res = rs + static_cast<std::size_t>(r) * hidden;
                auto element = [&](int c, unsigned keep) {
                    const float v = keep != 0u ? __fmul_rn(to_f32<T>(row[c]), args.scale) : 0.f;
                    const T stored = from_f32<T>(v + to_f32<T>(res[c]));
                    row[c] = stored;                          // the norm is of the stored value
                    sum[e0 + c] = stored;
                    s[0] += to_f32<T>(stored);
                };
                // 256 elements from a generator block's first one on are 32 blocks: a block per lane, handed round bit by bit
                for (int c0 = begin - static_cast<int>((e0 + begin) & 7); c0 < end; c0 += 256) {
                    std::uint32_t kept = 255u;
                    if (args.threshold != 0) kept = kept_bits(gen.block(static_cast<std::uint32_t>((e0 + c0) >> 3) + lane), args.threshold);
                    const bool whole = c0 >= begin && c0 + 256 <= end;
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const unsigned keep = (__shfl_sync(0xffffffffu, kept, u * 4 + (lane >> 3)) >> (lane & 7)) & 1u;
                        const int c = c0 + u * 32 + lane;
                        if (whole || (c >= begin && c < end)) element(c, keep);
                    }
                }
                // columns were dealt out from a generator block's start, below they are from `begin`: lanes read what others wrote
                __syncwarp();
            } else {
                each_column(begin, end, lane, [&](int c) { s[0] += to_f32<T>(row[c]); });
            }
            s[0] = warp_sum(s[0]);
            if (la.warps_per_row > 1) ring_kernels::warps_sum<1>(s, la.warps_per_row, warp_in_row, group + 1, red);
            const float mean = s[0] * inv_hidden;
            s[0] = 0.f;
            each_column(begin, end, lane, [&](int c) {
                const float d = to_f32<T>(row[c]) - mean;
                s[0] = fmaf(d, d, s[0]);
            });
            s[0] = warp_sum(s[0]);
            if (la.warps_per_row > 1) ring_kernels::warps_sum<1>(s, la.warps_per_row, warp_in_row, group + 1, red + 16);
            const float rstd = rsqrtf(fmaf(s[0], inv_hidden, epsilon));
            T* out = y + e0;
            each_column(begin, end, lane, [&](int c) { out[c] = from_f32<T>(fmaf(normalised(to_f32<T>(row[c]), mean, rstd), ws[c], bs[c])); });
        }
        if constexpr (FUSED) stores_before_copies();
        meet(la.warps_per_row, group + 1);
        if (leader) ring.fill(ring.stage, x, second, none, row0 + ring.stages * step, la.step_rows, rows, hidden);
        ring.next();
    }
}

// Tiles of rows in two phases, as ring_kernels: a warp group per row for the sums, then a thread per column. K columns per thread,
// THREADS apart; with K == 1 the threads cover `groups` rows at a time, element after element. partial: [gridDim.x][2][hidden].
template <typename T, int K, int THREADS, bool FUSED>
__global__ void __launch_bounds__(THREADS, kBackwardThreads / THREADS)
layernorm_backward_loose_kernel(T* dx, T* din, float* __restrict__ partial, const T* __restrict__ dy, const T* __restrict__ x,
                                const T* __restrict__ w, const T* residual, long long rows, int hidden, float epsilon, const LooseArgs la,
                                const DropoutArgs args) {
    extern __shared__ __align__(128) unsigned char shared[];
    __shared__ float4 stats[2][kMaxTileRows];                // mean, rstd, c1, c2 of the tile's rows
    float* ws = reinterpret_cast<float*>(shared + kVectorsOffset);
    const int lanes = la.warps_per_row * 32, unit = threadIdx.x / lanes, units = THREADS / lanes, tid = threadIdx.x - unit * lanes;
    const int warp_in_row = tid >> 5, lane = threadIdx.x & 31, part = (hidden + la.warps_per_row - 1) / la.warps_per_row;
    const int begin = warp_in_row * part, end = begin + part < hidden ? begin + part : hidden;
    float* red = reinterpret_cast<float*>(shared + kSumsOffset) + unit * 64;
    launch_dependents();
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    const long long step = static_cast<long long>(gridDim.x) * la.step_rows;
    const long long first = static_cast<long long>(blockIdx.x) * la.step_rows;
    Ring ring{};
    ring.tensor_bytes = la.tensor_bytes;
    ring.stage_bytes = 3 * la.tensor_bytes;
    ring.stages = la.stages;
    ring.full = reinterpret_cast<std::uint64_t*>(shared);
    ring.data = shared + la.data_offset;
    ring.status = la.status;
    if (threadIdx.x == 0) {
        ring.init();
        for (int s = 0; s < la.stages; ++s) ring.fill(s, x, dy, residual, first + s * step, la.step_rows, rows, hidden);
    }
    stage_vector(ws, w, hidden);
    const KeptPhilox gen(args);
    const int row_group = K == 1 ? threadIdx.x / hidden : 0;
    const int column = K == 1 ? threadIdx.x - row_group * hidden : threadIdx.x;
    const bool works = K > 1 || row_group < la.groups;
    __syncthreads();
    float wv[K], aw[K] = {}, ab[K] = {};
#pragma unroll
    for (int k = 0; k < K; ++k) wv[k] = column + k * THREADS < hidden ? ws[column + k * THREADS] : 0.f;

    int buffer = 0;
    for (long long row0 = first; row0 < rows; row0 += step, buffer ^= 1) {
        const int tile_rows = rows - row0 < la.step_rows ? static_cast<int>(rows - row0) : la.step_rows;
        unsigned char* stage = ring.wait();
        T *xs, *gs, *rs = nullptr;
        bool loaded = complete(xs, stage, x, row0, tile_rows, rows, hidden, threadIdx.x, THREADS);
        loaded |= complete(gs, stage + ring.tensor_bytes, dy, row0, tile_rows, rows, hidden, threadIdx.x, THREADS);
        if (residual != nullptr) loaded |= complete(rs, stage + 2 * ring.tensor_bytes, residual, row0, tile_rows, rows, hidden, threadIdx.x, THREADS);
        if (loaded) __syncthreads();
        // ---- rows: four sums each
        for (int row = unit; row < tile_rows; row += units) {
            const T *xr = xs + row * hidden, *gr = gs + row * hidden;
            float m[1] = {0.f}, s[3] = {0.f, 0.f, 0.f};
            each_column(begin, end, lane, [&](int c) { m[0] += to_f32<T>(xr[c]); });
            m[0] = warp_sum(m[0]);
            if (la.warps_per_row > 1) ring_kernels::warps_sum<1>(m, la.warps_per_row, warp_in_row, unit + 1, red);
            const float mean = m[0] * inv_hidden;
            each_column(begin, end, lane, [&](int c) { norm_sums(s, to_f32<T>(gr[c]), ws[c], to_f32<T>(xr[c]) - mean); });
#pragma unroll
            for (int i = 0; i < 3; ++i) s[i] = warp_sum(s[i]);
            if (la.warps_per_row > 1) ring_kernels::warps_sum<3>(s, la.warps_per_row, warp_in_row, unit + 1, red + 16);
            if (tid == 0) {
                const float rstd = rsqrtf(fmaf(s[0], inv_hidden, epsilon));
                stats[buffer][row] = make_float4(mean, rstd, s[1] * inv_hidden, s[2] * inv_hidden * rstd);
            }
        }
        __syncthreads();
        // Every thread is past the columns of the tile before: its stage is free.
        if (threadIdx.x == 0 && !ring.failed && row0 != first)
            ring.fill(ring.stage == 0 ? ring.stages - 1 : ring.stage - 1, x, dy, residual, row0 + (ring.stages - 1) * step, la.step_rows, rows, hidden);
        // ---- columns: RJ rows (of the row group) at a time; with dropout the lanes of a warp share the decisions of four elements
        constexpr int RJ = K >= 4 ? 1 : 4 / K;
        for (int r0 = 0; r0 < tile_rows; r0 += RJ * la.groups) {
            float4 st[RJ];
            bool has_row[RJ];
#pragma unroll
            for (int q = 0; q < RJ; ++q) {
                const int row = r0 + q * la.groups + row_group;
                has_row[q] = works && row < tile_rows;
                st[q] = stats[buffer][has_row[q] ? row : 0];
            }
            const int in_tile = (r0 + row_group) * hidden + column, next_row = la.groups * hidden;
            const T *xr = xs + in_tile, *gr = gs + in_tile, *rr = rs + in_tile;
            const long long e = row0 * hidden + in_tile;
            T *to = dx + e, *to_in = FUSED ? din + e : nullptr;
#pragma unroll
            for (int i0 = 0; i0 < RJ * K; i0 += 4) {
                std::uint32_t kept = 15u;
                if constexpr (FUSED) {
                    if (args.threshold != 0) {
                        long long start[4];                   // element of lane 0: threads are consecutive elements, also across row groups
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            start[j] = (row0 + r0) * hidden + static_cast<int>(threadIdx.x) - lane + (i0 + j) / K * next_row + (i0 + j) % K * THREADS;
                        kept = keep_four_runs(start, gen, args.threshold);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int q = (i0 + j) / K, k = (i0 + j) % K, at = q * next_row + k * THREADS;
                    if (has_row[q] && (K == 1 || column + k * THREADS < hidden)) {
                        const float g = to_f32<T>(gr[at]), xh = normalised(to_f32<T>(xr[at]), st[q].x, st[q].y);
                        const float out = norm_dx(g, wv[k], xh, st[q].y, st[q].z, st[q].w, residual != nullptr ? to_f32<T>(rr[at]) : 0.f);
                        aw[k] = fmaf(g, xh, aw[k]);
                        ab[k] += g;
                        to[at] = from_f32<T>(out);
                        if constexpr (FUSED) to_in[at] = from_f32<T>((kept >> j) & 1u ? __fmul_rn(out, args.scale) : 0.f);
                    }
                }
            }
        }
        ring.next();
    }
    // One partial row of dw and of db per CTA: its row groups add up one after the other, in the memory of the ring, whose copies
    // have all been waited for. Where a wait ran out they may not have come, and the rows are worth nothing.
    if (__syncthreads_or(ring.failed)) return;
    float* out_w = partial + static_cast<long long>(blockIdx.x) * 2 * hidden;
    float* joined = reinterpret_cast<float*>(shared + la.data_offset);
    const int groups = K == 1 ? la.groups : 1;
    for (int q = 0; q < groups; ++q) {
        if (q > 0) __syncthreads();
        if (works && row_group == q) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int col = column + k * THREADS;
                if (col < hidden) {
                    const float tw = (q == 0 ? 0.f : joined[col]) + aw[k], tb = (q == 0 ? 0.f : joined[hidden + col]) + ab[k];
                    (q + 1 < groups ? joined : out_w)[col] = tw;
                    (q + 1 < groups ? joined : out_w)[hidden + col] = tb;
                }
            }
        }
    }
}

}  // namespace loose_kernels
