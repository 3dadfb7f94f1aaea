// Layer norm of rows that are whole 16-byte vectors. Included by layernorm.cu only.
//
// What limits these kernels once memory is read ahead is the number of instructions: at the rate memory delivers 16-bit
// elements an SM has about 20 issue slots for each. Hence
//  * rows come through rings of stages in shared memory, filled by bulk copies (consecutive rows are contiguous: one copy per
//    tensor and stage), so that nothing but one thread per ring deals with memory and its latency;
//  * arithmetic is on pairs (fma / mul / add .f32x2): one issue slot for two elements;
//  * a row is summed by as few warps as hold it in registers, so that the shuffles of a sum are shared by up to 64 elements of a
//    lane, and by up to four rows where rows are short; what is read is converted to fp32 once;
//  * w and b are kept in shared memory as fp32: no conversion per row.
//
// Forward: every group of warps walks rows through a ring of its own. Backward: a CTA takes tiles of rows in two phases, rows
// first (a warp group per row: mean, rstd and the two sums of dx, left in shared memory), then columns (a thread per vector of
// columns: dx, and the running dw and db of its columns in registers). Lanes that keep both a row's values and dw and db of
// their columns need 168 registers, and 12 warps an SM hide less: measured 62 against 57 us at 16384 x 2048 bf16.
//
// Measured (16-bit, device times): forward 32768 x 1024 26.1 us (5.1 TB/s, 80 % of a plain copy's rate; a copy of the same bytes
// takes 28.7), with dropout and residual 50.3 (5.3 TB/s), 4096 x 8192 with both 56.1 (4.8 TB/s); backward 16384 x 2048 with a residual
// 54.8 (4.9 TB/s), 32768 x 1024 45.3 (4.4 TB/s), 4096 x 8192 with a residual 66.6 (4.0 TB/s), the fused one at 32768 x 1024 72.2
// (4.6 TB/s). What the backward waits for is the border between its two phases: half the issue slots are empty (0.52 instructions per
// scheduler and cycle), with one warp eligible on average. Rows of 1025 to 1752 vectors spill 300 to 326 bytes a thread (four
// vectors of columns and of dw and db each), 2048 x 12008 takes 87 us (1.7 TB/s); rows of fewer than 32 vectors that fill no
// power of two of lanes 22.
#pragma once

namespace ring_kernels {

constexpr int kMaxStages = 4;
constexpr int kForwardThreads = 512;     // one CTA per SM (128 registers)
constexpr int kBackwardThreads = 512;    // per SM: two CTAs of 256, or one of 512 for rows of more than 256 vectors
constexpr int kTileVectors = 4;          // vectors of each tensor that a thread of the backward takes per tile
constexpr int kMaxTileRows = 128;
constexpr std::size_t kStatsBytes = 2 * kMaxTileRows * 32;   // static shared memory of the backward

// Rows a warp group takes at a time: a lane with few vectors per row holds several rows.
__host__ __device__ constexpr int rows_at_once(int cpt) { return cpt >= 4 ? 1 : 4 / cpt; }

// Ring of stages of consecutive rows of one tensor or two.
struct Ring : BulkRing {
    unsigned row_bytes;

    // Rows row0 .. row0 + step_rows of a and b (which may be null) into stage s, as far as there are such rows.
    template <typename T>
    __device__ __forceinline__ void fill(int s, const T* a, const T* b, long long row0, int step_rows, long long rows, int hidden) const {
        if (row0 >= rows) return;
        const unsigned n = static_cast<unsigned>(rows - row0 < step_rows ? rows - row0 : step_rows) * row_bytes;
        unsigned char* to = data + s * stage_bytes;
        sm100::mbar_expect_tx(&full[s], (1 + (b != nullptr)) * n);
        sm100::bulk_load_1d(to, a + row0 * hidden, n, &full[s]);
        if (b != nullptr) sm100::bulk_load_1d(to + tensor_bytes, b + row0 * hidden, n, &full[s]);
    }
};

// Layout of a launch: vectors per row, lanes per row (fewer than 32 where a warp holds several rows), warps per row, rows a group
// of such warps takes at a time, groups in a CTA, stages of each group's ring.
struct RingArgs {
    unsigned int* status;
    int vectors, lanes, warps_per_row, step_rows, groups, stages;
    unsigned data_offset;               // of the rings in shared memory
};

// Totals of N values over the `lanes` lanes (a power of two) of a row.
template <int N>
__device__ __forceinline__ void lanes_sum(float (&v)[N], int lanes) {
    if (lanes == 32) {
        if constexpr (N > 1) {
            WarpSums<N>::reduce(v, threadIdx.x & 31);
            WarpSums<N>::broadcast(v);
        } else {
            v[0] = warp_sum(v[0]);
        }
        return;
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
}

// Totals of N values over the warps of a row (one value of the row per lane set before). `red`: [16][N] floats of this call and
// group; two calls in a row use different areas, so that the barrier of one also says that the area of the other has been read.
template <int N>
__device__ __forceinline__ void warps_sum(float (&v)[N], int warps, int warp, int barrier, float* red) {
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) red[warp * N + i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = red[i];
    for (int w = 1; w < warps; ++w) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += red[w * N + i];
    }
}

// w or b (null: zeros) as fp32 in shared memory, four values at a time: the lanes that read consecutive vectors of eight find
// their first halves side by side in one area and their second halves in the next (no bank conflicts).
template <typename T>
__device__ __forceinline__ void stage_vector(float* to, const T* from, int vectors) {
    constexpr int VEC = 16 / sizeof(T), NP = VEC / 2;
    for (int i = threadIdx.x; i < vectors; i += blockDim.x) {
        Pair v[NP];
        to_pairs<T>(v, from != nullptr ? *reinterpret_cast<const uint4*>(from + i * VEC) : make_uint4(0u, 0u, 0u, 0u));
#pragma unroll
        for (int j = 0; j < NP / 2; ++j) reinterpret_cast<ulonglong2*>(to)[j * vectors + i] = make_ulonglong2(v[2 * j], v[2 * j + 1]);
    }
}
template <int NP>
__device__ __forceinline__ void read_pairs(Pair (&p)[NP], const float* from, int vec, int vectors) {
#pragma unroll
    for (int j = 0; j < NP / 2; ++j) {
        const ulonglong2 u = reinterpret_cast<const ulonglong2*>(from)[j * vectors + vec];
        p[2 * j] = u.x;
        p[2 * j + 1] = u.y;
    }
}

// Shared memory: [barriers][sums of multi-warp rows: 64 floats per group][w][b (forward)][rings]
constexpr int kMaxGroups = 16;                     // at most half as many where a row takes several warps
constexpr unsigned kSumsOffset = kMaxGroups * kMaxStages * 8, kVectorsOffset = kSumsOffset + kMaxGroups / 2 * 64 * 4;

// FULL: the lanes of a row hold exactly its vectors, so that no column is checked.
template <typename T, int CPT, bool FULL, bool FUSED>
__global__ void __launch_bounds__(kForwardThreads, 1)
layernorm_forward_ring_kernel(T* __restrict__ y, T* sum, const T* x, const T* residual, const T* __restrict__ w, const T* __restrict__ b,
                              long long rows, int hidden, float epsilon, const RingArgs ra, const DropoutArgs args) {
    constexpr int VEC = 16 / sizeof(T), NP = VEC / 2, R = rows_at_once(CPT);
    extern __shared__ __align__(128) unsigned char shared[];
    float* ws = reinterpret_cast<float*>(shared + kVectorsOffset);
    float* bs = ws + hidden;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = warp / ra.warps_per_row, warp_in_row = warp - group * ra.warps_per_row;
    const int per_warp = 32 / ra.lanes;                      // rows side by side in a warp
    const int lane_row = lane / ra.lanes, vec0 = warp_in_row * (32 * CPT) + (lane & (ra.lanes - 1));
    float* red = reinterpret_cast<float*>(shared + kSumsOffset) + group * 64;
    const long long step = static_cast<long long>(gridDim.x) * ra.groups * ra.step_rows;
    const long long first = (static_cast<long long>(blockIdx.x) * ra.groups + group) * ra.step_rows;
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    bool leader = warp_in_row == 0 && lane == 0;
    Ring ring{};
    ring.row_bytes = static_cast<unsigned>(hidden) * sizeof(T);
    ring.tensor_bytes = ra.step_rows * ring.row_bytes;
    ring.stage_bytes = FUSED ? 2 * ring.tensor_bytes : ring.tensor_bytes;
    ring.stages = ra.stages;
    ring.full = reinterpret_cast<std::uint64_t*>(shared) + group * kMaxStages;
    ring.data = shared + ra.data_offset + static_cast<std::size_t>(group) * ra.stages * ring.stage_bytes;
    ring.status = ra.status;
    const T* second = FUSED ? residual : nullptr;
    if (leader) {
        ring.init();
        for (int s = 0; s < ra.stages; ++s) ring.fill(s, x, second, first + s * step, ra.step_rows, rows, hidden);
    }
    stage_vector(ws, w, ra.vectors);
    stage_vector(bs, b, ra.vectors);
    const std::conditional_t<CPT == 8, KeptPhilox, Philox> gen(args);
    const unsigned lane_bytes = lane_row * ring.row_bytes + vec0 * 16, next_row = per_warp * ring.row_bytes;
    __syncthreads();

    for (long long row0 = first; row0 < rows; row0 += step) {
        const unsigned char* at = ring.wait(&leader) + lane_bytes;
        const int left = rows - row0 < ra.step_rows ? static_cast<int>(rows - row0) : ra.step_rows;   // rows of this step
        const long long e0 = (row0 + lane_row) * hidden + vec0 * VEC;                                 // the lane's first element
        Pair v[R][CPT][NP];
        float mean[R], rstd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            Pair acc = 0;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
#pragma unroll
                for (int i = 0; i < NP; ++i) v[r][c][i] = 0;         // a stage keeps what an earlier step left there
                if ((R == 1 || r * per_warp + lane_row < left) && (FULL || vec0 + c * 32 < ra.vectors)) {
                    to_pairs<T>(v[r][c], *reinterpret_cast<const uint4*>(at + r * next_row + c * 512));
                    if constexpr (FUSED) {
                        const long long e = e0 + r * per_warp * hidden + c * (32 * VEC);
                        if (args.threshold != 0) drop_pairs<NP>(v[r][c], gen, e, args);
                        Pair res[NP];
                        to_pairs<T>(res, *reinterpret_cast<const uint4*>(at + ring.tensor_bytes + r * next_row + c * 512));
#pragma unroll
                        for (int i = 0; i < NP; ++i) v[r][c][i] = add2(v[r][c][i], res[i]);
                        const uint4 stored = to_raw<T>(v[r][c]);
                        *reinterpret_cast<uint4*>(sum + e) = stored;
                        to_pairs<T>(v[r][c], stored);                // the norm is of the stored value
                    }
                }
#pragma unroll
                for (int i = 0; i < NP; ++i) acc = add2(acc, v[r][c][i]);
            }
            mean[r] = halves_sum(acc);
        }
        lanes_sum<R>(mean, ra.lanes);
        if constexpr (R == 1) {
            if (ra.warps_per_row > 1) warps_sum<1>(mean, ra.warps_per_row, warp_in_row, group + 1, red);
        }
        // Every warp of the row has lifted its part of the stage (one warp: its lanes meet here).
        __syncwarp();
        if (leader) ring.fill(ring.stage, x, second, row0 + ring.stages * step, ra.step_rows, rows, hidden);
        ring.next();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Pair shift = pair(-mean[r] * inv_hidden);
            Pair acc = 0;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                if (FULL || vec0 + c * 32 < ra.vectors) {
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        v[r][c][i] = add2(v[r][c][i], shift);
                        acc = fma2(v[r][c][i], v[r][c][i], acc);
                    }
                }
            }
            rstd[r] = halves_sum(acc);
        }
        lanes_sum<R>(rstd, ra.lanes);
        if constexpr (R == 1) {
            if (ra.warps_per_row > 1) warps_sum<1>(rstd, ra.warps_per_row, warp_in_row, group + 1, red + 16);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) rstd[r] = rsqrtf(fmaf(rstd[r], inv_hidden, epsilon));
        T* out = y + e0;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            if (FULL || vec0 + c * 32 < ra.vectors) {
                Pair wv[NP], bv[NP];
                read_pairs<NP>(wv, ws, vec0 + c * 32, ra.vectors);
                read_pairs<NP>(bv, bs, vec0 + c * 32, ra.vectors);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (R == 1 || r * per_warp + lane_row < left) {
                        const Pair scale = pair(rstd[r]);
#pragma unroll
                        for (int i = 0; i < NP; ++i) v[r][c][i] = fma2(mul2(v[r][c][i], scale), wv[i], bv[i]);
                        *reinterpret_cast<uint4*>(out + r * per_warp * hidden + c * (32 * VEC)) = to_raw<T>(v[r][c]);
                    }
                }
            }
        }
    }
}

// CPT: vectors per lane in the row phase (FULL: exactly the row's). COLS: vectors per thread and row in the column phase.
// partial: [gridDim.x][2][hidden].
template <typename T, int CPT, int COLS, bool FULL, bool FUSED>
__global__ void __launch_bounds__(kBackwardThreads, 1)
layernorm_backward_ring_kernel(T* dx, T* din, float* __restrict__ partial, const T* __restrict__ dy, const T* __restrict__ x,
                               const T* __restrict__ w, const T* residual, long long rows, int hidden, float epsilon, const RingArgs ra,
                               const DropoutArgs args) {
    constexpr int VEC = 16 / sizeof(T), NP = VEC / 2, R = rows_at_once(CPT), RC = kTileVectors / COLS;
    extern __shared__ __align__(128) unsigned char shared[];
    __shared__ ulonglong2 stats[2][kMaxTileRows][2];         // -mean, rstd; -c1, -c2 of the tile's rows, each as a pair of equals
    float* ws = reinterpret_cast<float*>(shared + kVectorsOffset);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int unit = warp / ra.warps_per_row, warp_in_row = warp - unit * ra.warps_per_row;
    const int units = (blockDim.x >> 5) / ra.warps_per_row;
    const int per_warp = 32 / ra.lanes;
    const int lane_row = lane / ra.lanes, vec0 = warp_in_row * (32 * CPT) + (lane & (ra.lanes - 1));
    float* red = reinterpret_cast<float*>(shared + kSumsOffset) + unit * 64;
    launch_dependents();
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    const long long step = static_cast<long long>(gridDim.x) * ra.step_rows;
    const long long first = static_cast<long long>(blockIdx.x) * ra.step_rows;
    Ring ring{};
    ring.row_bytes = static_cast<unsigned>(hidden) * sizeof(T);
    ring.tensor_bytes = ra.step_rows * ring.row_bytes;
    ring.stage_bytes = 2 * ring.tensor_bytes;
    ring.stages = ra.stages;
    ring.full = reinterpret_cast<std::uint64_t*>(shared);
    ring.data = shared + ra.data_offset;
    ring.status = ra.status;
    if (threadIdx.x == 0) {
        ring.init();
        for (int s = 0; s < ra.stages; ++s) ring.fill(s, x, dy, first + s * step, ra.step_rows, rows, hidden);
    }
    stage_vector(ws, w, ra.vectors);
    const HoistedPhilox gen(args);
    // Column phase: with COLS == 1 the threads cover `groups` rows at a time, vector after vector, row after row.
    const int row_group = COLS == 1 ? threadIdx.x / ra.vectors : 0;
    const int column = COLS == 1 ? threadIdx.x - row_group * ra.vectors : threadIdx.x;      // in vectors
    const bool works = COLS > 1 || row_group < ra.groups;
    const unsigned column_bytes = row_group * ring.row_bytes + column * 16, next_rows = ra.groups * ring.row_bytes;
    const unsigned lane_bytes = lane_row * ring.row_bytes + vec0 * 16, next_row = per_warp * ring.row_bytes;
    const int next_elements = ra.groups * hidden;
    __syncthreads();
    Pair wv[NP] = {}, aw[COLS][NP], ab[COLS][NP];            // w of the thread's columns, if they are few: else read where needed
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int i = 0; i < NP; ++i) aw[c][i] = ab[c][i] = 0;
    if (COLS == 1) read_pairs<NP>(wv, ws, column, ra.vectors);

    int buffer = 0;
    for (long long row0 = first; row0 < rows; row0 += step, buffer ^= 1) {
        const int tile_rows = rows - row0 < ra.step_rows ? static_cast<int>(rows - row0) : ra.step_rows;
        const long long e0 = (row0 + row_group) * hidden + column * VEC;       // the thread's first element in the column phase
        const bool whole = tile_rows == ra.step_rows;
        // The residual is needed last: on its way past the ring while the row sums are taken.
        uint4 rp[RC][COLS];
        if (residual != nullptr && works) {
            const T* from = residual + e0;
#pragma unroll
            for (int k = 0; k < RC; ++k, from += next_elements)
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if ((whole || k * ra.groups + row_group < tile_rows) && (COLS == 1 || column + c * blockDim.x < ra.vectors))
                        rp[k][c] = __ldcs(reinterpret_cast<const uint4*>(from + c * blockDim.x * VEC));
        }
        const unsigned char* stage = ring.wait();
        // ---- rows: four sums each
        for (int base = unit * R * per_warp; base < tile_rows; base += units * R * per_warp) {
            const unsigned char* at = stage + base * ring.row_bytes + lane_bytes;
            Pair v[R][CPT][NP];
            uint4 gp[R][CPT];
            float mean[R], sums[3 * R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                Pair acc = 0;
#pragma unroll
                for (int c = 0; c < CPT; ++c) {
                    gp[r][c] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                    for (int i = 0; i < NP; ++i) v[r][c][i] = 0;
                    if ((R == 1 || base + r * per_warp + lane_row < tile_rows) && (FULL || vec0 + c * 32 < ra.vectors)) {
                        gp[r][c] = *reinterpret_cast<const uint4*>(at + ring.tensor_bytes + r * next_row + c * 512);
                        to_pairs<T>(v[r][c], *reinterpret_cast<const uint4*>(at + r * next_row + c * 512));
                    }
#pragma unroll
                    for (int i = 0; i < NP; ++i) acc = add2(acc, v[r][c][i]);
                }
                mean[r] = halves_sum(acc);
            }
            lanes_sum<R>(mean, ra.lanes);
            if constexpr (R == 1) {
                if (ra.warps_per_row > 1) warps_sum<1>(mean, ra.warps_per_row, warp_in_row, unit + 1, red);
            }
            Pair s0[R], s1[R], s2[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                mean[r] *= -inv_hidden;
                s0[r] = s1[r] = s2[r] = 0;
            }
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                if (FULL || vec0 + c * 32 < ra.vectors) {
                    Pair wr[NP];
                    read_pairs<NP>(wr, ws, vec0 + c * 32, ra.vectors);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const Pair shift = pair(mean[r]);
                        Pair g[NP];
                        to_pairs<T>(g, gp[r][c]);
#pragma unroll
                        for (int i = 0; i < NP; ++i) {
                            const Pair d = add2(v[r][c][i], shift), gw = mul2(g[i], wr[i]);
                            s0[r] = fma2(d, d, s0[r]);
                            s1[r] = add2(s1[r], gw);
                            s2[r] = fma2(gw, d, s2[r]);
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                sums[r] = halves_sum(s0[r]);
                sums[R + r] = halves_sum(s1[r]);
                sums[2 * R + r] = halves_sum(s2[r]);
            }
            lanes_sum<3 * R>(sums, ra.lanes);
            if constexpr (R == 1) {
                if (ra.warps_per_row > 1) warps_sum<3>(sums, ra.warps_per_row, warp_in_row, unit + 1, red + 16);
            }
            if (warp_in_row == 0 && (lane & (ra.lanes - 1)) == 0) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int row = base + r * per_warp + lane_row;
                    const float rstd = rsqrtf(fmaf(sums[r], inv_hidden, epsilon));
                    if (row < tile_rows) {
                        stats[buffer][row][0] = make_ulonglong2(pair(mean[r]), pair(rstd));
                        stats[buffer][row][1] = make_ulonglong2(pair(-sums[R + r] * inv_hidden), pair(-(sums[2 * R + r] * inv_hidden * rstd)));
                    }
                }
            }
        }
        __syncthreads();
        // Every thread is past the columns of the tile before: its stage is free.
        if (threadIdx.x == 0 && !ring.failed && row0 != first)
            ring.fill(ring.stage == 0 ? ring.stages - 1 : ring.stage - 1, x, dy, row0 + (ring.stages - 1) * step, ra.step_rows, rows, hidden);
        // ---- columns
        auto columns = [&](auto all_rows) {
            const unsigned char* at = stage + column_bytes;
            const ulonglong2(*st)[2] = stats[buffer] + row_group;
            long long e = e0;
#pragma unroll
            for (int k = 0; k < RC; ++k, at += next_rows, st += ra.groups, e += next_elements) {
                if (all_rows.value || k * ra.groups + row_group < tile_rows) {
                    const ulonglong2 norm = st[0][0], cs = st[0][1];
#pragma unroll
                    for (int c = 0; c < COLS; ++c) {
                        if (COLS == 1 || column + c * blockDim.x < ra.vectors) {
                            Pair v[NP], g[NP], out[NP];
                            to_pairs<T>(v, *reinterpret_cast<const uint4*>(at + c * blockDim.x * 16));
                            to_pairs<T>(g, *reinterpret_cast<const uint4*>(at + ring.tensor_bytes + c * blockDim.x * 16));
#pragma unroll
                            for (int i = 0; i < NP; ++i) out[i] = 0;
                            if (residual != nullptr) to_pairs<T>(out, rp[k][c]);
                            if constexpr (COLS > 1) read_pairs<NP>(wv, ws, column + c * blockDim.x, ra.vectors);
#pragma unroll
                            for (int i = 0; i < NP; ++i) {
                                const Pair xh = mul2(add2(v[i], norm.x), norm.y);
                                out[i] = fma2(norm.y, fma2(xh, cs.y, fma2(g[i], wv[i], cs.x)), out[i]);
                                aw[c][i] = fma2(g[i], xh, aw[c][i]);
                                ab[c][i] = add2(ab[c][i], g[i]);
                            }
                            *reinterpret_cast<uint4*>(dx + e + c * blockDim.x * VEC) = to_raw<T>(out);
                            if constexpr (FUSED) {
                                if (args.threshold != 0) drop_pairs<NP>(out, gen, e + c * blockDim.x * VEC, args);
                                *reinterpret_cast<uint4*>(din + e + c * blockDim.x * VEC) = to_raw<T>(out);
                            }
                        }
                    }
                }
            }
        };
        if (works) {
            if (whole) columns(std::true_type{});
            else columns(std::false_type{});
        }
        ring.next();
    }

    // One partial row of dw and of db per CTA: its row groups add up one after the other, in the memory of the ring, whose copies
    // have all been waited for. Where a wait ran out they may not have come, and the rows are worth nothing.
    if (__syncthreads_or(ring.failed)) return;
    float* out_w = partial + static_cast<long long>(blockIdx.x) * 2 * hidden;
    Pair* joined = reinterpret_cast<Pair*>(shared + ra.data_offset);           // [pair][dw, db][vector]: no bank conflicts
    const int groups = COLS == 1 ? ra.groups : 1;
    for (int k = 0; k < groups; ++k) {
        if (k > 0) __syncthreads();
        if (works && row_group == k) {
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const int vec = column + c * blockDim.x;
                if (vec < ra.vectors) {
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const int at = (i * 2) * ra.vectors + vec;
                        Pair tw = aw[c][i], tb = ab[c][i];
                        if (k > 0) {
                            tw = add2(joined[at], tw);
                            tb = add2(joined[at + ra.vectors], tb);
                        }
                        if (k + 1 < groups) {
                            joined[at] = tw;
                            joined[at + ra.vectors] = tb;
                        } else {
                            *reinterpret_cast<Pair*>(out_w + vec * VEC + 2 * i) = tw;
                            *reinterpret_cast<Pair*>(out_w + hidden + vec * VEC + 2 * i) = tb;
                        }
                    }
                }
            }
        }
    }
}

}  // namespace ring_kernels
