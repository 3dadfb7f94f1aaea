// Layer norm of rows that are whole 16-byte vectors. Included by layernorm.cu only.
//
// What limits these kernels once memory is read ahead is the number of instructions: at the rate memory delivers 16-bit
// elements an SM has about 20 issue slots for each. Hence
//  * rows come through rings of stages in shared memory, filled by bulk copies (consecutive rows are contiguous: one copy per
//    tensor and stage), so that nothing but one thread per ring deals with memory and its latency;
//  * arithmetic is on pairs (fma / mul / add .f32x2): one issue slot for two elements;
//  * a row is summed by one warp wherever 128 vectors hold it, four vectors per lane: the shuffles of a sum are shared by up to
//    32 elements of a lane, and by up to four rows where rows are short;
//  * w and b are kept in shared memory as fp32: no conversion per row.
//
// Forward: every group of warps walks rows through a ring of its own. Backward: a CTA takes tiles of rows in two phases, rows
// first (a warp group per row: mean, rstd and the two sums of dx, left in shared memory), then columns (a thread per vector of
// columns: dx, and the running dw and db of its columns in registers).
#pragma once

namespace ring_kernels {

constexpr int kMaxStages = 4;
constexpr int kLaneVectors = 4;          // vectors of a row step that a lane holds: CPT vectors of R = 4 / CPT rows
constexpr int kForwardThreads = 1024;    // one CTA per SM (64 registers)
constexpr int kFusedThreads = 640;       // the fused forward needs up to 96
constexpr int kBackwardThreads = 512;    // per SM: two CTAs of 256 or one of 512 (128 registers)
constexpr int kMaxTileRows = 256;

using Pair = unsigned long long;         // two fp32 values in a 64-bit register

__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ Pair pair(float a) { return pair(a, a); }
__device__ __forceinline__ float2 both(Pair p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float halves_sum(Pair p) {
    const float2 f = both(p);
    return f.x + f.y;
}

template <typename T> __device__ __forceinline__ Pair pair_of(std::uint32_t two);
template <> __device__ __forceinline__ Pair pair_of<__half>(std::uint32_t two) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
    return pair(f.x, f.y);
}
template <> __device__ __forceinline__ Pair pair_of<__nv_bfloat16>(std::uint32_t two) {
    return pair(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ std::uint32_t two_of(Pair p);
template <> __device__ __forceinline__ std::uint32_t two_of<__half>(Pair p) {
    const float2 f = both(p);
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const std::uint32_t*>(&h);
}
template <> __device__ __forceinline__ std::uint32_t two_of<__nv_bfloat16>(Pair p) {
    const float2 f = both(p);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const std::uint32_t*>(&h);
}

// A 16-byte vector as pairs, and back (one rounding to T).
template <typename T>
__device__ __forceinline__ void to_pairs(Pair (&p)[8 / sizeof(T)], const uint4& raw) {
    if constexpr (sizeof(T) == 4) {
        p[0] = pair(__uint_as_float(raw.x), __uint_as_float(raw.y));
        p[1] = pair(__uint_as_float(raw.z), __uint_as_float(raw.w));
    } else {
        p[0] = pair_of<T>(raw.x);
        p[1] = pair_of<T>(raw.y);
        p[2] = pair_of<T>(raw.z);
        p[3] = pair_of<T>(raw.w);
    }
}
template <typename T>
__device__ __forceinline__ uint4 to_raw(const Pair (&p)[8 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        const float2 a = both(p[0]), b = both(p[1]);
        return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    } else {
        return make_uint4(two_of<T>(p[0]), two_of<T>(p[1]), two_of<T>(p[2]), two_of<T>(p[3]));
    }
}
template <typename T>
__device__ __forceinline__ void drop_pairs(Pair (&p)[8 / sizeof(T)], const Philox& gen, long long e, const DropoutArgs& args) {
    constexpr int VEC = 16 / sizeof(T);
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
        const float2 f = both(p[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
    drop_vec<VEC>(v, gen, e, args);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) p[i] = pair(v[2 * i], v[2 * i + 1]);
}

// Makes packed values opaque to the optimiser, so that it converts them again at their next use instead of keeping twice as many
// fp32 registers alive from one use to the next.
__device__ __forceinline__ void keep_packed(uint4& v) { asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)); }

// A ring of stages. A wait that runs out sets the library's status word; the CTA then goes on with what is there (every barrier
// is still met, nothing is written out of bounds) and waits no more.
struct Ring {
    unsigned char* data;
    std::uint64_t* full;
    unsigned int* status;
    unsigned stage_bytes, tensor_bytes, row_bytes;
    int stages, stage;
    std::uint32_t parity;
    bool failed;

    __device__ __forceinline__ void init() const {   // by one thread, before the CTA's first barrier
        for (int s = 0; s < stages; ++s) sm100::mbar_init(&full[s], 1);
        sm100::mbar_init_fence();
    }
    // Rows row0 .. row0 + step_rows of a and b (b may be null) into stage s, as far as there are such rows.
    template <typename T>
    __device__ __forceinline__ void fill(int s, const T* a, const T* b, long long row0, int step_rows, long long rows, int hidden) const {
        if (row0 >= rows) return;
        const unsigned n = static_cast<unsigned>(rows - row0 < step_rows ? rows - row0 : step_rows) * row_bytes;
        sm100::mbar_expect_tx(&full[s], b != nullptr ? 2 * n : n);
        sm100::bulk_load_1d(data + s * stage_bytes, a + row0 * hidden, n, &full[s]);
        if (b != nullptr) sm100::bulk_load_1d(data + s * stage_bytes + tensor_bytes, b + row0 * hidden, n, &full[s]);
    }
    __device__ __forceinline__ const unsigned char* wait() {
        if (!failed && !sm100::mbar_wait(&full[stage], parity)) {
            failed = true;
            atomicExch(status, 5u);
        }
        return data + stage * stage_bytes;
    }
    __device__ __forceinline__ void next() {
        if (++stage == stages) { stage = 0; parity ^= 1u; }
    }
};

// Layout of a launch (make_ring_plan): vectors per row, lanes per row (fewer than 32 where a warp holds several rows), warps
// per row, rows a step or tile has, groups (forward: warp groups; backward: row groups of the column phase).
struct RingArgs {
    unsigned int* status;
    int vectors, lanes, warps_per_row, step_rows, groups, stages;
    unsigned data_offset;               // of the ring(s) in shared memory
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

// w or b (null: zeros) as fp32 in shared memory.
template <typename T>
__device__ __forceinline__ void stage_vector(float* to, const T* from, int vectors) {
    constexpr int VEC = 16 / sizeof(T), NP = VEC / 2;
    for (int i = threadIdx.x; i < vectors; i += blockDim.x) {
        Pair v[NP];
        to_pairs<T>(v, from != nullptr ? *reinterpret_cast<const uint4*>(from + i * VEC) : make_uint4(0u, 0u, 0u, 0u));
#pragma unroll
        for (int j = 0; j < NP / 2; ++j) reinterpret_cast<ulonglong2*>(to + i * VEC)[j] = make_ulonglong2(v[2 * j], v[2 * j + 1]);
    }
}
template <int NP>
__device__ __forceinline__ void read_pairs(Pair (&p)[NP], const float* from) {
    const ulonglong2* v = reinterpret_cast<const ulonglong2*>(from);
#pragma unroll
    for (int i = 0; i < NP / 2; ++i) {
        const ulonglong2 u = v[i];
        p[2 * i] = u.x;
        p[2 * i + 1] = u.y;
    }
}

// Shared memory: [barriers 1 KB][sums of multi-warp rows 2 KB][w][b][rings]
constexpr unsigned kSumsOffset = 1024, kVectorsOffset = 3072;

template <typename T, int CPT, bool FUSED>
__global__ void __launch_bounds__(FUSED ? kFusedThreads : kForwardThreads, 1)
layernorm_forward_ring_kernel(T* __restrict__ y, T* sum, const T* x, const T* residual, const T* __restrict__ w, const T* __restrict__ b,
                              long long rows, int hidden, float epsilon, const RingArgs ra, const DropoutArgs args) {
    constexpr int VEC = 16 / sizeof(T), NP = VEC / 2, R = kLaneVectors / CPT;
    extern __shared__ __align__(128) unsigned char shared[];
    float* ws = reinterpret_cast<float*>(shared + kVectorsOffset);
    float* bs = ws + hidden;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = warp / ra.warps_per_row, warp_in_row = warp - group * ra.warps_per_row;
    const int per_warp = 32 / ra.lanes;                      // rows side by side in a warp
    const int lane_row = lane / ra.lanes, vec0 = warp_in_row * 32 + (lane & (ra.lanes - 1)), vec_step = ra.warps_per_row * ra.lanes;
    float* red = reinterpret_cast<float*>(shared + kSumsOffset) + group * 32;
    const long long step = static_cast<long long>(gridDim.x) * ra.groups * ra.step_rows;
    const long long first = (static_cast<long long>(blockIdx.x) * ra.groups + group) * ra.step_rows;
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    const bool leader = warp_in_row == 0 && lane == 0;
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
    const Philox gen(args);
    __syncthreads();

    for (long long row0 = first; row0 < rows; row0 += step) {
        const unsigned char* stage = ring.wait();
        uint4 xp[R][CPT];
        float mean[R], rstd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int in_step = r * per_warp + lane_row;
            Pair acc = 0;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const int vec = vec0 + c * vec_step;
                const bool in = row0 + in_step < rows && vec < ra.vectors;
                xp[r][c] = make_uint4(0u, 0u, 0u, 0u);      // a stage keeps what an earlier step left there
                if (in) {
                    xp[r][c] = *reinterpret_cast<const uint4*>(stage + in_step * ring.row_bytes + vec * 16);
                    Pair v[NP];
                    to_pairs<T>(v, xp[r][c]);
                    if constexpr (FUSED) {
                        const long long e = (row0 + in_step) * hidden + vec * VEC;
                        if (args.threshold != 0) drop_pairs<T>(v, gen, e, args);
                        Pair res[NP];
                        to_pairs<T>(res, *reinterpret_cast<const uint4*>(stage + ring.tensor_bytes + in_step * ring.row_bytes + vec * 16));
#pragma unroll
                        for (int i = 0; i < NP; ++i) v[i] = add2(v[i], res[i]);
                        xp[r][c] = to_raw<T>(v);
                        *reinterpret_cast<uint4*>(sum + e) = xp[r][c];
                        to_pairs<T>(v, xp[r][c]);            // the norm is of the stored value
                    }
#pragma unroll
                    for (int i = 0; i < NP; ++i) acc = add2(acc, v[i]);
                }
                keep_packed(xp[r][c]);
            }
            mean[r] = halves_sum(acc);
        }
        lanes_sum<R>(mean, ra.lanes);
        if constexpr (R == 1) {
            if (ra.warps_per_row > 1) warps_sum<1>(mean, ra.warps_per_row, warp_in_row, group, red);
        }
        // Every warp of the row has lifted its part of the stage (one warp: its lanes meet here).
        __syncwarp();
        if (leader) ring.fill(ring.stage, x, second, row0 + ring.stages * step, ra.step_rows, rows, hidden);
        ring.next();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] *= -inv_hidden;
            const Pair shift = pair(mean[r]);
            Pair acc = 0;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                if (vec0 + c * vec_step < ra.vectors) {
                    Pair v[NP];
                    to_pairs<T>(v, xp[r][c]);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        v[i] = add2(v[i], shift);
                        acc = fma2(v[i], v[i], acc);
                    }
                }
                keep_packed(xp[r][c]);
            }
            rstd[r] = halves_sum(acc);
        }
        lanes_sum<R>(rstd, ra.lanes);
        if constexpr (R == 1) {
            if (ra.warps_per_row > 1) warps_sum<1>(rstd, ra.warps_per_row, warp_in_row, group, red + 16);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) rstd[r] = rsqrtf(fmaf(rstd[r], inv_hidden, epsilon));
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int vec = vec0 + c * vec_step;
            if (vec < ra.vectors) {
                Pair wv[NP], bv[NP];
                read_pairs<NP>(wv, ws + vec * VEC);
                read_pairs<NP>(bv, bs + vec * VEC);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int in_step = r * per_warp + lane_row;
                    if (row0 + in_step < rows) {
                        const Pair shift = pair(mean[r]), scale = pair(rstd[r]);
                        Pair v[NP];
                        to_pairs<T>(v, xp[r][c]);
#pragma unroll
                        for (int i = 0; i < NP; ++i) v[i] = fma2(mul2(add2(v[i], shift), scale), wv[i], bv[i]);
                        *reinterpret_cast<uint4*>(y + (row0 + in_step) * hidden + vec * VEC) = to_raw<T>(v);
                    }
                }
            }
        }
    }
}

// CPT: vectors per lane in the row phase. COLS: vectors per thread and row in the column phase. partial: [gridDim.x][2][hidden].
template <typename T, int CPT, int COLS, bool FUSED>
__global__ void __launch_bounds__(kBackwardThreads, 1)
layernorm_backward_ring_kernel(T* dx, T* din, float* __restrict__ partial, const T* __restrict__ dy, const T* __restrict__ x,
                               const T* __restrict__ w, const T* residual, long long rows, int hidden, float epsilon, const RingArgs ra,
                               const DropoutArgs args) {
    constexpr int VEC = 16 / sizeof(T), NP = VEC / 2, R = kLaneVectors / CPT, RC = kLaneVectors / COLS;
    extern __shared__ __align__(128) unsigned char shared[];
    __shared__ float4 stats[2][kMaxTileRows];                // -mean, rstd, -c1, -c2 of the tile's rows
    float* ws = reinterpret_cast<float*>(shared + kVectorsOffset);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int unit = warp / ra.warps_per_row, warp_in_row = warp - unit * ra.warps_per_row;
    const int units = (blockDim.x >> 5) / ra.warps_per_row;
    const int per_warp = 32 / ra.lanes;
    const int lane_row = lane / ra.lanes, vec0 = warp_in_row * 32 + (lane & (ra.lanes - 1)), vec_step = ra.warps_per_row * ra.lanes;
    float* red = reinterpret_cast<float*>(shared + kSumsOffset) + unit * 64;
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
    const Philox gen(args);
    // Column phase: with COLS == 1 the threads cover `groups` rows at a time, vector after vector, row after row.
    const int row_group = COLS == 1 ? threadIdx.x / ra.vectors : 0;
    const int column = COLS == 1 ? threadIdx.x - row_group * ra.vectors : threadIdx.x;      // in vectors
    const bool works = COLS > 1 || row_group < ra.groups;
    __syncthreads();
    Pair wv[COLS][NP], aw[COLS][NP], ab[COLS][NP];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const int vec = column + c * blockDim.x;
        if (vec < ra.vectors) read_pairs<NP>(wv[c], ws + vec * VEC);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (vec >= ra.vectors) wv[c][i] = 0;
            aw[c][i] = 0;
            ab[c][i] = 0;
        }
    }

    int buffer = 0;
    for (long long row0 = first; row0 < rows; row0 += step, buffer ^= 1) {
        const int tile_rows = rows - row0 < ra.step_rows ? static_cast<int>(rows - row0) : ra.step_rows;
        // The residual is needed last: on its way past the ring while the row sums are taken.
        uint4 rp[RC][COLS];
#pragma unroll
        for (int k = 0; k < RC; ++k)
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const int row = k * ra.groups + row_group, vec = column + c * blockDim.x;
                rp[k][c] = residual != nullptr && works && row < tile_rows && vec < ra.vectors
                               ? __ldcs(reinterpret_cast<const uint4*>(residual + (row0 + row) * hidden + vec * VEC)) : make_uint4(0u, 0u, 0u, 0u);
            }
        const unsigned char* stage = ring.wait();
        // ---- rows: four sums each
        for (int base = unit * R * per_warp; base < tile_rows; base += units * R * per_warp) {
            uint4 xp[R][CPT], gp[R][CPT];
            float mean[R], sums[3 * R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int row = base + r * per_warp + lane_row;
                Pair acc = 0;
#pragma unroll
                for (int c = 0; c < CPT; ++c) {
                    const int vec = vec0 + c * vec_step;
                    const unsigned char* at = stage + row * ring.row_bytes + vec * 16;
                    const bool in = row < tile_rows && vec < ra.vectors;
                    xp[r][c] = in ? *reinterpret_cast<const uint4*>(at) : make_uint4(0u, 0u, 0u, 0u);
                    gp[r][c] = in ? *reinterpret_cast<const uint4*>(at + ring.tensor_bytes) : make_uint4(0u, 0u, 0u, 0u);
                    Pair v[NP];
                    to_pairs<T>(v, xp[r][c]);
#pragma unroll
                    for (int i = 0; i < NP; ++i) acc = add2(acc, v[i]);
                    keep_packed(xp[r][c]);
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
                const int vec = vec0 + c * vec_step;
                if (vec < ra.vectors) {
                    Pair wr[NP];
                    read_pairs<NP>(wr, ws + vec * VEC);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const Pair shift = pair(mean[r]);
                        Pair v[NP], g[NP];
                        to_pairs<T>(v, xp[r][c]);
                        to_pairs<T>(g, gp[r][c]);
#pragma unroll
                        for (int i = 0; i < NP; ++i) {
                            const Pair d = add2(v[i], shift), gw = mul2(g[i], wr[i]);
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
                    if (row < tile_rows) stats[buffer][row] = make_float4(mean[r], rstd, -sums[R + r] * inv_hidden, -(sums[2 * R + r] * inv_hidden * rstd));
                }
            }
        }
        __syncthreads();
        // Every thread is past the columns of the tile before: its stage is free.
        if (threadIdx.x == 0 && row0 != first)
            ring.fill(ring.stage == 0 ? ring.stages - 1 : ring.stage - 1, x, dy, row0 + (ring.stages - 1) * step, ra.step_rows, rows, hidden);
        // ---- columns
        if (works) {
#pragma unroll
            for (int k = 0; k < RC; ++k) {
                const int row = k * ra.groups + row_group;
                if (row < tile_rows) {
                    const float4 st = stats[buffer][row];
                    const Pair shift = pair(st.x), rstd = pair(st.y), c1 = pair(st.z), c2 = pair(st.w);
#pragma unroll
                    for (int c = 0; c < COLS; ++c) {
                        const int vec = column + c * blockDim.x;
                        if (vec < ra.vectors) {
                            const unsigned char* at = stage + row * ring.row_bytes + vec * 16;
                            const long long e = (row0 + row) * hidden + vec * VEC;
                            Pair v[NP], g[NP], out[NP];
                            to_pairs<T>(v, *reinterpret_cast<const uint4*>(at));
                            to_pairs<T>(g, *reinterpret_cast<const uint4*>(at + ring.tensor_bytes));
                            to_pairs<T>(out, rp[k][c]);
#pragma unroll
                            for (int i = 0; i < NP; ++i) {
                                const Pair xh = mul2(add2(v[i], shift), rstd);
                                out[i] = fma2(rstd, fma2(xh, c2, fma2(g[i], wv[c][i], c1)), out[i]);
                                aw[c][i] = fma2(g[i], xh, aw[c][i]);
                                ab[c][i] = add2(ab[c][i], g[i]);
                            }
                            *reinterpret_cast<uint4*>(dx + e) = to_raw<T>(out);
                            if constexpr (FUSED) {
                                if (args.threshold != 0) drop_pairs<T>(out, gen, e, args);
                                *reinterpret_cast<uint4*>(din + e) = to_raw<T>(out);
                            }
                        }
                    }
                }
            }
        }
        ring.next();
    }

    // One partial row of dw and of db per CTA: its row groups add up one after the other, in the memory of the ring, whose copies
    // have all been waited for.
    float* out_w = partial + static_cast<long long>(blockIdx.x) * 2 * hidden;
    float* joined = reinterpret_cast<float*>(shared + ra.data_offset);
    const int groups = COLS == 1 ? ra.groups : 1;
    for (int k = 0; k < groups; ++k) {
        __syncthreads();
        if (works && row_group == k) {
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const int vec = column + c * blockDim.x;
                if (vec < ra.vectors) {
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const int at = (i * 2) * ra.vectors + vec;       // pairs, one per thread: no bank conflicts
                        Pair* s = reinterpret_cast<Pair*>(joined);
                        Pair tw = aw[c][i], tb = ab[c][i];
                        if (k > 0) {
                            tw = add2(s[at], tw);
                            tb = add2(s[at + ra.vectors], tb);
                        }
                        if (k + 1 < groups) {
                            s[at] = tw;
                            s[at + ra.vectors] = tb;
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
