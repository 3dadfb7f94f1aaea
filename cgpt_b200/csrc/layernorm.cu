// Layer norm forward and backward, and the same fused with dropout and the residual add in front of it, for sm_100a.
//
//   forward    mean = sum x / H, var = sum (x - mean)^2 / H, rstd = 1 / sqrt(var + eps), y = (x - mean) rstd w + b
//   backward   xh = (x - mean) rstd, g = dy w:   dx = rstd (g - mean(g) - xh mean(g xh)) (+ residual)
//              dw = sum_rows dy xh,  db = sum_rows dy
//   fused      x = residual + dropout(in), rounded to the storage type and written, then the norm of the rounded value;
//              backward: d = dsum + dx, dresidual = d, din = dropout map of d
//
// The variance is taken around the mean (a second pass over values that are already on the chip): sum x^2 - mean^2 loses
// everything for a row whose offset is large against its spread. The backward recomputes mean and rstd from x, which it reads
// in any case, so the forward stores no statistics. Sums are fp32; a row's dw and db contributions are added in a fixed order
// (per-CTA partial rows, then one pass over them), so results repeat bit for bit.
//
// Memory-bound: 2 * H * sizeof(T) bytes per row forward, 3 backward (+1 with a residual), 4 and 5 for the fused pair.
#include <type_traits>

#include "bulk_ring.cuh"
#include "dependent_launch.cuh"
#include "philox.cuh"
#include "launch_counter.h"

namespace cgpt {

unsigned int* tc_status_device_ptr();   // gemm.cu: status word raised when a bounded device-side wait runs out

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Sum of `vals` over the CTA; every thread gets the totals. Contains barriers.
template <int NV, int WARPS>
__device__ __forceinline__ void block_sum(float (&vals)[NV], float* smem /* [WARPS * NV] */) {
#pragma unroll
    for (int i = 0; i < NV; ++i) vals[i] = warp_sum(vals[i]);
    __syncthreads();   // the previous call's totals have been read
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) smem[(threadIdx.x >> 5) * NV + i] = vals[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) acc += smem[w * NV + i];
        vals[i] = acc;
    }
}

// The element-wise formulas, with every fused multiply-add written out: left to the compiler, the contractions differ between
// instantiations, and the fused operators would not give the bits of their parts.
__device__ __forceinline__ float normalised(float x, float mean, float rstd) { return __fmul_rn(x - mean, rstd); }
__device__ __forceinline__ float norm_dx(float dy, float w, float xh, float rstd, float c1, float c2, float residual) {
    return fmaf(rstd, fmaf(-xh, c2, fmaf(dy, w, -c1)), residual);
}
// sums of (x - mean)^2, g and g (x - mean) with g = dy w
__device__ __forceinline__ void norm_sums(float (&s)[3], float dy, float w, float d) {
    s[0] = fmaf(d, d, s[0]);
    s[1] = fmaf(dy, w, s[1]);
    s[2] = fmaf(__fmul_rn(dy, w), d, s[2]);
}

// Sums NV values over a warp. Halves the set of values a lane is responsible for while lanes still differ in what they hold, so
// NV = 4 takes 6 shuffles and NV = 12 takes 18 (5 NV one value at a time). Afterwards every lane holds kCount totals, in
// v[0 .. kCount); which ones, lane bits 4 and 3 say.
template <int NV>
struct WarpSums {
    static constexpr int kFirst = NV % 2 == 0 ? NV / 2 : NV;
    static constexpr int kCount = NV % 4 == 0 ? NV / 4 : kFirst;
    // A lane of those that hold value i.
    static __device__ __forceinline__ constexpr int holder_of(int i) {
        int l = 0;
        if (NV % 2 == 0 && i >= NV / 2) { l += 16; i -= NV / 2; }
        if (NV % 4 == 0 && i >= NV / 4) l += 8;
        return l;
    }
    static __device__ __forceinline__ void reduce(float (&v)[NV], int lane) {
        if constexpr (NV % 2 == 0) {
            const bool up = (lane & 16) != 0;
#pragma unroll
            for (int i = 0; i < NV / 2; ++i) {
                const float send = up ? v[i] : v[i + NV / 2], keep = up ? v[i + NV / 2] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 16);
        }
        if constexpr (NV % 4 == 0) {
            const bool up = (lane & 8) != 0;
#pragma unroll
            for (int i = 0; i < NV / 4; ++i) {
                const float send = up ? v[i] : v[i + NV / 4], keep = up ? v[i + NV / 4] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 8);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kFirst; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 8);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < kCount; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        }
    }
    // Every lane gets every total (and has it already where nothing was halved).
    static __device__ __forceinline__ void broadcast(float (&v)[NV]) {
        if constexpr (NV % 2 == 0) {
            float t[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) t[i] = __shfl_sync(0xffffffffu, v[i % kCount], holder_of(i));
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = t[i];
        }
    }
};

// ------------------------------------------------------------------------------------------ rows of any length
// One CTA per row, the row read again (from L1/L2) for every pass over it. Any H, any alignment. Element by element, and fused a
// generator block for every element: 4096 x 16384 bf16 takes 141 us forward, 406 backward, 372 and 617 fused, 3.4 to 6.5 times the
// bytes' time. These rows are longer than rings hold.
template <typename T, bool FUSED>
__global__ void __launch_bounds__(kThreads)
layernorm_forward_any_kernel(T* __restrict__ y, T* sum, const T* x, const T* residual, const T* __restrict__ w,
                             const T* __restrict__ b, long long rows, long long hidden, float epsilon, const DropoutArgs args) {
    __shared__ float red[kWarps];
    const Philox gen(args);
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = (FUSED ? sum : x) + row * hidden;
        float s[1] = {0.f};
        for (long long c = threadIdx.x; c < hidden; c += kThreads) {
            if constexpr (FUSED) {
                const long long e = row * hidden + c;
                float v = to_f32<T>(x[e]);
                if (args.threshold != 0) v = apply_one(v, gen, e, args);
                const T stored = from_f32<T>(v + to_f32<T>(residual[e]));
                sum[e] = stored;             // read again below by this thread only
                s[0] += to_f32<T>(stored);
            } else {
                s[0] += to_f32<T>(in[c]);
            }
        }
        block_sum<1, kWarps>(s, red);
        const float mean = s[0] * inv_hidden;
        s[0] = 0.f;
        for (long long c = threadIdx.x; c < hidden; c += kThreads) {
            const float d = to_f32<T>(in[c]) - mean;
            s[0] = fmaf(d, d, s[0]);
        }
        block_sum<1, kWarps>(s, red);
        const float rstd = rsqrtf(fmaf(s[0], inv_hidden, epsilon));
        for (long long c = threadIdx.x; c < hidden; c += kThreads)
            y[row * hidden + c] = from_f32<T>(fmaf(normalised(to_f32<T>(in[c]), mean, rstd), to_f32<T>(w[c]), b != nullptr ? to_f32<T>(b[c]) : 0.f));
    }
}

// dx (FUSED: dresidual and din) of one row per CTA; the row's (mean, rstd) go to `stats` for the column sums.
template <typename T, bool FUSED>
__global__ void __launch_bounds__(kThreads)
layernorm_backward_any_kernel(T* dx, T* din, float2* __restrict__ stats, const T* __restrict__ dy, const T* __restrict__ x,
                              const T* __restrict__ w, const T* residual, long long rows, long long hidden, float epsilon,
                              const DropoutArgs args) {
    __shared__ float red[kWarps * 3];
    const Philox gen(args);
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * hidden;
        const T* gr = dy + row * hidden;
        float m[1] = {0.f};
        for (long long c = threadIdx.x; c < hidden; c += kThreads) m[0] += to_f32<T>(xr[c]);
        block_sum<1, kWarps>(m, red);
        const float mean = m[0] * inv_hidden;
        float s[3] = {0.f, 0.f, 0.f};   // sum (x - mean)^2, sum g, sum g (x - mean)
        for (long long c = threadIdx.x; c < hidden; c += kThreads) norm_sums(s, to_f32<T>(gr[c]), to_f32<T>(w[c]), to_f32<T>(xr[c]) - mean);
        block_sum<3, kWarps>(s, red);
        const float rstd = rsqrtf(fmaf(s[0], inv_hidden, epsilon));
        const float c1 = s[1] * inv_hidden, c2 = s[2] * inv_hidden * rstd;
        for (long long c = threadIdx.x; c < hidden; c += kThreads) {
            const long long e = row * hidden + c;
            const float d = norm_dx(to_f32<T>(gr[c]), to_f32<T>(w[c]), normalised(to_f32<T>(xr[c]), mean, rstd), rstd, c1, c2,
                                    residual != nullptr ? to_f32<T>(residual[e]) : 0.f);
            dx[e] = from_f32<T>(d);
            if constexpr (FUSED) din[e] = from_f32<T>(args.threshold != 0 ? apply_one(d, gen, e, args) : d);
        }
        if (threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
    }
}

// Column sums of dy * xh and dy over a share of the rows: 32 columns and 8 row lanes per CTA, rows split over blockIdx.y.
// partial: [splits][2][hidden].
template <typename T>
__global__ void __launch_bounds__(kThreads)
layernorm_columns_any_kernel(float* __restrict__ partial, const T* __restrict__ dy, const T* __restrict__ x,
                             const float2* __restrict__ stats, long long rows, long long hidden) {
    __shared__ float tile[2][kWarps][33];
    launch_dependents();
    const int lane = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const long long col = static_cast<long long>(blockIdx.x) * 32 + lane;
    const long long share = (rows + gridDim.y - 1) / gridDim.y;
    const long long first = blockIdx.y * share, last = first + share < rows ? first + share : rows;
    float aw = 0.f, ab = 0.f;
    if (col < hidden) {
        for (long long r = first + rl; r < last; r += kWarps) {
            const float2 st = stats[r];
            const float g = to_f32<T>(dy[r * hidden + col]);
            aw = fmaf(g, normalised(to_f32<T>(x[r * hidden + col]), st.x, st.y), aw);
            ab += g;
        }
    }
    tile[0][rl][lane] = aw;
    tile[1][rl][lane] = ab;
    __syncthreads();
    if (rl < 2 && col < hidden) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) t += tile[rl][k][lane];
        partial[(static_cast<long long>(blockIdx.y) * 2 + rl) * hidden + col] = t;
    }
}

// dw and db from `parts` partial rows ([parts][2][hidden]) in a fixed order: 32 columns, 32 row lanes per CTA; blockIdx.y
// chooses dw or db.
template <typename T>
__global__ void __launch_bounds__(1024)
layernorm_reduce_kernel(T* dw, T* db, const float* partial, int parts, long long hidden) {
    __shared__ float tile[32][33];
    const int lane = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const long long col = static_cast<long long>(blockIdx.x) * 32 + lane;
    float acc = 0.f;
    wait_for_previous();
    if (col < hidden)
        for (int p = rl; p < parts; p += 32) acc += partial[(static_cast<long long>(p) * 2 + blockIdx.y) * hidden + col];
    tile[rl][lane] = acc;
    __syncthreads();
    if (rl == 0 && col < hidden) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) t += tile[r][lane];
        (blockIdx.y == 0 ? dw : db)[col] = from_f32<T>(t);
    }
}

#include "layernorm_ring.cuh"
#include "layernorm_loose.cuh"

// How a call's rows are laid out. It follows from the sizes and the alignment of all its tensors alone, not from which operator is
// called, so that the fused operators give the bits of their parts for tensors of like alignment.
enum class Form { kAny, kLoose, kRing };

constexpr std::size_t kSmemPerSm = 227 * 1024;

// Where the rings begin behind `vectors` fp32 vectors.
std::size_t vectors_end(std::size_t hidden, std::size_t vectors) { return ring_kernels::kVectorsOffset + (vectors * hidden * sizeof(float) + 127) / 128 * 128; }

// Rings take rows of which shared memory holds two stages of both tensors of the fused forward beside w and b, and of which a
// CTA of the backward holds a row (14 k 16-bit or 8192 fp32 elements). Others take the loose form up to 8192 elements.
Form form_of(std::size_t hidden, std::size_t elem, bool vector) {
    if (vector && hidden * elem % 16 == 0)
        return hidden * elem / 16 <= ring_kernels::kTileVectors * ring_kernels::kBackwardThreads && vectors_end(hidden, 2) + 4 * hidden * elem <= kSmemPerSm ? Form::kRing : Form::kAny;
    const std::size_t row = hidden * elem + loose_kernels::kSlack + 128;      // the backward: two stages of three tensors beside w
    return hidden <= loose_kernels::kMostColumns * loose_kernels::kBackwardThreads &&
                   loose_kernels::kVectorsOffset + hidden * sizeof(float) + 6 * row + loose_kernels::kStatsBytes + 256 <= kSmemPerSm ? Form::kLoose : Form::kAny;
}

struct RingPlan {
    ring_kernels::RingArgs args;
    int cpt, cols, threads;
    bool full;        // the lanes of a row hold exactly its vectors
    unsigned grid;
    std::size_t smem;
};

// Lanes and warps of a row whose lanes hold up to most_cpt vectors.
RingPlan plan_row(std::size_t hidden, std::size_t elem, int most_cpt) {
    RingPlan p{};
    auto& a = p.args;
    const int v = static_cast<int>(hidden * elem / 16);
    a.vectors = v;
    a.lanes = 32;
    while (a.lanes / 2 >= v && a.lanes > 1) a.lanes /= 2;
    p.cpt = 1;
    while (p.cpt < most_cpt && 32 * p.cpt < v) p.cpt *= 2;
    a.warps_per_row = 1;
    while (a.warps_per_row * 32 * p.cpt < v) a.warps_per_row *= 2;
    p.full = a.warps_per_row * a.lanes * p.cpt == v;
    return p;
}
std::size_t at_most(std::size_t n, std::size_t limit) { return n < limit ? n : limit; }
std::size_t over(std::size_t n, std::size_t d) { return (n + d - 1) / d; }

// As many groups as threads and two stages each allow, fewer when there are few rows: then every SM gets some.
RingPlan plan_forward_ring(std::size_t rows, std::size_t hidden, std::size_t elem, bool fused) {
    RingPlan p = plan_row(hidden, elem, 8);
    auto& a = p.args;
    a.step_rows = ring_kernels::rows_at_once(p.cpt) * (32 / a.lanes);
    a.data_offset = static_cast<unsigned>(vectors_end(hidden, 2));
    const std::size_t stage = a.step_rows * hidden * elem * (fused ? 2 : 1), room = kSmemPerSm - a.data_offset;
    std::size_t groups = ring_kernels::kForwardThreads / 32 / a.warps_per_row;
    groups = at_most(at_most(groups, room / (2 * stage)), over(rows, static_cast<std::size_t>(kNumSMs) * a.step_rows));
    a.groups = static_cast<int>(groups);
    a.stages = static_cast<int>(at_most(room / groups / stage, ring_kernels::kMaxStages));
    p.threads = a.groups * a.warps_per_row * 32;
    p.smem = a.data_offset + groups * a.stages * stage;
    p.grid = static_cast<unsigned>(at_most(over(rows, groups * a.step_rows), kNumSMs));
    return p;
}

// Threads of a CTA of the backward; kBackwardThreads in all on an SM.
int backward_ring_threads(std::size_t vectors) { return vectors <= 256 ? 256 : ring_kernels::kBackwardThreads; }
int backward_loose_threads(std::size_t hidden) { return hidden <= 2048 ? 256 : loose_kernels::kBackwardThreads; }

// Threads cover as many rows at a time as they have vectors for, fewer when there are few rows.
RingPlan plan_backward_ring(std::size_t rows, std::size_t hidden, std::size_t elem) {
    RingPlan p = plan_row(hidden, elem, 4);
    auto& a = p.args;
    const std::size_t v = a.vectors;
    p.threads = backward_ring_threads(v);
    p.cols = v <= 512 ? 1 : v <= 1024 ? 2 : 4;
    const std::size_t ctas = ring_kernels::kBackwardThreads / p.threads, rows_each = ring_kernels::kTileVectors / p.cols;
    std::size_t groups = p.cols == 1 ? p.threads / v : 1;
    groups = at_most(at_most(groups, ring_kernels::kMaxTileRows / rows_each), over(rows, kNumSMs * ctas * rows_each));
    a.groups = static_cast<int>(groups);
    a.step_rows = static_cast<int>(groups * rows_each);
    a.data_offset = static_cast<unsigned>(vectors_end(hidden, 1));
    const std::size_t stage = 2 * a.step_rows * hidden * elem, fixed = ring_kernels::kStatsBytes + 1024;   // 1024: kept by the hardware
    a.stages = static_cast<int>(at_most((kSmemPerSm + 1024) / ctas - fixed - a.data_offset, ring_kernels::kMaxStages * stage) / stage);
    p.smem = a.data_offset + a.stages * stage;
    p.grid = static_cast<unsigned>(at_most(over(rows, a.step_rows), kNumSMs * ctas));
    return p;
}

struct LoosePlan {
    loose_kernels::LooseArgs args;
    int columns, threads;      // columns per thread (backward)
    unsigned grid;
    std::size_t smem;
};
std::size_t loose_vectors_end(std::size_t hidden, std::size_t vectors) {
    return loose_kernels::kVectorsOffset + (vectors * hidden * sizeof(float) + 127) / 128 * 128;
}
unsigned loose_tensor_bytes(std::size_t rows, std::size_t hidden, std::size_t elem) {
    return static_cast<unsigned>((rows * hidden * elem + loose_kernels::kSlack + 127) / 128 * 128);
}

LoosePlan plan_forward_loose(std::size_t rows, std::size_t hidden, std::size_t elem, bool fused) {
    LoosePlan p{};
    auto& a = p.args;
    a.warps_per_row = hidden <= 2048 ? 1 : hidden <= 4096 ? 2 : 4;
    a.step_rows = static_cast<int>(hidden >= 1024 ? 1 : over(1024, hidden) < 32 ? over(1024, hidden) : 32);
    a.data_offset = static_cast<unsigned>(loose_vectors_end(hidden, 2));
    a.tensor_bytes = loose_tensor_bytes(a.step_rows, hidden, elem);
    const std::size_t stage = (fused ? 2 : 1) * static_cast<std::size_t>(a.tensor_bytes), room = kSmemPerSm - a.data_offset;
    std::size_t groups = loose_kernels::kForwardThreads / 32 / a.warps_per_row;
    groups = at_most(at_most(groups, room / (2 * stage)), over(rows, static_cast<std::size_t>(kNumSMs) * a.step_rows));
    if (a.warps_per_row > 1) groups = at_most(groups, 15);     // a named barrier each
    a.groups = static_cast<int>(groups);
    a.stages = static_cast<int>(at_most(room / groups / stage, ring_kernels::kMaxStages));
    p.threads = a.groups * a.warps_per_row * 32;
    p.smem = a.data_offset + groups * a.stages * stage;
    p.grid = static_cast<unsigned>(at_most(over(rows, groups * a.step_rows), kNumSMs));
    return p;
}

LoosePlan plan_backward_loose(std::size_t rows, std::size_t hidden, std::size_t elem) {
    LoosePlan p{};
    auto& a = p.args;
    p.threads = backward_loose_threads(hidden);
    p.columns = 1;
    while (static_cast<std::size_t>(p.columns) * p.threads < hidden) p.columns *= 2;
    const std::size_t ctas = loose_kernels::kBackwardThreads / p.threads;
    a.groups = p.columns == 1 ? static_cast<int>(at_most(p.threads / hidden, loose_kernels::kMaxTileRows / 4)) : 1;
    // Tiles of about 16 KB per tensor and CTA (more for one CTA), fewer rows when there are few: then every SM gets some.
    std::size_t tile = at_most(16 * 1024 * (2 / ctas) / (hidden * elem), loose_kernels::kMaxTileRows);
    tile = at_most(tile, over(rows, kNumSMs * ctas));
    a.step_rows = static_cast<int>(tile < 1 ? 1 : tile);
    const int warps = p.threads / 32;                          // 16 at most: 8 units of several warps, 64 floats of sums each
    a.warps_per_row = 1;
    while (a.warps_per_row * a.step_rows * 2 <= warps && static_cast<std::size_t>(a.warps_per_row) * 64 < hidden) a.warps_per_row *= 2;
    a.data_offset = static_cast<unsigned>(loose_vectors_end(hidden, 1));
    const std::size_t room = (kSmemPerSm + 1024) / ctas - 1024 - loose_kernels::kStatsBytes - a.data_offset;
    std::size_t stage = 0;
    for (;; --a.step_rows) {                                   // two stages at least, of one row if need be (form_of)
        a.tensor_bytes = loose_tensor_bytes(a.step_rows, hidden, elem);
        stage = 3 * static_cast<std::size_t>(a.tensor_bytes);     // room for a residual, whether there is one or not
        if (a.step_rows == 1 || 2 * stage <= room) break;
    }
    a.stages = static_cast<int>(at_most(room / stage, ring_kernels::kMaxStages));
    p.smem = a.data_offset + a.stages * stage;
    const std::size_t joined = a.data_offset + 2 * hidden * sizeof(float);
    if (p.smem < joined) p.smem = joined;
    p.grid = static_cast<unsigned>(at_most(over(rows, a.step_rows), kNumSMs * ctas));
    return p;
}

constexpr std::size_t kMaxSplits = 64;
std::size_t any_splits(std::size_t rows) {
    const std::size_t n = (rows + 63) / 64;
    return n < kMaxSplits ? n : kMaxSplits;
}

unsigned any_grid(std::size_t rows) { return static_cast<unsigned>(rows < kNumSMs * 8ull ? rows : kNumSMs * 8ull); }

bool valid_rows(std::size_t rows, std::size_t hidden) {
    return rows != 0 && hidden != 0 && hidden <= 0x7fffffffull && rows <= (1ull << 46) / hidden;
}

template <typename Kernel>
int allow_smem(Kernel kernel, PerDeviceOnce* once, std::size_t fixed = 0) {
    if (once->needed()) {
        CGPT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemPerSm - fixed)));
        once->done();
    }
    return CGPT_OK;
}

// Enough for the call's layout whatever its type and alignment turn out to be, and for every call with fewer rows: a CTA has a row
// at least, and no more CTAs are launched than the SMs hold. (A plan's own grid falls where a CTA starts to take more rows.)
std::size_t workspace_bytes(std::size_t rows, std::size_t hidden) {
    std::size_t parts = 0, stats = 0;
    for (std::size_t elem : {2, 4})
        for (bool vector : {false, true}) {
            const Form form = form_of(hidden, elem, vector);
            const std::size_t ring_ctas = ring_kernels::kBackwardThreads / backward_ring_threads(hidden * elem / 16);
            const std::size_t loose_ctas = loose_kernels::kBackwardThreads / backward_loose_threads(hidden);
            const std::size_t n = form == Form::kRing ? at_most(rows, kNumSMs * ring_ctas)
                                  : form == Form::kLoose ? at_most(rows, kNumSMs * loose_ctas) : any_splits(rows);
            if (n > parts) parts = n;
            if (form == Form::kAny) stats = rows * sizeof(float2);
        }
    return parts * 2 * hidden * sizeof(float) + stats;
}

template <int N> using Int = std::integral_constant<int, N>;

template <typename T, bool FUSED>
int launch_forward(void* y, void* sum, const void* x, const void* residual, const void* w, const void* b, std::size_t rows,
                   std::size_t hidden, float epsilon, const DropoutArgs& args, cudaStream_t s) {
    const bool al = aligned16(y) && aligned16(sum) && aligned16(x) && aligned16(residual) && aligned16(w) && aligned16(b);
    const Form form = form_of(hidden, sizeof(T), al);
    if (form == Form::kRing) {
        const RingPlan p = plan_forward_ring(rows, hidden, sizeof(T), FUSED);
        auto launch = [&](auto cpt, auto full) {
            auto kernel = ring_kernels::layernorm_forward_ring_kernel<T, cpt.value, full.value, FUSED>;
            static PerDeviceOnce once;
            CGPT_TRY(allow_smem(kernel, &once));
            auto args_on_device = p.args;
            args_on_device.status = tc_status_device_ptr();
            if (args_on_device.status == nullptr) return CGPT_ERR_STATE;
            kernel<<<p.grid, p.threads, p.smem, s>>>(
                static_cast<T*>(y), static_cast<T*>(sum), static_cast<const T*>(x), static_cast<const T*>(residual),
                static_cast<const T*>(w), static_cast<const T*>(b), static_cast<long long>(rows), static_cast<int>(hidden), epsilon,
                args_on_device, args);
            count_launch();
            CGPT_LAUNCH_CHECK();
            return CGPT_OK;
        };
        auto either = [&](auto cpt) { return p.full ? launch(cpt, std::true_type{}) : launch(cpt, std::false_type{}); };
        return p.cpt == 1 ? either(Int<1>{}) : p.cpt == 2 ? either(Int<2>{}) : p.cpt == 4 ? either(Int<4>{}) : either(Int<8>{});
    }
    if (form == Form::kLoose) {
        LoosePlan p = plan_forward_loose(rows, hidden, sizeof(T), FUSED);
        auto kernel = loose_kernels::layernorm_forward_loose_kernel<T, FUSED>;
        static PerDeviceOnce once;
        CGPT_TRY(allow_smem(kernel, &once));
        p.args.status = tc_status_device_ptr();
        if (p.args.status == nullptr) return CGPT_ERR_STATE;
        kernel<<<p.grid, p.threads, p.smem, s>>>(
            static_cast<T*>(y), static_cast<T*>(sum), static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(w),
            static_cast<const T*>(b), static_cast<long long>(rows), static_cast<int>(hidden), epsilon, p.args, args);
        count_launch();
        CGPT_LAUNCH_CHECK();
        return CGPT_OK;
    }
    layernorm_forward_any_kernel<T, FUSED><<<any_grid(rows), kThreads, 0, s>>>(
        static_cast<T*>(y), static_cast<T*>(sum), static_cast<const T*>(x), static_cast<const T*>(residual),
        static_cast<const T*>(w), static_cast<const T*>(b), static_cast<long long>(rows), static_cast<long long>(hidden), epsilon, args);
    count_launch();
    CGPT_LAUNCH_CHECK();
    return CGPT_OK;
}

template <typename T, bool FUSED>
int launch_backward(void* dx, void* din, void* dw, void* db, const void* dy, const void* x, const void* w, const void* residual,
                    void* workspace, std::size_t rows, std::size_t hidden, float epsilon, const DropoutArgs& args, cudaStream_t s) {
    float* partial = static_cast<float*>(workspace);
    const unsigned columns = static_cast<unsigned>((hidden + 31) / 32);
    auto reduce = [&](std::size_t parts) {
        CGPT_CUDA_TRY(launch_after_previous(layernorm_reduce_kernel<T>, dim3(columns, db != nullptr ? 2 : 1), 1024, 0, s, static_cast<T*>(dw),
                                            static_cast<T*>(db), partial, static_cast<int>(parts), static_cast<long long>(hidden)));
        count_launch();
        return CGPT_OK;
    };
    const bool al = aligned16(dx) && aligned16(din) && aligned16(dy) && aligned16(x) && aligned16(w) && aligned16(residual);
    const Form form = form_of(hidden, sizeof(T), al);
    if (form == Form::kRing) {
        const RingPlan p = plan_backward_ring(rows, hidden, sizeof(T));
        auto launch = [&](auto cpt, auto cols, auto full) {
            auto kernel = ring_kernels::layernorm_backward_ring_kernel<T, cpt.value, cols.value, full.value, FUSED>;
            static PerDeviceOnce once;
            CGPT_TRY(allow_smem(kernel, &once, ring_kernels::kStatsBytes));
            auto args_on_device = p.args;
            args_on_device.status = tc_status_device_ptr();
            if (args_on_device.status == nullptr) return CGPT_ERR_STATE;
            kernel<<<p.grid, p.threads, p.smem, s>>>(
                static_cast<T*>(dx), static_cast<T*>(din), partial, static_cast<const T*>(dy), static_cast<const T*>(x),
                static_cast<const T*>(w), static_cast<const T*>(residual), static_cast<long long>(rows), static_cast<int>(hidden),
                epsilon, args_on_device, args);
            count_launch();
            CGPT_LAUNCH_CHECK();
            return reduce(p.grid);
        };
        auto either = [&](auto cpt, auto cols) { return p.full ? launch(cpt, cols, std::true_type{}) : launch(cpt, cols, std::false_type{}); };
        if (p.cols == 1) return p.cpt == 1 ? either(Int<1>{}, Int<1>{}) : p.cpt == 2 ? either(Int<2>{}, Int<1>{}) : either(Int<4>{}, Int<1>{});
        if (p.cols == 2) return either(Int<4>{}, Int<2>{});
        // 16-bit rows that fill the lanes of four vectors a thread are longer than rings take
        if constexpr (sizeof(T) == 2) return launch(Int<4>{}, Int<4>{}, std::false_type{});
        else return either(Int<4>{}, Int<4>{});
    }
    if (form == Form::kLoose) {
        const LoosePlan p = plan_backward_loose(rows, hidden, sizeof(T));
        auto launch = [&](auto columns, auto threads) {
            auto kernel = loose_kernels::layernorm_backward_loose_kernel<T, columns.value, threads.value, FUSED>;
            static PerDeviceOnce once;
            CGPT_TRY(allow_smem(kernel, &once, loose_kernels::kStatsBytes));
            auto args_on_device = p.args;
            args_on_device.status = tc_status_device_ptr();
            if (args_on_device.status == nullptr) return CGPT_ERR_STATE;
            kernel<<<p.grid, p.threads, p.smem, s>>>(
                static_cast<T*>(dx), static_cast<T*>(din), partial, static_cast<const T*>(dy), static_cast<const T*>(x),
                static_cast<const T*>(w), static_cast<const T*>(residual), static_cast<long long>(rows), static_cast<int>(hidden),
                epsilon, args_on_device, args);
            count_launch();
            CGPT_LAUNCH_CHECK();
            return reduce(p.grid);
        };
        if (p.threads == 256) {
            switch (p.columns) {
                case 1: return launch(Int<1>{}, Int<256>{});
                case 2: return launch(Int<2>{}, Int<256>{});
                case 4: return launch(Int<4>{}, Int<256>{});
                default: return launch(Int<8>{}, Int<256>{});
            }
        }
        return p.columns == 8 ? launch(Int<8>{}, Int<512>{}) : launch(Int<16>{}, Int<512>{});
    }
    const std::size_t splits = any_splits(rows);
    float2* stats = reinterpret_cast<float2*>(partial + splits * 2 * hidden);
    layernorm_backward_any_kernel<T, FUSED><<<any_grid(rows), kThreads, 0, s>>>(
        static_cast<T*>(dx), static_cast<T*>(din), stats, static_cast<const T*>(dy), static_cast<const T*>(x),
        static_cast<const T*>(w), static_cast<const T*>(residual), static_cast<long long>(rows), static_cast<long long>(hidden),
        epsilon, args);
    count_launch();
    CGPT_LAUNCH_CHECK();
    layernorm_columns_any_kernel<T><<<dim3(columns, static_cast<unsigned>(splits)), kThreads, 0, s>>>(
        partial, static_cast<const T*>(dy), static_cast<const T*>(x), stats, static_cast<long long>(rows), static_cast<long long>(hidden));
    count_launch();
    CGPT_LAUNCH_CHECK();
    return reduce(splits);
}

}  // namespace
}  // namespace cgpt

using namespace cgpt;

extern "C" int cgpt_layernorm_forward(void* y, const void* x, const void* w, const void* b, size_t rows, size_t hidden,
                                      float epsilon, int dtype, cgpt_stream_t stream) {
    if (!y || !x || !w) return CGPT_ERR_NULL;
    if (!valid_float_dtype(dtype)) return CGPT_ERR_DTYPE;
    if (!valid_rows(rows, hidden)) return CGPT_ERR_SHAPE;
    if (!(epsilon > 0.f) || y == x) return CGPT_ERR_OPTION;
    if (!element_aligned(dtype, {y, x, w, b})) return CGPT_ERR_ALIGN;
    auto s = static_cast<cudaStream_t>(stream);
    CGPT_DISPATCH_DTYPE(dtype, T, { return (launch_forward<T, false>(y, nullptr, x, nullptr, w, b, rows, hidden, epsilon, DropoutArgs{}, s)); });
    return CGPT_OK;
}

extern "C" size_t cgpt_layernorm_backward_workspace_bytes(size_t rows, size_t hidden) {
    return valid_rows(rows, hidden) ? workspace_bytes(rows, hidden) : 0;
}

extern "C" int cgpt_layernorm_backward(void* dx, void* dw, void* db, const void* dy, const void* x, const void* w,
                                       const void* residual, void* workspace, size_t workspace_size, size_t rows, size_t hidden,
                                       float epsilon, int dtype, cgpt_stream_t stream) {
    if (!dx || !dw || !dy || !x || !w || !workspace) return CGPT_ERR_NULL;
    if (!valid_float_dtype(dtype)) return CGPT_ERR_DTYPE;
    if (!valid_rows(rows, hidden) || workspace_size < workspace_bytes(rows, hidden)) return CGPT_ERR_SHAPE;
    if (!(epsilon > 0.f) || dx == dy || dx == x) return CGPT_ERR_OPTION;
    if (!element_aligned(dtype, {dx, dw, db, dy, x, w, residual}) || !aligned16(workspace)) return CGPT_ERR_ALIGN;
    auto s = static_cast<cudaStream_t>(stream);
    CGPT_DISPATCH_DTYPE(dtype, T, {
        return (launch_backward<T, false>(dx, nullptr, dw, db, dy, x, w, residual, workspace, rows, hidden, epsilon, DropoutArgs{}, s));
    });
    return CGPT_OK;
}

extern "C" int cgpt_dropout_add_layernorm_forward(void* y, void* sum, const void* x, const void* residual, const void* w,
                                                  const void* b, size_t rows, size_t hidden, float epsilon, float probability,
                                                  const uint64_t* state, uint32_t site, int dtype, cgpt_stream_t stream) {
    if (!y || !sum || !x || !residual || !w) return CGPT_ERR_NULL;
    if (!valid_float_dtype(dtype)) return CGPT_ERR_DTYPE;
    if (!valid_rows(rows, hidden)) return CGPT_ERR_SHAPE;
    if (!(epsilon > 0.f) || y == x || y == residual || y == sum) return CGPT_ERR_OPTION;
    if (!element_aligned(dtype, {y, sum, x, residual, w, b})) return CGPT_ERR_ALIGN;
    DropoutArgs args;
    CGPT_TRY(dropout_args(&args, probability, state, site, rows * hidden));
    auto s = static_cast<cudaStream_t>(stream);
    CGPT_DISPATCH_DTYPE(dtype, T, { return (launch_forward<T, true>(y, sum, x, residual, w, b, rows, hidden, epsilon, args, s)); });
    return CGPT_OK;
}

extern "C" int cgpt_dropout_add_layernorm_backward(void* dx, void* dresidual, void* dw, void* db, const void* dy,
                                                   const void* dsum, const void* sum, const void* w, void* workspace,
                                                   size_t workspace_size, size_t rows, size_t hidden, float epsilon,
                                                   float probability, const uint64_t* state, uint32_t site, int dtype,
                                                   cgpt_stream_t stream) {
    if (!dx || !dresidual || !dw || !dy || !sum || !w || !workspace) return CGPT_ERR_NULL;
    if (!valid_float_dtype(dtype)) return CGPT_ERR_DTYPE;
    if (!valid_rows(rows, hidden) || workspace_size < workspace_bytes(rows, hidden)) return CGPT_ERR_SHAPE;
    if (!(epsilon > 0.f) || dx == dresidual || dx == dy || dx == sum || dx == dsum || dresidual == dy || dresidual == sum) return CGPT_ERR_OPTION;
    if (!element_aligned(dtype, {dx, dresidual, dw, db, dy, dsum, sum, w}) || !aligned16(workspace)) return CGPT_ERR_ALIGN;
    DropoutArgs args;
    CGPT_TRY(dropout_args(&args, probability, state, site, rows * hidden));
    auto s = static_cast<cudaStream_t>(stream);
    CGPT_DISPATCH_DTYPE(dtype, T, {
        return (launch_backward<T, true>(dresidual, dx, dw, db, dy, sum, w, dsum, workspace, rows, hidden, epsilon, args, s));
    });
    return CGPT_OK;
}
