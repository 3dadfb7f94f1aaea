// Dropout without a stored mask (decisions: philox.cuh), forward with an optional residual and backward, for sm_100a.
//
//   out = [residual +] (keep ? in * scale : 0)        backward: the same map of the gradient
//
// Memory-bound: 2 (3 with a residual or accumulation) * sizeof(T) bytes per element.
#include "philox.cuh"
#include "launch_counter.h"

namespace cgpt {
namespace {

constexpr int kThreads = 256;

// Aligned tensors: BLOCKS generator blocks of eight elements per thread and trip, all loads of a trip (the residual's too) on
// their way before the first block is worked out: four 16-byte loads a thread.
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads)
dropout_vector_kernel(T* out, const T* in, const T* residual, long long count, const DropoutArgs args) {
    constexpr int V = 16 / sizeof(T), N = 8 / V;              // 16-byte vectors per block
    constexpr int BLOCKS = 4 / (N * (RESIDUAL ? 2 : 1));
    const PhiloxOf<RESIDUAL ? Constants::kLeft : Constants::kHoisted> gen(args);   // round keys kept only where nothing else is on its way
    const long long whole = count >> 3;
    if (blockIdx.x == 0 && threadIdx.x < (count & 7)) {       // the last elements fill no block
        const long long e = whole * 8 + threadIdx.x;
        float v = to_f32<T>(in[e]);
        if (args.threshold != 0) v = apply_one(v, gen, e, args);
        out[e] = from_f32<T>(RESIDUAL ? v + to_f32<T>(residual[e]) : v);
    }
    const long long stride = static_cast<long long>(gridDim.x) * kThreads;
    uint4 x[BLOCKS][N], r[BLOCKS][N];
    auto load = [&](int k, long long block) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            x[k][c] = __ldcs(reinterpret_cast<const uint4*>(in) + block * N + c);
            if constexpr (RESIDUAL) r[k][c] = __ldcs(reinterpret_cast<const uint4*>(residual) + block * N + c);
        }
    };
    auto finish = [&](int k, long long block) {
        Pair v[4];
#pragma unroll
        for (int c = 0; c < N; ++c) to_pairs<T>(*reinterpret_cast<Pair(*)[V / 2]>(&v[c * V / 2]), x[k][c]);
        if (args.threshold != 0) drop_pairs<4>(v, gen, block * 8, args);
#pragma unroll
        for (int c = 0; c < N; ++c) {
            Pair(&part)[V / 2] = *reinterpret_cast<Pair(*)[V / 2]>(&v[c * V / 2]);
            if constexpr (RESIDUAL) {
                Pair res[V / 2];
                to_pairs<T>(res, r[k][c]);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) part[i] = add2(part[i], res[i]);
            }
            *reinterpret_cast<uint4*>(out + block * 8 + c * V) = to_raw<T>(part);
        }
    };
    for (long long block0 = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; block0 < whole; block0 += stride * BLOCKS) {
        if (block0 + (BLOCKS - 1) * stride < whole) {
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k) load(k, block0 + k * stride);
#pragma unroll
            for (int k = 0; k < BLOCKS; ++k) finish(k, block0 + k * stride);
        } else {
            for (long long block = block0; block < whole; block += stride) {
                load(0, block);
                finish(0, block);
            }
        }
    }
}

// Any alignment, element by element; a thread still has the eight elements of a block.
template <typename T>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(T* out, const T* in, const T* residual, long long count, const DropoutArgs args) {
    const Philox gen(args);
    const long long stride = static_cast<long long>(gridDim.x) * kThreads * 8;
    for (long long i = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) * 8; i < count; i += stride) {
        Pair p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            p[k] = pair(i + 2 * k < count ? to_f32<T>(in[i + 2 * k]) : 0.f, i + 2 * k + 1 < count ? to_f32<T>(in[i + 2 * k + 1]) : 0.f);
        if (args.threshold != 0) drop_pairs<4>(p, gen, i, args);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 f = both(p[k >> 1]);
            const float v = (k & 1) != 0 ? f.y : f.x;
            if (i + k < count) out[i + k] = from_f32<T>(residual != nullptr ? v + to_f32<T>(residual[i + k]) : v);
        }
    }
}

__global__ void advance_kernel(unsigned long long* state, unsigned long long steps) { state[1] += steps; }

int run(void* out, const void* in, const void* residual, std::size_t count, float probability, const void* state,
        std::uint32_t site, int dtype, cgpt_stream_t stream) {
    if (!out || !in) return CGPT_ERR_NULL;
    if (!valid_float_dtype(dtype)) return CGPT_ERR_DTYPE;
    if (count == 0 || count > (1ull << 46)) return CGPT_ERR_SHAPE;
    if (!element_aligned(dtype, {out, in, residual})) return CGPT_ERR_ALIGN;
    DropoutArgs args;
    CGPT_TRY(dropout_args(&args, probability, state, site, count));
    auto s = static_cast<cudaStream_t>(stream);
    const bool al = aligned16(out) && aligned16(in) && aligned16(residual);
    CGPT_DISPATCH_DTYPE(dtype, T, {
        auto kernel = !al ? dropout_kernel<T> : residual != nullptr ? dropout_vector_kernel<T, true> : dropout_vector_kernel<T, false>;
        const std::size_t per_thread = !al ? 8 : residual != nullptr ? 32 / sizeof(T) : 64 / sizeof(T);   // elements per trip
        const std::size_t need = (count + kThreads * per_thread - 1) / (kThreads * per_thread);
        constexpr std::size_t cap = std::size_t{1} << 30;
        kernel<<<static_cast<unsigned>(need < cap ? need : cap), kThreads, 0, s>>>(
            static_cast<T*>(out), static_cast<const T*>(in), static_cast<const T*>(residual), static_cast<long long>(count), args);
        count_launch();
        CGPT_LAUNCH_CHECK();
    });
    return CGPT_OK;
}

}  // namespace
}  // namespace cgpt

using namespace cgpt;

extern "C" int cgpt_dropout_forward(void* out, const void* in, const void* residual, size_t count, float probability,
                                    const uint64_t* state, uint32_t site, int dtype, cgpt_stream_t stream) {
    return run(out, in, residual, count, probability, state, site, dtype, stream);
}

extern "C" int cgpt_dropout_backward(void* din, const void* dout, size_t count, float probability, const uint64_t* state,
                                     uint32_t site, int accumulate, int dtype, cgpt_stream_t stream) {
    if (accumulate && din != nullptr && din == dout) return CGPT_ERR_OPTION;
    return run(din, dout, accumulate ? din : nullptr, count, probability, state, site, dtype, stream);
}

extern "C" int cgpt_dropout_advance(uint64_t* state, uint64_t steps, cgpt_stream_t stream) {
    if (!state) return CGPT_ERR_NULL;
    if ((reinterpret_cast<std::uintptr_t>(state) & 7u) != 0) return CGPT_ERR_ALIGN;
    advance_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(reinterpret_cast<unsigned long long*>(state), steps);
    count_launch();
    CGPT_LAUNCH_CHECK();
    return CGPT_OK;
}
