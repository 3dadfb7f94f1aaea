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

// Eight consecutive elements per thread and trip: one generator block. VECTOR: 16-byte accesses (aligned bases).
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(T* out, const T* in, const T* residual, long long count, const DropoutArgs args) {
    const Philox gen(args);
    const long long stride = static_cast<long long>(gridDim.x) * kThreads * 8;
    for (long long i = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) * 8; i < count; i += stride) {
        float v[8];
        const bool whole = VECTOR && i + 8 <= count;
        if (whole) {
            constexpr int V = 16 / sizeof(T);
#pragma unroll
            for (int c = 0; c < 8; c += V) load_vec_stream<T, V>(*reinterpret_cast<float(*)[V]>(&v[c]), in + i + c);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = i + k < count ? to_f32<T>(in[i + k]) : 0.f;
        }
        if (args.threshold != 0) apply_block(v, gen.block(static_cast<std::uint32_t>(i >> 3)), args.threshold, args.scale);
        if (whole) {
            constexpr int V = 16 / sizeof(T);
            if (residual != nullptr) {
                float r[8];
#pragma unroll
                for (int c = 0; c < 8; c += V) load_vec_stream<T, V>(*reinterpret_cast<float(*)[V]>(&r[c]), residual + i + c);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] += r[k];
            }
#pragma unroll
            for (int c = 0; c < 8; c += V) store_vec<T, V>(out + i + c, *reinterpret_cast<float(*)[V]>(&v[c]));
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k < count) out[i + k] = from_f32<T>(residual != nullptr ? v[k] + to_f32<T>(residual[i + k]) : v[k]);
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
        auto kernel = al ? dropout_kernel<T, true> : dropout_kernel<T, false>;
        const std::size_t need = (count + kThreads * 8 - 1) / (kThreads * 8);
        const std::size_t cap = static_cast<std::size_t>(kNumSMs) * resident_ctas_per_sm(reinterpret_cast<const void*>(kernel), kThreads, 0);
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
