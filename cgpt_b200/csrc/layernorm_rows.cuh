// Layer norm of rows that no 16-byte vector fits (odd lengths, unaligned tensors) but that registers hold. Included by
// layernorm.cu only.
//
// A row is owned by a group of `tpr` threads (whole warps); a thread owns the same CPT columns (tpr apart, so that the lanes of a
// load are consecutive) of every row its group visits, and keeps their dw and db in registers. R rows are taken at a time: their
// loads are in flight together and their sums share one reduction.
#pragma once

namespace rows_kernels {

constexpr int kMaxTpr = 512;

// A row group inside its CTA: `warps` warps that meet at a barrier of their own (one warp needs none).
struct Group {
    int index, warps, warp, lane;   // warp: within the group
    __device__ __forceinline__ void sync() const {
        asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(warps * 32) : "memory");
    }
};

// Totals of NV values over the group, in every thread. `red`: the group's [NV][16] floats of this call; two calls in a row use
// different areas, so that the barrier of one call also says that the area of the call before it has been read.
template <int NV>
__device__ __forceinline__ void group_sum(float (&v)[NV], const Group& g, float* red) {
    using W = WarpSums<NV>;
    W::reduce(v, g.lane);
    if (g.warps > 1) {
        if ((g.lane & 7) == 0) {
            const int first = W::first_of(g.lane);
#pragma unroll
            for (int i = 0; i < W::kCount; ++i) red[(first + i) * 16 + g.warp] = v[i];
        }
        g.sync();
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = g.lane < g.warps ? red[i * 16 + g.lane] : 0.f;
        W::reduce(v, g.lane);
    }
    W::broadcast(v);
}

// R rows of a tensor; zeros past the rows and columns.
template <typename T, int CPT, int R>
__device__ __forceinline__ void load_rows(float (&v)[R][CPT], const T* from, long long row0, long long rows, int hidden, int tpr, int tid) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = c * tpr + tid;
            v[r][c] = from != nullptr && row0 + r < rows && col < hidden ? to_f32<T>(from[(row0 + r) * hidden + col]) : 0.f;
        }
}

// The dropout map of a thread's R x CPT elements. Every lane of the warp must call this, whatever columns and rows it has.
template <int CPT, int R>
__device__ __forceinline__ void drop_rows(float (&v)[R][CPT], long long row0, int hidden, int tpr, int tid, const Philox& gen, const DropoutArgs& args) {
    if (args.threshold == 0) return;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j0 = 0; j0 < R * CPT; j0 += 4) {
        long long start[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) start[j] = (row0 + (j0 + j) / CPT) * hidden + (j0 + j) % CPT * tpr + tid - lane;
        const std::uint32_t kept = keep_four_runs(start, gen, args.threshold);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float& x = v[(j0 + j) / CPT][(j0 + j) % CPT];
            x = (kept >> j) & 1u ? __fmul_rn(x, args.scale) : 0.f;
        }
    }
}

template <typename T, int CPT, int R, bool FUSED>
__global__ void __launch_bounds__(kMaxTpr)
layernorm_forward_rows_kernel(T* __restrict__ y, T* sum, const T* x, const T* residual, const T* __restrict__ w,
                              const T* __restrict__ b, long long rows, int hidden, float epsilon, int tpr, const DropoutArgs args) {
    __shared__ float red_all[2][16][R * 16];
    const int index = threadIdx.x / tpr, tid = threadIdx.x - index * tpr;
    const Group g{index, tpr >> 5, tid >> 5, static_cast<int>(threadIdx.x & 31)};
    const Philox gen(args);
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    const int groups = blockDim.x / tpr;
    const long long step = static_cast<long long>(gridDim.x) * groups * R;
    for (long long row0 = (static_cast<long long>(blockIdx.x) * groups + index) * R; row0 < rows; row0 += step) {
        float v[R][CPT], mean[R], var[R];
        load_rows<T, CPT, R>(v, x, row0, rows, hidden, tpr, tid);
        if constexpr (FUSED) {
            float res[R][CPT];
            load_rows<T, CPT, R>(res, residual, row0, rows, hidden, tpr, tid);
            drop_rows<CPT, R>(v, row0, hidden, tpr, tid, gen, args);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < CPT; ++c) {
                    const int col = c * tpr + tid;
                    const T stored = from_f32<T>(v[r][c] + res[r][c]);
                    v[r][c] = to_f32<T>(stored);             // the norm is of the stored value
                    if (row0 + r < rows && col < hidden) sum[(row0 + r) * hidden + col] = stored;
                    else v[r][c] = 0.f;
                }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] = 0.f;
#pragma unroll
            for (int c = 0; c < CPT; ++c) mean[r] += v[r][c];
        }
        group_sum<R>(mean, g, red_all[0][index]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] *= inv_hidden;
            var[r] = 0.f;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const float d = c * tpr + tid < hidden ? v[r][c] - mean[r] : 0.f;
                var[r] = fmaf(d, d, var[r]);
            }
        }
        group_sum<R>(var, g, red_all[1][index]);
#pragma unroll
        for (int r = 0; r < R; ++r) var[r] = rsqrtf(fmaf(var[r], inv_hidden, epsilon));
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = c * tpr + tid;
            if (col < hidden) {
                const float wv = to_f32<T>(w[col]), bv = b != nullptr ? to_f32<T>(b[col]) : 0.f;
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (row0 + r < rows) y[(row0 + r) * hidden + col] = from_f32<T>(fmaf(normalised(v[r][c], mean[r], var[r]), wv, bv));
            }
        }
    }
}

// partial: [gridDim.x][2][hidden]
template <typename T, int CPT, int R, bool FUSED>
__global__ void __launch_bounds__(kMaxTpr)
layernorm_backward_rows_kernel(T* dx, T* din, float* __restrict__ partial, const T* __restrict__ dy, const T* __restrict__ x,
                               const T* __restrict__ w, const T* residual, long long rows, int hidden, float epsilon, int tpr,
                               const DropoutArgs args) {
    extern __shared__ float shared[];                          // the groups' sums, then (reused) their dw and db
    const int index = threadIdx.x / tpr, tid = threadIdx.x - index * tpr;
    const Group g{index, tpr >> 5, tid >> 5, static_cast<int>(threadIdx.x & 31)};
    float* red = shared + index * (4 * R * 16);
    const Philox gen(args);
    launch_dependents();
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    const int groups = blockDim.x / tpr;
    float aw[CPT] = {}, ab[CPT] = {};
    const long long step = static_cast<long long>(gridDim.x) * groups * R;
    for (long long row0 = (static_cast<long long>(blockIdx.x) * groups + index) * R; row0 < rows; row0 += step) {
        float v[R][CPT], gy[R][CPT], out[R][CPT], mean[R], sums[3 * R];
        load_rows<T, CPT, R>(v, x, row0, rows, hidden, tpr, tid);
        load_rows<T, CPT, R>(gy, dy, row0, rows, hidden, tpr, tid);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] = 0.f;
#pragma unroll
            for (int c = 0; c < CPT; ++c) mean[r] += v[r][c];
        }
        load_rows<T, CPT, R>(out, residual, row0, rows, hidden, tpr, tid);   // needed last: on its way while the sums are reduced
        group_sum<R>(mean, g, red);
#pragma unroll
        for (int i = 0; i < 3 * R; ++i) sums[i] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) mean[r] *= inv_hidden;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = c * tpr + tid;
            const float wv = col < hidden ? to_f32<T>(w[col]) : 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float s[3] = {sums[r], sums[R + r], sums[2 * R + r]};
                norm_sums(s, gy[r][c], wv, col < hidden ? v[r][c] - mean[r] : 0.f);
                sums[r] = s[0];
                sums[R + r] = s[1];
                sums[2 * R + r] = s[2];
            }
        }
        group_sum<3 * R>(sums, g, red + R * 16);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sums[r] = rsqrtf(fmaf(sums[r], inv_hidden, epsilon));                // rstd
            sums[R + r] *= inv_hidden;                                           // c1
            sums[2 * R + r] = sums[2 * R + r] * inv_hidden * sums[r];            // c2
        }
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = c * tpr + tid;
            const float wv = col < hidden ? to_f32<T>(w[col]) : 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float xh = normalised(v[r][c], mean[r], sums[r]);
                out[r][c] = norm_dx(gy[r][c], wv, xh, sums[r], sums[R + r], sums[2 * R + r], out[r][c]);
                aw[c] = fmaf(gy[r][c], xh, aw[c]);             // rows past the end: dy = 0
                ab[c] += gy[r][c];
                if (row0 + r < rows && col < hidden) dx[(row0 + r) * hidden + col] = from_f32<T>(out[r][c]);
            }
        }
        if constexpr (FUSED) {
            drop_rows<CPT, R>(out, row0, hidden, tpr, tid, gen, args);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < CPT; ++c)
                    if (row0 + r < rows && c * tpr + tid < hidden) din[(row0 + r) * hidden + c * tpr + tid] = from_f32<T>(out[r][c]);
        }
    }
    // The groups of a CTA add up their columns one after the other: one partial row of dw and of db per CTA.
    float* out_w = partial + static_cast<long long>(blockIdx.x) * 2 * hidden;
    for (int k = 0; k < groups; ++k) {
        __syncthreads();
        if (index == k) {
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                float* s = shared + c * tpr * 2 + tid;
                const float tw = (k == 0 ? 0.f : s[0]) + aw[c], tb = (k == 0 ? 0.f : s[tpr]) + ab[c];
                if (k + 1 < groups) {
                    s[0] = tw;
                    s[tpr] = tb;
                } else if (c * tpr + tid < hidden) {
                    out_w[c * tpr + tid] = tw;
                    out_w[hidden + c * tpr + tid] = tb;
                }
            }
        }
    }
}

}  // namespace rows_kernels
