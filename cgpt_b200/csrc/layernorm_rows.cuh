// Layer norm of rows that fit in registers. Included by layernorm.cu only.
//
// A row is owned by a group of `tpr` threads (whole warps), and a thread owns the same CPT vectors of VEC columns of every row
// its group visits. Its share of dw and db is therefore 2 * CPT * VEC registers for the whole launch, whatever the number of
// rows, and x, dy and the residual are read from memory once. R rows are taken at a time: their loads are in flight together,
// and their sums share one reduction, so the shuffles and the barrier of a reduction are paid once per R rows.
#pragma once

namespace rows_kernels {

constexpr int kMaxTpr = 512;

// Bytes of one vector as a register type.
template <typename T, int VEC> using RawOf = typename RawVec<sizeof(T) * VEC>::type;

template <typename T, int VEC>
__device__ __forceinline__ void unpack_raw(float (&out)[VEC], const RawOf<T, VEC>& raw) {
    Pack<T, VEC> pk;
    *reinterpret_cast<RawOf<T, VEC>*>(&pk) = raw;
    unpack_pack(out, pk);
}
template <typename T, int VEC>
__device__ __forceinline__ RawOf<T, VEC> pack_raw(const float (&in)[VEC]) {
    Pack<T, VEC> pk;
    convert_pack(pk, in);
    return *reinterpret_cast<const RawOf<T, VEC>*>(&pk);
}

// Makes packed 16-bit values opaque to the optimiser, so that it unpacks them again at their next use instead of keeping twice as
// many fp32 registers alive from one use to the next.
template <typename Raw>
__device__ __forceinline__ void keep_packed(Raw& v) {
    if constexpr (std::is_same<Raw, uint4>::value) asm volatile("" : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w));
}
template <typename Raw, int R, int CPT>
__device__ __forceinline__ void keep_packed_all(Raw (&v)[R][CPT]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < CPT; ++c) keep_packed(v[r][c]);
}

// Sums NV values over a warp. Halves the set of values a lane is responsible for while lanes still differ in what they hold, so
// NV = 4 takes 6 shuffles and NV = 12 takes 18 (5 NV one value at a time). Afterwards lane l holds, in v[0 .. count), the
// totals of the values first_of(l) .. first_of(l) + count.
template <int NV>
struct WarpSums {
    static constexpr int kFirst = NV % 2 == 0 ? NV / 2 : NV;
    static constexpr int kCount = NV % 4 == 0 ? NV / 4 : kFirst;
    static __device__ __forceinline__ int first_of(int lane) {
        int f = 0;
        if constexpr (NV % 2 == 0) f += ((lane >> 4) & 1) * (NV / 2);
        if constexpr (NV % 4 == 0) f += ((lane >> 3) & 1) * (NV / 4);
        return f;
    }
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
    // Every lane gets every total.
    static __device__ __forceinline__ void broadcast(float (&v)[NV]) {
        float t[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) t[i] = __shfl_sync(0xffffffffu, v[i % kCount], holder_of(i));
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = t[i];
    }
};

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

// Decisions for four runs of 32 consecutive elements, one element of each run per lane: bit j of the result belongs to run j,
// whose lane 0 has element start[j]. A run touches at most 5 generator blocks, so 8 lanes work out the blocks of one run and
// hand the decisions round: one block per lane and 4 elements, not one per element.
__device__ __forceinline__ std::uint32_t keep_four_runs(const long long (&start)[4], const Philox& gen, std::uint32_t threshold) {
    const int lane = threadIdx.x & 31;
    long long mine = start[0];
#pragma unroll
    for (int j = 1; j < 4; ++j)
        if ((lane >> 3) == j) mine = start[j];
    const uint4 c = gen.block(static_cast<std::uint32_t>(mine >> 3) + (lane & 7));
    const std::uint32_t w[4] = {c.x, c.y, c.z, c.w};
    std::uint32_t kept = 0, out = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) kept |= (((i & 1) != 0 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu) >= threshold ? 1u : 0u) << i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = static_cast<int>(start[j] & 7) + lane;      // element of lane `lane`, counted from the run's first block
        out |= ((__shfl_sync(0xffffffffu, kept, j * 8 + (at >> 3)) >> (at & 7)) & 1u) << j;
    }
    return out;
}

// Hands every vector of a thread's R x CPT to `finish(r, c, values)` after its dropout map, reading them from `in`. Every lane of
// the warp must call this, whatever columns and rows it has.
template <typename T, int VEC, int CPT, int R, typename F>
__device__ __forceinline__ void drop_all(const RawOf<T, VEC> (&in)[R][CPT], long long row0, int hidden, int tpr, int tid, const Philox& gen,
                                         const DropoutArgs& args, const F& finish) {
    if constexpr (VEC == 1) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int j0 = 0; j0 < R * CPT; j0 += 4) {
            long long start[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) start[j] = (row0 + (j0 + j) / CPT) * hidden + (j0 + j) % CPT * tpr + tid - lane;
            const std::uint32_t kept = args.threshold != 0 ? keep_four_runs(start, gen, args.threshold) : 15u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = (j0 + j) / CPT, c = (j0 + j) % CPT;
                float v[1];
                unpack_raw<T, 1>(v, in[r][c]);
                v[0] = (kept >> j) & 1u ? __fmul_rn(v[0], args.scale) : 0.f;
                finish(r, c, v);
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                float v[VEC];
                unpack_raw<T, VEC>(v, in[r][c]);
                if (args.threshold != 0) drop_vec<VEC>(v, gen, (row0 + r) * hidden + (c * tpr + tid) * VEC, args);
                finish(r, c, v);
            }
    }
}

template <typename T, int VEC, int CPT, int R, bool FUSED>
__global__ void __launch_bounds__(kMaxTpr)
layernorm_forward_rows_kernel(T* __restrict__ y, T* sum, const T* x, const T* residual, const T* __restrict__ w,
                              const T* __restrict__ b, long long rows, int hidden, float epsilon, int tpr, const DropoutArgs args) {
    using Raw = RawOf<T, VEC>;
    __shared__ float red_all[2][16][R * 16];
    const int index = threadIdx.x / tpr, tid = threadIdx.x - index * tpr;
    const Group g{index, tpr >> 5, tid >> 5, static_cast<int>(threadIdx.x & 31)};
    const Philox gen(args);
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    const int groups = blockDim.x / tpr;
    const long long step = static_cast<long long>(gridDim.x) * groups * R;
    for (long long row0 = (static_cast<long long>(blockIdx.x) * groups + index) * R; row0 < rows; row0 += step) {
        Raw xp[R][CPT];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const int col = (c * tpr + tid) * VEC;
                xp[r][c] = row0 + r < rows && col < hidden ? __ldcs(reinterpret_cast<const Raw*>(x + (row0 + r) * hidden + col)) : Raw{};
            }
        if constexpr (FUSED) {
            Raw rp[R][CPT];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < CPT; ++c) {
                    const int col = (c * tpr + tid) * VEC;
                    rp[r][c] = row0 + r < rows && col < hidden ? __ldcs(reinterpret_cast<const Raw*>(residual + (row0 + r) * hidden + col)) : Raw{};
                }
            // the stored sum of vector j replaces the input in xp
            auto finish = [&](int r, int c, float (&v)[VEC]) {
                float rv[VEC];
                unpack_raw<T, VEC>(rv, rp[r][c]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] += rv[i];
                xp[r][c] = pack_raw<T, VEC>(v);
                const int col = (c * tpr + tid) * VEC;
                if (row0 + r < rows && col < hidden) *reinterpret_cast<Raw*>(sum + (row0 + r) * hidden + col) = xp[r][c];
                else xp[r][c] = Raw{};
            };
            drop_all<T, VEC, CPT, R>(xp, row0, hidden, tpr, tid, gen, args, finish);
        }
        float mean[R], var[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] = 0.f;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                float v[VEC];
                unpack_raw<T, VEC>(v, xp[r][c]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) mean[r] += v[i];
            }
        }
        keep_packed_all(xp);
        group_sum<R>(mean, g, red_all[0][index]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] *= inv_hidden;
            var[r] = 0.f;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                if ((c * tpr + tid) * VEC < hidden) {
                    float v[VEC];
                    unpack_raw<T, VEC>(v, xp[r][c]);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float d = v[i] - mean[r];
                        var[r] = fmaf(d, d, var[r]);
                    }
                }
            }
        }
        keep_packed_all(xp);
        group_sum<R>(var, g, red_all[1][index]);
#pragma unroll
        for (int r = 0; r < R; ++r) var[r] = rsqrtf(fmaf(var[r], inv_hidden, epsilon));
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = (c * tpr + tid) * VEC;
            if (col < hidden) {
                float wv[VEC], bv[VEC];
                load_vec<T, VEC>(wv, w + col);
                if (b != nullptr) load_vec<T, VEC>(bv, b + col);
                else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) bv[i] = 0.f;
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (row0 + r < rows) {
                        float v[VEC];
                        unpack_raw<T, VEC>(v, xp[r][c]);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) v[i] = fmaf(normalised(v[i], mean[r], var[r]), wv[i], bv[i]);
                        *reinterpret_cast<Raw*>(y + (row0 + r) * hidden + col) = pack_raw<T, VEC>(v);
                    }
                }
            }
        }
    }
}

// partial: [gridDim.x][2][hidden]
template <typename T, int VEC, int CPT, int R, bool FUSED>
__global__ void __launch_bounds__(kMaxTpr)
layernorm_backward_rows_kernel(T* dx, T* din, float* __restrict__ partial, const T* __restrict__ dy, const T* __restrict__ x,
                               const T* __restrict__ w, const T* residual, long long rows, int hidden, float epsilon, int tpr,
                               const DropoutArgs args) {
    using Raw = RawOf<T, VEC>;
    extern __shared__ float shared[];                          // the groups' sums, then (reused) their dw and db
    const int index = threadIdx.x / tpr, tid = threadIdx.x - index * tpr;
    const Group g{index, tpr >> 5, tid >> 5, static_cast<int>(threadIdx.x & 31)};
    float* red = shared + index * (4 * R * 16);
    const Philox gen(args);
    const float inv_hidden = 1.0f / static_cast<float>(hidden);
    const int groups = blockDim.x / tpr;
    float aw[CPT][VEC] = {}, ab[CPT][VEC] = {};
    const long long step = static_cast<long long>(gridDim.x) * groups * R;
    for (long long row0 = (static_cast<long long>(blockIdx.x) * groups + index) * R; row0 < rows; row0 += step) {
        Raw xp[R][CPT], gp[R][CPT], rp[R][CPT];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const int col = (c * tpr + tid) * VEC;
                const bool in = row0 + r < rows && col < hidden;
                const long long e = (row0 + r) * hidden + col;
                xp[r][c] = in ? __ldcs(reinterpret_cast<const Raw*>(x + e)) : Raw{};
                gp[r][c] = in ? __ldcs(reinterpret_cast<const Raw*>(dy + e)) : Raw{};
            }
        float mean[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] = 0.f;
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                float v[VEC];
                unpack_raw<T, VEC>(v, xp[r][c]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) mean[r] += v[i];
            }
        }
        // only the output needs the residual: on its way while the sums are reduced
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const int col = (c * tpr + tid) * VEC;
                rp[r][c] = residual != nullptr && row0 + r < rows && col < hidden
                               ? __ldcs(reinterpret_cast<const Raw*>(residual + (row0 + r) * hidden + col)) : Raw{};
            }
        keep_packed_all(xp);
        group_sum<R>(mean, g, red);
        float sums[3 * R];
#pragma unroll
        for (int r = 0; r < R; ++r) mean[r] *= inv_hidden;
#pragma unroll
        for (int i = 0; i < 3 * R; ++i) sums[i] = 0.f;
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = (c * tpr + tid) * VEC;
            if (col < hidden) {
                float wv[VEC];
                load_vec<T, VEC>(wv, w + col);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float xv[VEC], gv[VEC], s[3] = {sums[r], sums[R + r], sums[2 * R + r]};
                    unpack_raw<T, VEC>(xv, xp[r][c]);
                    unpack_raw<T, VEC>(gv, gp[r][c]);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) norm_sums(s, gv[i], wv[i], xv[i] - mean[r]);
                    sums[r] = s[0];
                    sums[R + r] = s[1];
                    sums[2 * R + r] = s[2];
                }
            }
        }
        keep_packed_all(xp);
        keep_packed_all(gp);
        group_sum<3 * R>(sums, g, red + R * 16);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sums[r] = rsqrtf(fmaf(sums[r], inv_hidden, epsilon));                // rstd
            sums[R + r] *= inv_hidden;                                           // c1
            sums[2 * R + r] = sums[2 * R + r] * inv_hidden * sums[r];            // c2
        }
        float single[VEC == 1 && FUSED ? R * CPT : 1];   // outputs of single elements, whose decisions are made four at a time
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = (c * tpr + tid) * VEC;
            float wv[VEC] = {};
            if (col < hidden) load_vec<T, VEC>(wv, w + col);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const long long e = (row0 + r) * hidden + col;
                const bool in = row0 + r < rows && col < hidden;
                float xv[VEC], gv[VEC], out[VEC];
                unpack_raw<T, VEC>(xv, xp[r][c]);
                unpack_raw<T, VEC>(gv, gp[r][c]);
                unpack_raw<T, VEC>(out, rp[r][c]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = normalised(xv[i], mean[r], sums[r]);
                    out[i] = norm_dx(gv[i], wv[i], xh, sums[r], sums[R + r], sums[2 * R + r], out[i]);
                    aw[c][i] = fmaf(gv[i], xh, aw[c][i]);      // rows past the end: dy = 0
                    ab[c][i] += gv[i];
                }
                if (in) *reinterpret_cast<Raw*>(dx + e) = pack_raw<T, VEC>(out);
                if constexpr (FUSED && VEC > 1) {
                    if (args.threshold != 0) drop_vec<VEC>(out, gen, e, args);
                    if (in) *reinterpret_cast<Raw*>(din + e) = pack_raw<T, VEC>(out);
                } else if constexpr (FUSED) {
                    single[r * CPT + c] = out[0];
                }
            }
        }
        if constexpr (FUSED && VEC == 1) {
            const int lane = threadIdx.x & 31;
#pragma unroll
            for (int j0 = 0; j0 < R * CPT; j0 += 4) {
                long long start[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) start[j] = (row0 + (j0 + j) / CPT) * hidden + (j0 + j) % CPT * tpr + tid - lane;
                const std::uint32_t kept = args.threshold != 0 ? keep_four_runs(start, gen, args.threshold) : 15u;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = (j0 + j) / CPT, c = (j0 + j) % CPT;
                    if (row0 + r < rows && c * tpr + tid < hidden)
                        din[start[j] + lane] = from_f32<T>((kept >> j) & 1u ? __fmul_rn(single[j0 + j], args.scale) : 0.f);
                }
            }
        }
    }
    // The groups of a CTA add up their columns one after the other: one partial row of dw and of db per CTA.
    float* out_w = partial + static_cast<long long>(blockIdx.x) * 2 * hidden;
    if (groups == 1) {
#pragma unroll
        for (int c = 0; c < CPT; ++c) {
            const int col = (c * tpr + tid) * VEC;
            if (col < hidden) {
                store_floats<VEC>(out_w + col, aw[c]);
                store_floats<VEC>(out_w + hidden + col, ab[c]);
            }
        }
        return;
    }
    for (int k = 0; k < groups; ++k) {
        __syncthreads();
        if (index == k) {
#pragma unroll
            for (int c = 0; c < CPT; ++c) {
                const int at = (c * tpr + tid) * VEC;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float* s = shared + (i * CPT + c) * tpr * 2 + tid;   // one float per thread and value: no bank conflicts
                    const float tw = (k == 0 ? 0.f : s[0]) + aw[c][i], tb = (k == 0 ? 0.f : s[tpr]) + ab[c][i];
                    s[0] = tw;
                    s[tpr] = tb;
                    if (k == groups - 1 && at + i < hidden) {
                        out_w[at + i] = tw;
                        out_w[hidden + at + i] = tb;
                    }
                }
            }
        }
    }
}

}  // namespace rows_kernels
