// Counter-based dropout decisions: Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011), one 128-bit block per eight elements.
//
// Element e of a tensor (row-major index) takes 16 bits of the block with
//     key = (seed low, seed high), counter = (e / 8, site, step low, step high):
// half e % 8 of the four words, low halves first. It is kept where those bits are >= threshold = round(65536 p) and then
// multiplied by 65536 / (65536 - threshold), so the expectation is exact for the probability that is realised (p in steps of
// 2^-16). Forward and backward recompute the same bits; no mask is stored. seed and step are read from device memory
// ({seed, step}, two 64-bit words), so that a captured graph draws new masks when the step is advanced between replays.
//
// Sixteen bits a decision, not 32: a block's ten rounds (two 32x32->64 products, four XORs and two key additions each) then
// cover 16 bytes of a 16-bit tensor. With them dropout of a bf16 tensor still runs at memory speed (32768 x 2048 with a residual:
// 98 % of a plain copy's rate in a loop, 94 % with other work between the calls).
#pragma once

#include <cmath>
#include <initializer_list>

#include "common.cuh"
#include "pairs.cuh"

namespace cgpt {

struct DropoutArgs {
    const unsigned long long* state;   // {seed, step} in device memory; not read when threshold == 0
    std::uint32_t site;
    std::uint32_t threshold;           // 0: nothing is dropped
    float scale;                       // 65536 / (65536 - threshold)
};

// The generator of one call. Of a block's counter only the first word differs within a call, so half of the first two rounds is
// the same for all blocks and worked out once: of the second word's product in round 1 and the first word's in round 2 only what
// the later rounds XOR in is kept, with the round keys (fused backward 32768 x 1024 2.5 us less of 74, lookup of as many 1 of 28).
//
// What a call's constants take in registers is chosen by kernel. kLeft: the compiler works them out again where registers are short.
// kKept: it may not. At every block the two products and their loads cost more than the registers: fused odd rows 128 | 152 us
// forward (32768 x 1001 bf16) and 225 | 246 backward (8192 x 4099 fp16), fused forward of 4096 x 8192 bf16 56 | 62. The fused
// forward of up to four vectors a lane has better use for them (32768 x 1024 fp16 51.6 | 50.3). kHoisted: the keys of all rounds
// are kept as well, which saves their additions where registers are free; then the constants are left (lookup 24.6 | 23.8 us).
enum class Constants { kLeft, kKept, kHoisted };

template <Constants C>
struct PhiloxOf {
    static constexpr bool HOIST = C == Constants::kHoisted;
    static constexpr std::uint32_t kMul0 = 0xD2511F53u, kMul1 = 0xCD9E8D57u, kKey0 = 0x9E3779B9u, kKey1 = 0xBB67AE85u;
    std::uint32_t z1, x2, z2, z3;                                    // what rounds 1 to 3 XOR into words 2, 0, 2 and 2
    std::uint32_t k0[HOIST ? 8 : 1], k1[HOIST ? 8 : 1];              // keys of rounds 3 and later (k1[0] is in z3)

    __device__ __forceinline__ explicit PhiloxOf(const DropoutArgs& a) {
        const unsigned long long seed = a.threshold != 0 ? a.state[0] : 0ull, step = a.threshold != 0 ? a.state[1] : 0ull;
        const std::uint32_t s0 = static_cast<std::uint32_t>(seed), s1 = static_cast<std::uint32_t>(seed >> 32);
        const unsigned long long q = static_cast<unsigned long long>(kMul1) * static_cast<std::uint32_t>(step);
        const unsigned long long p = static_cast<unsigned long long>(kMul0) * (static_cast<std::uint32_t>(q >> 32) ^ a.site ^ s0);
        z1 = static_cast<std::uint32_t>(step >> 32) ^ s1;
        x2 = static_cast<std::uint32_t>(q) ^ (s0 + kKey0);
        z2 = static_cast<std::uint32_t>(p >> 32) ^ (s1 + kKey1);
        z3 = static_cast<std::uint32_t>(p) ^ (s1 + 2 * kKey1);
        k0[0] = s0 + 2 * kKey0;
        k1[0] = s1 + 2 * kKey1;
        if constexpr (C == Constants::kKept) asm volatile("" : "+r"(z1), "+r"(x2), "+r"(z2), "+r"(z3), "+r"(k0[0]), "+r"(k1[0]));
        if constexpr (HOIST) {
#pragma unroll
            for (int r = 1; r < 8; ++r) {
                k0[r] = k0[r - 1] + kKey0;
                k1[r] = k1[r - 1] + kKey1;
                asm volatile("" : "+r"(k0[r]), "+r"(k1[r]));   // or they are added up again at every use
            }
        }
    }
    __device__ __forceinline__ uint4 block(std::uint32_t index) const {
        const unsigned long long p1 = static_cast<unsigned long long>(kMul0) * index;
        const unsigned long long q2 = static_cast<unsigned long long>(kMul1) * (static_cast<std::uint32_t>(p1 >> 32) ^ z1);
        uint4 c = make_uint4(static_cast<std::uint32_t>(q2 >> 32) ^ x2, static_cast<std::uint32_t>(q2), static_cast<std::uint32_t>(p1) ^ z2, 0u);
        std::uint32_t ka = k0[0], kb = k1[0];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if constexpr (HOIST) {
                ka = k0[r];
                kb = k1[r];
            }
            const unsigned long long p = static_cast<unsigned long long>(kMul0) * c.x;
            const unsigned long long q = static_cast<unsigned long long>(kMul1) * c.z;
            c = make_uint4(static_cast<std::uint32_t>(q >> 32) ^ c.y ^ ka, static_cast<std::uint32_t>(q),
                           static_cast<std::uint32_t>(p >> 32) ^ (r == 0 ? z3 : c.w ^ kb), static_cast<std::uint32_t>(p));
            if constexpr (!HOIST) {
                ka += kKey0;
                kb += kKey1;
            }
        }
        return c;
    }
};
using Philox = PhiloxOf<Constants::kLeft>;
using KeptPhilox = PhiloxOf<Constants::kKept>;
using HoistedPhilox = PhiloxOf<Constants::kHoisted>;

// Decisions are made on the high half of a word (its low half may hold anything: u >= t * 2^16 exactly if its high half >= t).
// Products by the scale are rounded by themselves (no contraction with a residual added to them), so that every kernel gives the
// same bits.

// The dropout map of NP pairs that start at element e of the tensor (e % (2 NP) == 0, NP 2 or 4). Dropped elements become +0
// whatever they held. SCALED: kept elements are multiplied by the scale (else the caller does that later).
template <int NP, bool SCALED = true, typename Generator>
__device__ __forceinline__ void drop_pairs(Pair (&p)[NP], const Generator& gen, long long e, const DropoutArgs& args) {
    const uint4 c = gen.block(static_cast<std::uint32_t>(e >> 3));
    const bool upper = NP == 2 && (e & 4) != 0;
    const std::uint32_t w[4] = {upper ? c.z : c.x, upper ? c.w : c.y, c.z, c.w};
    const Pair scale = pair(args.scale);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const float2 f = both(SCALED ? mul2(p[i], scale) : p[i]);
        p[i] = pair(w[i] << 16 >= args.threshold << 16 ? f.x : 0.f, w[i] >= args.threshold << 16 ? f.y : 0.f);
    }
}

// The decision of one element, for places that cannot share a block (its other seven decisions are thrown away).
template <bool SCALED = true, typename Generator>
__device__ __forceinline__ float apply_one(float v, const Generator& gen, long long e, const DropoutArgs& a) {
    const uint4 c = gen.block(static_cast<std::uint32_t>(e >> 3));
    const int i = static_cast<int>(e & 7);
    const std::uint32_t w = i < 4 ? (i < 2 ? c.x : c.y) : (i < 6 ? c.z : c.w);
    return ((i & 1) != 0 ? w : w << 16) >= a.threshold << 16 ? (SCALED ? __fmul_rn(v, a.scale) : v) : 0.f;
}

// A block's eight decisions as bits.
__device__ __forceinline__ std::uint32_t kept_bits(const uint4& c, std::uint32_t threshold) {
    const std::uint32_t w[4] = {c.x, c.y, c.z, c.w};
    std::uint32_t kept = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) kept |= ((i & 1) != 0 ? w[i >> 1] : w[i >> 1] << 16) >= threshold << 16 ? 1u << i : 0u;
    return kept;
}

// Decisions for four runs of 32 consecutive elements, one element of each run per lane: bit j of the result belongs to run j,
// whose lane 0 has element start[j]. A run touches at most 5 generator blocks, so 8 lanes work out the blocks of one run and
// hand the decisions round: one block per lane and 4 elements, not one per element.
template <typename Generator>
__device__ __forceinline__ std::uint32_t keep_four_runs(const long long (&start)[4], const Generator& gen, std::uint32_t threshold) {
    const int lane = threadIdx.x & 31;
    long long mine = start[0];
#pragma unroll
    for (int j = 1; j < 4; ++j)
        if ((lane >> 3) == j) mine = start[j];
    const std::uint32_t kept = kept_bits(gen.block(static_cast<std::uint32_t>(mine >> 3) + (lane & 7)), threshold);
    std::uint32_t out = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = static_cast<int>(start[j] & 7) + lane;      // element of lane `lane`, counted from the run's first block
        out |= ((__shfl_sync(0xffffffffu, kept, j * 8 + (at >> 3)) >> (at & 7)) & 1u) << j;
    }
    return out;
}

// Whether every pointer given (NULL ones aside) is aligned to an element of `dtype`.
inline bool element_aligned(int dtype, std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if ((reinterpret_cast<std::uintptr_t>(p) & (dtype_size(dtype) - 1)) != 0) return false;
    return true;
}

// Checks the options of a call with dropout over `elements` elements and fills `out`. A probability of 0 reads no state.
inline int dropout_args(DropoutArgs* out, float probability, const void* state, std::uint32_t site, unsigned long long elements) {
    *out = DropoutArgs{static_cast<const unsigned long long*>(state), site, 0u, 1.0f};
    if (!(probability >= 0.f && probability < 1.f)) return CGPT_ERR_OPTION;
    if (probability == 0.f) return CGPT_OK;
    if (state == nullptr) return CGPT_ERR_NULL;
    if ((reinterpret_cast<std::uintptr_t>(state) & 7u) != 0) return CGPT_ERR_ALIGN;
    if (elements > (1ull << 35)) return CGPT_ERR_SHAPE;   // the block counter has 32 bits
    const double t = std::nearbyint(static_cast<double>(probability) * 65536.0);
    out->threshold = static_cast<std::uint32_t>(t > 65535.0 ? 65535.0 : t);
    out->scale = static_cast<float>(65536.0 / (65536.0 - static_cast<double>(out->threshold)));
    return CGPT_OK;
}

}  // namespace cgpt
