// A ring of stages in shared memory that one thread (the leader) fills with bulk copies and others read: what the rings of the
// layer norm kernels have in common. They add a fill() for their layout of rows.
#pragma once

#include "sm100.cuh"

namespace cgpt {

// Every thread that reads keeps its own copy of this state. Where a wait runs out, the thread sets the library's status word and
// waits once more for all that may be on its way, so that no copy outlives the CTA; it then goes on with what is there (every
// barrier of the CTA is still met, nothing is written out of bounds) and waits no more. A leader must not copy anything after that:
// the stage's barrier is in a phase that has had its one arrival, and the stage may still be written to. The forward kernels keep
// whether a thread fills in a variable that wait() clears, the backward ones ask `failed` before a fill. The other way round cost
// registers: fused forward 4096 x 8192 bf16 61.5 instead of 60.0 us, fused backward 8192 x 4099 fp16 259 instead of 245.
struct BulkRing {
    unsigned char* data;
    std::uint64_t* full;
    unsigned int* status;
    unsigned stage_bytes, tensor_bytes;
    int stages, stage;
    std::uint32_t parity;
    bool failed;

    __device__ __forceinline__ void init() const {   // by one thread, before the CTA's first barrier
        for (int s = 0; s < stages; ++s) sm100::mbar_init(&full[s], 1);
        sm100::mbar_init_fence();
    }
    __device__ __forceinline__ unsigned char* wait(bool* leader = nullptr, unsigned long long limit_ns = sm100::kWaitLimitNs) {
        if (!failed && !sm100::mbar_wait(&full[stage], parity, limit_ns)) {
            failed = true;
            if (leader != nullptr) *leader = false;
            atomicExch(status, 5u);
            let_copies_land(limit_ns);
        }
        return data + stage * stage_bytes;
    }
    __device__ __forceinline__ void next() {
        if (++stage == stages) { stage = 0; parity ^= 1u; }
    }

private:
    // This stage and those behind it, within one limit (which runs out where a stage was never filled).
    __device__ __forceinline__ void let_copies_land(unsigned long long limit_ns) const {
        const unsigned long long start = sm100::globaltimer_ns();
        int s = stage;
        std::uint32_t p = parity;
        for (int k = 0; k < stages; ++k) {
            while (!sm100::mbar_try_wait(&full[s], p) && sm100::globaltimer_ns() - start < limit_ns) { }
            if (++s == stages) { s = 0; p ^= 1u; }
        }
    }
};

}  // namespace cgpt
