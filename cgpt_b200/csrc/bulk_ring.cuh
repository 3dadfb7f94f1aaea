// A ring of stages in shared memory that one thread (the leader) fills with bulk copies and others read: what the rings of the
// layer norm kernels have in common. They add a fill() for their layout of rows.
#pragma once

#include "sm100.cuh"

namespace cgpt {

// A wait that runs out sets the library's status word; the CTA then goes on with what is there (every barrier is still met,
// nothing is written out of bounds) and waits no more.
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
    __device__ __forceinline__ unsigned char* wait() {
        if (!failed && !sm100::mbar_wait(&full[stage], parity)) {
            failed = true;
            atomicExch(status, 5u);
        }
        return data + stage * stage_bytes;
    }
    __device__ __forceinline__ void next() {
        if (++stage == stages) { stage = 0; parity ^= 1u; }
    }
    // Before the CTA leaves: copies that a failed wait gave up on get time to land while the memory is still its own.
    __device__ __forceinline__ void leave() const {
        if (failed) {
            const unsigned long long t0 = sm100::globaltimer_ns();
            while (sm100::globaltimer_ns() - t0 < 200000ull) { }
        }
    }
};

}  // namespace cgpt
