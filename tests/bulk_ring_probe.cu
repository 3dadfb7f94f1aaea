// One CTA walks a ring of three stages of which the last is never filled: the wait for it runs out after a short limit. Every
// access stays inside the buffers that run_probe's caller gives (source: kStages * kBytes * 2 bytes; report: Report) and every
// wait is bounded.
#include "../cgpt_b200/csrc/bulk_ring.cuh"

namespace {

constexpr int kThreads = 64, kStages = 3, kSteps = 7;
constexpr unsigned kBytes = kThreads * 4;
constexpr unsigned long long kLimitNs = 20000000ull;   // 20 ms

struct Report {
    unsigned status, armed, refused, failed_threads, late, failed_at[kSteps], seen[kSteps][kThreads], landed[2][kThreads];
};

__global__ void __launch_bounds__(kThreads) probe_kernel(const unsigned char* source, Report* report) {
    __shared__ __align__(128) unsigned char data[kStages * kBytes];
    __shared__ std::uint64_t full[kStages];
    cgpt::BulkRing ring{};
    ring.data = data;
    ring.full = full;
    ring.status = &report->status;
    ring.stage_bytes = kBytes;
    ring.stages = kStages;
    bool leader = threadIdx.x == 0;
    unsigned filled = 0;
    auto fill = [&](int s) {
        if (leader != (threadIdx.x == 0 && !ring.failed)) report->late = 2;      // the two ways to ask agree
        if (leader) {
            cgpt::sm100::mbar_expect_tx(&full[s], kBytes);
            cgpt::sm100::bulk_load_1d(data + s * kBytes, source + filled * kBytes, kBytes, &full[s]);
            ++filled;
        } else if (threadIdx.x == 0) {
            ++report->refused;
        }
    };
    if (leader) {
        ring.init();
        fill(0);
        fill(1);
    }
    __syncthreads();
    const unsigned long long start = cgpt::sm100::globaltimer_ns();
    for (int step = 0; step < kSteps; ++step) {
        const unsigned* at = reinterpret_cast<const unsigned*>(ring.wait(&leader, kLimitNs));
        if (step < 2) report->seen[step][threadIdx.x] = at[threadIdx.x];
        if (threadIdx.x == 0) report->failed_at[step] = ring.failed ? 1 + ring.stage : 0;
        __syncthreads();
        fill(ring.stage);
        ring.next();
    }
    if (__syncthreads_or(cgpt::sm100::globaltimer_ns() - start > 100 * kLimitNs)) report->late = 1;
    atomicAdd(&report->failed_threads, ring.failed ? 1u : 0u);
    for (int s = 0; s < 2; ++s) report->landed[s][threadIdx.x] = reinterpret_cast<const unsigned*>(data)[s * kThreads + threadIdx.x];
    if (threadIdx.x == 0) report->armed = filled;
}

}  // namespace

extern "C" int report_words() { return sizeof(Report) / 4; }
extern "C" int run_probe(const void* source, void* report, void* stream) {
    probe_kernel<<<1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const unsigned char*>(source), static_cast<Report*>(report));
    return static_cast<int>(cudaGetLastError());
}
