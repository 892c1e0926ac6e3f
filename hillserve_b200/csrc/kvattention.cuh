// kvattention.cuh -- what the paged attention's kernels share: the launch
// parameters, the partial results and the even split of the line of units.
#pragma once
#include "kvpages.cuh"

namespace hsb {

constexpr unsigned kAttnMaxCtas = 512;
constexpr int kPartFloats = kGroup * 2 + kGroup * kDim;  // (max in log2 units, sum) per head, then the outputs
constexpr size_t kMaxBatch = 1u << 20;
constexpr size_t kMaxTableEntries = 1ull << 31;  // keeps a stretch's half pages within 32 bits
// log2(e) / sqrt(128): logits in the unit of exp2
constexpr float kScaleLog2 = 1.4426950408889634f * 0.08838834764831845f;

// Of the run that begins in a CTA's stretch and ends in another's (run < 0: none).
struct RunInfo {
    long long run;             // sequence * heads + head
    unsigned long long units;  // of all stretches
    unsigned last;             // the CTA that ends it
};

struct PagedAttention {
    PagedView v;
    const int32_t* lengths;      // [batch], or null: `length` for every sequence
    unsigned long long length;
    unsigned long long batch;
    const void* q;               // [batch][4 heads][128]
    float* out;                  // final mode: F32 [batch][4 heads][128]
    float* part;                 // [CTA][2][kPartFloats]: runs cut at a stretch's begin, at its end
    float* whole;                // partial mode: [run][kPartFloats], runs of one stretch
    RunInfo* info;               // [CTA]
    unsigned long long* cum;     // partial mode: [batch + 1] pages before each sequence
    hsb_device_status* status;
    float scale_log2;
};

// Stretch c of n over `units`: [stretch_begin(c), stretch_begin(c + 1)).
__host__ __device__ inline unsigned long long stretch_begin(unsigned long long units, unsigned c, unsigned n) {
    return units * c / n;
}
// The stretch that holds unit u: the last c with stretch_begin(c) <= u.
__host__ __device__ inline unsigned stretch_of(unsigned long long units, unsigned long long u, unsigned n) {
    return (unsigned)(((u + 1) * n + units - 1) / units - 1);
}

unsigned paged_attention_grid(size_t units);
cudaError_t launch_paged_partials(int format, const PagedAttention& p, unsigned grid, cudaStream_t stream);

}  // namespace hsb
