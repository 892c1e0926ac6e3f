// kvattention.cuh -- what the paged attention's kernels share: the launch
// parameters, the partial results and the even split of the line of units.
#pragma once
#include "kvpages.cuh"

namespace hsb {

constexpr unsigned kAttnMaxCtas = 160;
constexpr int kPartFloats = kGroup * 2 + kGroup * kDim;  // (max in log2 units, sum) per head, then the outputs
constexpr size_t kMaxBatch = 1u << 20;
constexpr size_t kMaxTableEntries = 1ull << 27;  // keeps the units of 8 heads within 32 bits
constexpr size_t kMaxPrefix = 1ull << 30;
// log2(e) / sqrt(128): logits in the unit of exp2
constexpr float kScaleLog2 = 1.4426950408889634f * 0.08838834764831845f;

// Of the run that begins in a CTA's stretch and ends in another's (run < 0: none).
struct RunInfo {
    int run;     // sequence * heads + head
    uint32_t last;  // the CTA that ends it
};

struct PagedAttention {
    PagedView v;
    const int32_t* lengths;      // [batch]
    unsigned long long batch;
    const void* q;               // [batch][4 heads][128]
    float* out;                  // final mode: F32 [batch][4 heads][128]
    float* part;                 // [CTA][2][kPartFloats]: runs cut at a stretch's begin, at its end
    float* whole;                // partial mode: [run][kPartFloats], runs of one stretch
    RunInfo* info;               // [CTA], final mode
    int by_run;                  // CTA r has run r: nothing is cut, `part` and `info` are not used
    uint32_t* place;             // partial mode: [run], of a run with tokens: 0 (in `whole`) or cut_run()
    hsb_device_status* status;
    float scale_log2;
};

// An even split of `units` (places of the line) over n: the first units % n stretches have one more than the others.
struct Split {
    uint32_t each, more;
    Split() = default;
    __host__ __device__ Split(uint32_t units, uint32_t n) : each(units / n), more(units % n) {}
    __host__ __device__ uint32_t begin(uint32_t c) const { return each * c + (c < more ? c : more); }
    // The stretch that holds unit u.
    __host__ __device__ uint32_t of(uint32_t u) const {
        const uint32_t longer = (each + 1) * more;
        return u < longer ? u / (each + 1) : more + (u - longer) / each;
    }
};

// A run cut over `count` CTAs from `first` on: in the first CTA's part [1], the others' [0].
__host__ __device__ constexpr uint32_t cut_run(uint32_t first, uint32_t count) { return first << 16 | count; }
// The partials of a run with tokens, whose place is this word, in a grid of that many CTAs.  A warp that gave up
// its wait leaves its runs' places as the workspace was: a word that names CTAs outside the grid counts as none.
__host__ __device__ constexpr uint32_t run_partials(uint32_t place, uint32_t grid) {
    return place == 0 ? 1 : (place >> 16) + (place & 0xffffu) <= grid ? place & 0xffffu : 0;
}

// 2^x; a result below the normal range is 0.
__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// True in one lane of the warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
inline size_t align256(size_t b) { return (b + 255) / 256 * 256; }

// Whether a run is to be a CTA's whole work, by what the host knows of its length; and the grid.
bool paged_by_run(size_t batch, size_t table_width, int heads);
unsigned paged_attention_grid(size_t batch, size_t table_width, int heads);
// The tokens of a sequence; a length behind the table's end counts as none.
__device__ __forceinline__ uint32_t tokens_in(const int32_t* lengths, unsigned long long width, uint32_t b) {
    const int32_t n = lengths[b];
    return n < 0 || (unsigned long long)n > width * kPageTokens ? 0 : n;
}
cudaError_t launch_paged_partials(int format, const PagedAttention& p, unsigned grid, cudaStream_t stream);

}  // namespace hsb
