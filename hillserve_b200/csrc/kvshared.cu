// kvshared.cu -- decode attention of a batch whose sequences share a prefix.
//
// The prefix is where the arithmetic is: every row of the batch (four query
// heads to a sequence and KV head) meets the same K and V, so the batch's rows
// are the M dimension of two real matrix products and the prefix is read once
// (for 64 sequences; again from L2 for each further 64).  kv_prefix_kernel runs
// them on the tensor cores' own pipeline:
//
//   S[row][token] = Q K^T      A = Q (shared memory), B = K (shared memory, K-major)
//   O[row][ch]   += P V        A = P (tensor memory), B = V (shared memory, MN-major)
//
// with M = 128 rows (32 sequences), tiles of 128 tokens, both accumulators in
// tensor memory.  A page's F16 panels already are the operands' 128-byte
// swizzled layout, so the loader is four 8 KB bulk copies a tile and operand.
// Two warpgroups own one M tile each: thread = row reads its 128 logits from
// tensor memory, forms the weights without any exchange and writes them back
// as F16 over the logits; while one softmax runs, the other tile's products do.
// The next logits go over those weights once the product that reads them is done.
// For at most 32 sequences there is one M tile, and the two warpgroups take the
// even and the odd tokens' tiles of it instead.
//
// The (KV head, M tiles, token tile) units are split evenly over the SMs; each
// stretch of a run leaves F32 partials, summed in parts of 256 tiles.  A stretch that ends one run and begins
// the next pays for a second query tile and a second result, so long lines keep
// idle places for that before each run.  The sequences' own tokens go through
// the paged kernel (kvattention.cu), and kv_shared_combine_kernel folds both.
//
// Measured (B200, 8 KV heads, one call in a captured graph): 64 sequences on 32768
// tokens 58.2 us, 256 on 16461 94 to 100, 8 on 4097 14.5.  A unit (two M tiles, 128
// tokens) takes a SM 1.86 us where the prefix stays in L2 (256 sequences; 1.76 if
// the logits did not wait for the product before), with no waits for the weights
// either 1.38, 1.8 PFLOP/s over the chip; where it comes from memory (64 sequences)
// 1.95, its bytes alone 1.40.  192 KB of shared memory are read a
// unit and 64 KB written, as many cycles (2048) as the products take at best.
// Half-width logits, twice as many softmax warps, weights handed over in smaller
// parts, and a pair of SMs on one tile gained nothing.  Around that loop the prefix
// kernel spends 11 us on the queries, the first tile and the results; the own tokens
// add 11 and 20 us, the combine 7.
#include <algorithm>

#include "kvattention.cuh"

namespace hsb {
namespace {

constexpr int kTileRows = 128, kTileTokens = 128;
constexpr int kTileSeqs = kTileRows / kGroup;
constexpr int kTileBytes = kTileTokens * 256;       // K or V of a tile; also a Q tile
constexpr int kTilePanel = kTileTokens * 128;       // its 64-channel half
constexpr int kSoftmaxThreads = 256;
constexpr int kMmaWarp = 8, kLoadWarp = 9;          // of a third warpgroup, which gives its registers
constexpr int kPrefixThreads = 384;                 // to the other two (setmaxnreg)
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;
// Weights are at most 2^kTop, and 2^kUnit at the largest logit that moved the reference; it moves when one is 2^(kTop -
// kUnit) above it.  F16 ends at 2^16 and keeps 11 bits down to 2^-14, so a weight keeps them down to 2^-21 of a
// stretch's largest and is off by 2^-32 of it at most below that (with no unit, 2^-25: the tail behind one dominant
// token was lost).  A larger unit keeps more and moves more often: 64 x 32768 takes 58.6 us with 7, 59.1 with 11,
// 61.6 with 14 (58.4 with none).
constexpr float kTop = 15.0f, kUnit = 7.0f;
// Weights are 2^(logit x scale - reference), one FMA.  The reference is the largest logit's product, rounded: by 2^-4
// at most up to 2^20, where weights may just as well be relative to it.  Behind that the rounding would leave F16's
// range, so the difference is formed before the scale.
constexpr float kFar = 1048576.0f;
constexpr int kLive = 16;                           // ring of tiles' live counts
// a partial: outputs [32 channel quads][128 rows][4], then (max, sum) [128 rows]
constexpr int kRowsFloats = kTileRows * kDim + 2 * kTileRows;

// kDual: one M tile, the warpgroups take alternate token tiles.
template <bool kDual>
struct Plan {
    static constexpr int kQBytes = (kDual ? 1 : 2) * kTileBytes;
    static constexpr int kStages = kDual ? 6 : 5;
    static constexpr int kSmem = 1024 + kQBytes + kStages * kTileBytes;
};

struct PrefixParams {
    PagedView v;         // the prefix pool; table [ceil(tokens / 64)]
    uint32_t tokens, tiles;
    const uint16_t* q;   // F16 [batch][4 heads][128]
    uint32_t batch, groups;  // groups: of M tiles (one or two)
    uint32_t runs;       // heads x groups
    uint32_t run_cost;   // idle places of a run
    float* part;         // [stretch + run][2][kRowsFloats]
    hsb_device_status* status;
    float scale_log2;
};

// ---------------------------------------------------------------- tcgen05
__device__ __forceinline__ void tmem_alloc(uint32_t* out, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(out)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives on `bar` when every product this thread issued has completed.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
// Descriptor of a 128-byte-swizzled operand: 8-row groups 1024 bytes apart, and
// for an MN-major one the 64-element halves `leading` bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t leading) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// F16 operands, F32 accumulator, M = N = 128; B K-major or MN-major.
constexpr uint32_t kShapeK = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kShapeMN = kShapeK | (1u << 16);
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void tc_mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(shape), "r"((uint32_t)add)
        : "memory");
}
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_load32(uint32_t at, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Generic writes to shared memory before the tensor cores or bulk copies use it.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---------------------------------------------------------------- softmax
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// The larger one; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// Two F32 values in a register pair, and the paired operations.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void split_of(uint64_t d, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// With two M tiles one pair of kByPolynomial takes its powers of two from the FMA
// units, as the special-function unit alone (16 a clock) would take as long as the
// products:
// 2^y = 2^n 2^f with n the nearest integer (adding 1.5 2^23 rounds to it) and
// 2^f on [-0.5, 0.5] a polynomial of degree 4, fitted for the least largest
// relative error (2.7e-6; a weight is rounded to F16 by 5e-4 next).  256 x 16461
// takes 94.4 us with every fourth pair, 97.2 with every eighth, 95.8 with none; a
// single M tile, where nothing runs beside a tile's softmax but the other tokens',
// 14.7 (8 x 4097) and 14.5 with none.
constexpr int kByPolynomial = 4;
__device__ __forceinline__ void exp2_pair(uint64_t y2, float& a, float& b) {
    constexpr float kRound = 12582912.0f;
    float ya, yb;
    split_of(y2, ya, yb);
    const uint64_t y = pair_of(max_nan(ya, -126.0f), max_nan(yb, -126.0f));  // (-infinity too: 2^-126 is 0 in F16)
    const uint64_t t = add2(y, pair_of(kRound, kRound));
    const uint64_t f = add2(y, fma2(t, pair_of(-1.0f, -1.0f), pair_of(kRound, kRound)));
    uint64_t v = pair_of(0.0095701013f, 0.0095701013f);
    v = fma2(v, f, pair_of(0.0559178591f, 0.0559178591f));
    v = fma2(v, f, pair_of(0.2402474433f, 0.2402474433f));
    v = fma2(v, f, pair_of(0.6931217909f, 0.6931217909f));
    v = fma2(v, f, pair_of(0.9999992847f, 0.9999992847f));
    float ta, tb;
    split_of(t, ta, tb);
    // (a product, not a sum of exponents: NaN stays NaN)
    split_of(mul2(v, pair_of(__uint_as_float((__float_as_uint(ta) << 23) + 0x3f800000u),
                             __uint_as_float((__float_as_uint(tb) << 23) + 0x3f800000u))), a, b);
}

// Waits for a phase; gives up after kWaitLimitNs or once another role did.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* dead) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long start = global_ns();
    while (!mbar_try_wait(bar, parity))
        if (*dead || global_ns() - start > kWaitLimitNs) {
            *dead = 1;
            return false;
        }
    return true;
}

// A CTA's stretch of the line, one segment (its part of a run) at a time.  A run
// takes `idle` places, then one for each tile.  The tensor cores cut what they add
// to an accumulator, eight times a tile: a segment ends after kMostTiles, and its
// sums are added with rounding to those of its run so far.  Equal weights over 2^20
// tokens in one stretch: 4.1e-3 too little in one sum, 3e-5 so; 1216 sequences on
// 2^20 tokens take 15.06 ms, 14.94 in one sum.
constexpr uint32_t kMostTiles = 256;
struct Segment {
    uint32_t u, end, idle, places;
    bool more = false;  // of the run that the last segment had, in this stretch
    __device__ Segment(uint32_t begin, uint32_t stop, uint32_t cost, uint32_t tiles)
        : u(begin), end(stop), idle(cost), places(cost + tiles) {
        skip();
    }
    __device__ void skip() { u = max(u, run() * places + idle); }
    __device__ bool done() const { return u >= end; }
    __device__ uint32_t run() const { return u / places; }
    __device__ uint32_t first() const { return u % places - idle; }
    __device__ uint32_t count() const { return min(min(end - u, places - u % places), kMostTiles); }
    __device__ void next() {
        const uint32_t last = run();
        u += count();
        skip();
        more = run() == last;
    }
};

template <bool kDual>
__global__ void __launch_bounds__(kPrefixThreads, 1) kv_prefix_kernel(const __grid_constant__ PrefixParams p) {
    using P = Plan<kDual>;
    constexpr int kStages = P::kStages;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t full[kStages], empty[kStages], q_full, s_full[2], p_full[2][2], p_read[2], o_full[2], cleaned[kStages], last;
    __shared__ uint32_t tmem_s;
    __shared__ int live_s[kLive][2];  // tokens of a tile's two pages that count
    __shared__ volatile int dead;
    unsigned char* const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t q_s = smem_addr(smem), ring_s = q_s + P::kQBytes;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
            mbar_init(&cleaned[i], 1);
        }
        mbar_init(&q_full, kSoftmaxThreads);
        mbar_init(&last, 1);
        for (int w = 0; w < 2; ++w) {
            mbar_init(&s_full[w], 1);
            mbar_init(&p_full[w][0], 128);
            mbar_init(&p_full[w][1], 128);
            mbar_init(&p_read[w], 1);
            mbar_init(&o_full[w], 1);
        }
        mbar_fence_init();
        dead = 0;
    }
    if (warp == kMmaWarp) tmem_alloc(&tmem_s, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;  // columns: S 0, S 1, O 0, O 1 (128 each); P over the front of S
    pdl_wait();
    pdl_trigger();
    const Split split(p.runs * (p.run_cost + p.tiles), gridDim.x);
    Segment seg(split.begin(blockIdx.x), split.begin(blockIdx.x + 1), p.run_cost, p.tiles);

    if (warp >= kSoftmaxThreads / 32) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kLoadWarp) {
            // ================ loader: K and V tiles in the order the products take them
            uint32_t it = 0;
            bool ok = true;
            uint32_t ids_first = 0;  // this lane's page of the 16 tiles from there: its id and tokens
            int32_t id32 = -1;
            int live32 = 0;
            const auto look_up = [&](uint32_t tile) {
                ids_first = tile;
                const uint32_t token = tile * kTileTokens + lane * kPageTokens;
                id32 = -1;
                live32 = 0;
                if (token >= p.tokens) return;
                id32 = p.v.table[token / kPageTokens];
                if (id32 < 0 || (unsigned long long)id32 >= p.v.pages) {
                    id32 = -1;  // no such page: its tokens are left out
                    raise_status(p.status, HSB_E_KV_PAGE, 0);
                } else {
                    live32 = (int)min(p.tokens - token, (uint32_t)kPageTokens);
                }
            };
            const auto load = [&](uint32_t tile, int head, int part, uint32_t number) {
                const uint32_t s = it % kStages;
                if (it >= (uint32_t)kStages)
                    ok = ok && __all_sync(0xffffffffu, wait_phase(&empty[s], ((it / kStages) - 1) & 1, &dead));
                if (!ok) return;
                const int from = (int)(tile - ids_first) * 2 + (lane & 1);
                const int32_t id = __shfl_sync(0xffffffffu, id32, from);
                const int live = __shfl_sync(0xffffffffu, live32, from);
                if (lane < 2 && part == 0) live_s[number % kLive][lane] = live;
                const unsigned have = __ballot_sync(0xffffffffu, lane < 2 && id >= 0);
                __syncwarp();
                if (lane == 0) {
                    if (have) mbar_arrive_expect_tx(&full[s], __popc(have) * 2 * kPanelBytes);
                    else mbar_arrive(&full[s]);
                }
                __syncwarp();
                if (lane < 2 && id >= 0) {
                    const unsigned char* src = p.v.data + ((size_t)id * p.v.heads + head) * PageFormat<HSB_KV_F16>::kBytes;
    #pragma unroll
                    for (int i = 0; i < 2; ++i)
                        bulk_copy_g2s(smem + P::kQBytes + s * kTileBytes + i * kTilePanel + lane * kPanelBytes,
                                      src + (part * 2 + i) * kPanelBytes, kPanelBytes, &full[s]);
                }
                __syncwarp();
                const uint32_t parity = (it++ / kStages) & 1;
                // rows of V behind the last token (or of a page that is not there) may hold NaN: zero them
                const int l0 = __shfl_sync(0xffffffffu, live, 0), l1 = __shfl_sync(0xffffffffu, live, 1);
                if (part && l0 + l1 < kTileTokens) {
                    ok = ok && __all_sync(0xffffffffu, wait_phase(&full[s], parity, &dead));
                    for (int i = lane; i < kTileTokens * 16; i += 32) {
                        const int r = i >> 4, c = i & 15;
                        if (r < kPageTokens ? r >= l0 : r - kPageTokens >= l1)
                            *reinterpret_cast<uint4*>(smem + P::kQBytes + s * kTileBytes + (c >> 3) * kTilePanel + r * 128 +
                                                      (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&cleaned[s]);
                }
            };
            uint32_t number = 0;  // tiles of earlier segments
            for (; ok && !seg.done(); seg.next()) {
                const int head = (int)(seg.run() / p.groups);
                const uint32_t first = seg.first(), n = seg.count();
                look_up(first);
                load(first, head, 0, number);
                for (uint32_t i = 0; ok && i < n; ++i) {
                    if (first + i + 1 >= ids_first + 16) look_up(first + i);
                    if (kDual && i + 1 < n) load(first + i + 1, head, 0, number + i + 1);
                    if (ok) load(first + i, head, 1, number + i);
                    if (!kDual && ok && i + 1 < n) load(first + i + 1, head, 0, number + i + 1);
                }
                number += n;
            }
            if (!ok) {  // copies in flight land before shared memory is released
                const uint32_t from = it > (uint32_t)kStages ? it - kStages : 0;
                for (uint32_t j = from; j < it; ++j) (void)mbar_wait(&full[j % kStages], (j / kStages) & 1);
            }
        } else if (warp == kMmaWarp) {
            // ================ products: one thread issues them all
            if (elect_one()) {
                uint32_t it = 0, number = 0, segment = 0, weights[2] = {0, 0}, cleanings = 0;  // (a bit a stage)
                bool ok = true;
                const uint64_t q_desc = operand(q_s, 16), k_desc = operand(ring_s, 16), v_desc = operand(ring_s, kTilePanel);
                const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && wait_phase(bar, parity, &dead); };
                const auto take = [&]() {  // the next stage, filled
                    const uint32_t s = it % kStages;
                    wait(&full[s], (it / kStages) & 1);
                    ++it;
                    return s;
                };
                // Of a run's first tiles; later ones lie over the weights of the tile before, which that
                // tile's product has then read (the order of two products of one thread is only given where
                // they have the accumulator in common).
                uint32_t weights_read[2] = {0, 0};
                const auto logits = [&](int w, uint32_t s, bool over) {
                    if (over) wait(&p_read[w], weights_read[w]++ & 1);
                    if (!ok) return;
                    tc_fence_after();
                    const uint64_t a = q_desc + (kDual ? 0 : w * (kTileBytes >> 4)), b = k_desc + s * (kTileBytes >> 4);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int at = ((k >> 2) * kTilePanel + (k & 3) * 32) >> 4;
                        tc_mma(tmem + w * 128, a + at, b + at, kShapeK, k > 0);
                    }
                    tc_commit(&s_full[w]);
                };
                const auto output = [&](int w, uint32_t s, bool add, bool more) {
                    const uint64_t b = v_desc + s * (kTileBytes >> 4);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // the first 64 tokens' while the others' weights are made
                        wait(&p_full[w][half], weights[w] & 1);
                        if (!ok) return;
                        tc_fence_after();
#pragma unroll
                        for (int k = half * 4; k < half * 4 + 4; ++k)
                            tc_mma_tmem(tmem + 256 + w * 128, tmem + w * 128 + k * 8, b + ((k * 16 * 128) >> 4), kShapeMN,
                                        add || k > 0);
                    }
                    ++weights[w];
                    if (more) tc_commit(&p_read[w]);
                };
                const auto take_v = [&](uint32_t tile_number) {
                    const uint32_t s = take();
                    if (live_s[tile_number % kLive][0] + live_s[tile_number % kLive][1] < kTileTokens) {
                        wait(&cleaned[s], cleanings >> s & 1);
                        cleanings ^= 1u << s;
                    }
                    return s;
                };
                const auto commit = [&](uint64_t* bar) {
                    if (ok) tc_commit(bar);
                };
                for (; ok && !seg.done(); seg.next(), ++segment) {
                    const uint32_t n = seg.count();
                    wait(&q_full, segment & 1);
                    tc_fence_after();
                    if constexpr (kDual) {
                        for (uint32_t i = 0; i < 2 && i < n; ++i) {
                            const uint32_t s = take();
                            logits(i, s, false);
                            commit(&empty[s]);
                        }
                        for (uint32_t i = 0; ok && i < n; ++i) {
                            const int w = i & 1;
                            const uint32_t s = take_v(number + i);
                            output(w, s, i >= 2, i + 2 < n);
                            commit(&empty[s]);
                            if (i + 2 < n) {
                                const uint32_t next = take();
                                logits(w, next, true);
                                commit(&empty[next]);
                            } else {
                                commit(&o_full[w]);
                            }
                        }
                        if (n == 1) commit(&o_full[1]);
                    } else {
                        uint32_t s = take();
                        logits(0, s, false);
                        logits(1, s, false);
                        commit(&empty[s]);
                        for (uint32_t i = 0; ok && i < n; ++i) {
                            const uint32_t v = take_v(number + i);
                            output(0, v, i > 0, i + 1 < n);
                            if (i + 1 < n) {
                                s = take();
                                logits(0, s, true);
                            } else {
                                commit(&o_full[0]);
                            }
                            output(1, v, i > 0, i + 1 < n);
                            commit(&empty[v]);
                            if (i + 1 < n) {
                                logits(1, s, true);
                                commit(&empty[s]);
                            } else {
                                commit(&o_full[1]);
                            }
                        }
                    }
                    number += n;
                }
                if (!ok) {  // products in flight end before tensor memory is freed
                    tc_commit(&last);
                    (void)mbar_wait(&last, 0);
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ================ softmax: warpgroup w, thread = row
        const int w = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + w * 128, o_at = tmem + lanes + 256 + w * 128;
        uint32_t logits_seen = 0, number = 0, segment = 0;
        bool ok = true;
        for (; ok && !seg.done(); seg.next(), ++segment) {
            const uint32_t run = seg.run(), n = seg.count();
            const int head = (int)(run / p.groups);
            const uint32_t mtile = (run % p.groups) * 2;
            // ---- Q into its operand layout (the products of the last segment are done: o_full)
            constexpr int kLoads = kDual ? 8 : 16;
            uint4 x4[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = kDual ? i * 256 + tid : i * 128 + row, r = at >> 4, c = at & 15;
                const uint32_t seq = (mtile + (kDual ? 0 : w)) * kTileSeqs + r / kGroup;
                x4[i] = make_uint4(0, 0, 0, 0);  // rows behind the batch
                if (seq < p.batch)
                    x4[i] = *reinterpret_cast<const uint4*>(
                        p.q + (((size_t)seq * p.v.heads + head) * kGroup + r % kGroup) * kDim + c * 8);
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = kDual ? i * 256 + tid : i * 128 + row, r = at >> 4, c = at & 15;
                *reinterpret_cast<uint4*>(smem + (kDual ? 0 : w * kTileBytes) + (c >> 3) * kTilePanel + r * 128 +
                                          (((c & 7) ^ (r & 7)) << 4)) = x4[i];
            }
            fence_async_shared();
            mbar_arrive(&q_full);
            // The largest logit that moved the reference, before its scale; whether any of the warp's is far; the sum.
            float most = -INFINITY, l = 0.0f;
            bool far = false;
            const auto reference = [&]() { return __fsub_rn(__fmul_rn(most, p.scale_log2), kUnit); };  // (rounded, never part of an FMA)
            const auto residual = [&]() { return fmaf(most, p.scale_log2, -reference()) - kUnit; };
            const uint32_t step = kDual ? 2 : 1, first = kDual ? w : 0;
            for (uint32_t i = first; ok && i < n; i += step) {
                ok = __all_sync(0xffffffffu, wait_phase(&s_full[w], logits_seen++ & 1, &dead));
                if (!ok) break;
                tc_fence_after();
                float x[kTileTokens];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_load32(s_at + c * 32, x + c * 32);
                tmem_wait_load();
                const int l0 = live_s[(number + i) % kLive][0], l1 = live_s[(number + i) % kLive][1];
                if (l0 < kPageTokens || l1 < kPageTokens) {
#pragma unroll
                    for (int j = 0; j < kTileTokens; ++j)
                        if (j < kPageTokens ? j >= l0 : j - kPageTokens >= l1) x[j] = -INFINITY;
                }
                float tops[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int j = 4; j < kTileTokens; j += 8) {
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4)
                        tops[i4] = j + 4 + i4 < kTileTokens ? max3(tops[i4], x[j + i4], x[j + 4 + i4])
                                                            : fmaxf(tops[i4], x[j + i4]);
                }
                const float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
                if (__any_sync(0xffffffffu, (top - most) * p.scale_log2 > kTop - kUnit)) {
                    const float to = fmaxf(most, top), before = reference();
                    const float rest = far ? residual() : 0.0f;
                    const bool none = most == -INFINITY;
                    most = to;
                    far = __any_sync(0xffffffffu, fabsf(reference()) > kFar && to != -INFINITY);
                    const float f = none ? 0.0f : exp2_ftz((before - reference()) + (rest - (far ? residual() : 0.0f)));
                    l *= f;
                    if (i != first) {  // (the first product overwrites O; later ones are complete: s_full)
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            float o[32];
                            tmem_load32(o_at + c * 32, o);
                            tmem_wait_load();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] *= f;
                            tmem_store32(o_at + c * 32, reinterpret_cast<const uint32_t*>(o));
                        }
                    }
                }
                float base = most == -INFINITY ? 0.0f : reference();
                if (far) {
                    const float from = most == -INFINITY ? 0.0f : most;
#pragma unroll
                    for (int j = 0; j < kTileTokens; ++j) x[j] -= from;
                    base = -kUnit;
                }
                const uint64_t scale2 = pair_of(p.scale_log2, p.scale_log2), minus2 = pair_of(-base, -base);
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t h[kTileTokens / 4];
#pragma unroll
                    for (int j = 0; j < kTileTokens / 2; j += 2) {
                        const int at = half * (kTileTokens / 2) + j;
                        const uint64_t y = fma2(pair_of(x[at], x[at + 1]), scale2, minus2);
                        float a, b;
                        if (!kDual && (j >> 1) % kByPolynomial == 0) {
                            exp2_pair(y, a, b);
                        } else {
                            split_of(y, a, b);
                            a = exp2_ftz(a);
                            b = exp2_ftz(b);
                        }
                        sum2[(j >> 1) & 1] = add2(sum2[(j >> 1) & 1], pair_of(a, b));
                        const __half2 pair = __floats2half2_rn(a, b);
                        h[j >> 1] = *reinterpret_cast<const uint32_t*>(&pair);
                    }
                    tmem_store32(s_at + half * 32, h);
                    tmem_wait_store();
                    tc_fence_before();
                    mbar_arrive(&p_full[w][half]);
                }
                float la, lb;
                split_of(add2(sum2[0], sum2[1]), la, lb);
                l += la + lb;
            }
            // ---- the segment's partial
            if (ok) ok = __all_sync(0xffffffffu, wait_phase(&o_full[w], segment & 1, &dead));
            if (!ok) break;
            tc_fence_after();
            float* out = p.part + ((size_t)(blockIdx.x + run) * 2 + w) * kRowsFloats;
            // (rows behind the batch are not read)
            const bool wanted = (mtile + (kDual ? 0 : w)) * kTileSeqs + row / kGroup < p.batch;
            float2* const ml = reinterpret_cast<float2*>(out + kTileRows * kDim) + row;
            float4* const quads = reinterpret_cast<float4*>(out) + row;
            if (!seg.more) {
                if (wanted) *ml = make_float2(reference(), l);
                if (n > first) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        float o[32];
                        tmem_load32(o_at + c * 32, o);
                        tmem_wait_load();
                        if (!wanted) continue;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            quads[(c * 8 + j) * kTileRows] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                    }
                } else if (wanted) {  // no tile for this warpgroup
                    for (int c = 0; c < 32; ++c) quads[c * kTileRows] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            } else if (n > first) {  // added to the run's so far, which this thread wrote
                float by = 0.0f, held = 0.0f;
                if (wanted) {
                    const float2 was = *ml;
                    const float now = reference(), to = fmaxf(was.x, now);
                    held = was.x == -INFINITY ? 0.0f : exp2_ftz(was.x - to);
                    by = now == -INFINITY ? 0.0f : exp2_ftz(now - to);
                    *ml = make_float2(to, fmaf(held, was.y, by * l));
                }
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    tmem_load32(o_at + c * 32, o);
                    tmem_wait_load();
                    if (!wanted) continue;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float4& sum = quads[(c * 8 + j) * kTileRows];
                        const float4 was = sum;
                        sum = make_float4(fmaf(held, was.x, by * o[4 * j]), fmaf(held, was.y, by * o[4 * j + 1]),
                                          fmaf(held, was.z, by * o[4 * j + 2]), fmaf(held, was.w, by * o[4 * j + 3]));
                    }
                }
            }
            tc_fence_before();
            number += n;
        }
    }
    __syncthreads();
    if (tid == 0 && dead) raise_status(p.status, HSB_E_TIMEOUT, blockIdx.x);
    tc_fence_after();
    if (warp == kMmaWarp) {
        tmem_free(tmem, 512);
    }
}

// ---------------------------------------------------------------- combine
struct SharedCombine {
    // the prefix: partials [stretch + run][2][kRowsFloats]
    const float* prefix;
    Split split;  // of its line
    uint32_t groups, run_places, prefix_cost;
    int dual;
    // the sequences' own tokens (kvattention.cuh)
    const float* part;
    const float* whole;
    const uint32_t* place;
    uint32_t own_grid;  // of the kernel that left them
    const int32_t* lengths;
    unsigned long long table_width;
    uint32_t batch;
    int heads;
    uint16_t* out;
};

// CTA = (two sequences' eight rows, KV head, 128 / kSplit channels), thread =
// (row, kQuads quads of channels), every kSplit-th partial.  The (max, sum) pairs
// of all partials meet in shared memory and become weights there, while the first
// partials' outputs, whose loads wait for nothing, are on their way.  Bound by
// latency where rows are few and by the threads' own work where they are many, so
// with fewer rows there are more threads for them (8, 64, 128 and 256 sequences, 8
// heads, us a call): kSplit 4 14.5, 61.2, 66.8, 114; kSplit 2 16.1, 58.1, 60.1, 98.7;
// one part and four quads a thread 18.2, 65.0, 61.6, 94.4.
constexpr int kMaxParts = 3 * kAttnMaxCtas;  // two a CTA of the prefix, one a CTA of the own tokens
template <int kSplit, int kQuads, int kFirst>  // kFirst prefix partials are loaded ahead
__global__ void __launch_bounds__(256 / kQuads) kv_shared_combine_kernel(const __grid_constant__ SharedCombine p) {
    static_assert(kSplit == 1 || kQuads == 1, "one or the other");
    constexpr int kThreads = 256 / kQuads, kLines = kThreads / 8;
    __shared__ float2 ml_s[kMaxParts][8];            // (max, sum), then (weight, sum)
    __shared__ float4 acc_s[kSplit == 1 ? 1 : kThreads];
    __shared__ float sum_s[kSplit == 1 ? 1 : kThreads];
    const int tid = threadIdx.x, head = blockIdx.y, r8 = tid & 7, line = tid >> 3;
    const uint32_t seq = min(blockIdx.x * 2 + r8 / kGroup, p.batch - 1);
    const int h = r8 % kGroup;
    // the row's partials: `n` of the prefix, `m` of its own tokens
    const uint32_t mtile = blockIdx.x / (kTileSeqs / 2), row = (seq % kTileSeqs) * kGroup + h;
    const uint32_t run = head * p.groups + mtile / 2, own_run = seq * p.heads + head;
    const uint32_t p0 = p.split.of(run * p.run_places + p.prefix_cost), p1 = p.split.of((run + 1) * p.run_places - 1);
    const uint32_t n = (p1 - p0 + 1) * (p.dual ? 2 : 1);
    const float* base = p.prefix + ((size_t)(p0 + run) * 2 + (p.dual ? 0 : mtile & 1)) * kRowsFloats;
    const uint32_t step = (p.dual ? 1 : 2) * kRowsFloats;
    const int quad = kSplit == 1 ? line : blockIdx.z * (32 / kSplit) + line % (32 / kSplit);
    const uint32_t part = kSplit == 1 ? 0 : line / (32 / kSplit);
    const float4* at = reinterpret_cast<const float4*>(base) + quad * kTileRows + row;
    constexpr int kNext = kLines * kTileRows;  // float4s to the thread's second quad
    pdl_wait();
    pdl_trigger();
    const uint32_t tokens = tokens_in(p.lengths, p.table_width, seq), place = p.place[own_run];
    float4 v[kFirst][kQuads];
#pragma unroll
    for (int k = 0; k < kFirst; ++k) {
        const uint32_t i = part + k * kSplit;
#pragma unroll
        for (int q = 0; q < kQuads; ++q)
            if (i < n) v[k][q] = __ldcg(at + (size_t)i * (step / 4) + q * kNext);
    }
    for (uint32_t i = line; i < n; i += kLines)
        ml_s[i][r8] = __ldcg(reinterpret_cast<const float2*>(base + (size_t)i * step + kTileRows * kDim) + row);
    const uint32_t m = tokens == 0 ? 0 : run_partials(place, p.own_grid);
    const float* own = place == 0 ? p.whole + (size_t)own_run * kPartFloats : p.part + (size_t)(place >> 16) * 2 * kPartFloats;
    const auto own_at = [&](uint32_t i) { return own + (place == 0 ? 0 : ((size_t)i * 2 + (i == 0)) * kPartFloats); };
    for (uint32_t i = line; i < m; i += kLines) ml_s[n + i][r8] = __ldcg(reinterpret_cast<const float2*>(own_at(i)) + h);
    __syncthreads();
    const uint32_t total = n + m;
    float top = -INFINITY;
    for (uint32_t i = line & 3; i < total; i += 4) top = fmaxf(top, ml_s[i][r8].x);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    __syncthreads();
    // (all -infinity: no token, sums 0; a NaN sum comes through)
    for (uint32_t i = line; i < total; i += kLines)
        ml_s[i][r8].x = top == -INFINITY ? 1.0f : exp2_ftz(ml_s[i][r8].x - top);
    __syncthreads();
    float4 acc[kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; ++q) acc[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
    const auto add = [&](float f, int q, float4 x) {
        acc[q] = make_float4(fmaf(f, x.x, acc[q].x), fmaf(f, x.y, acc[q].y), fmaf(f, x.z, acc[q].z), fmaf(f, x.w, acc[q].w));
    };
    const auto weight = [&](uint32_t i) {
        const float2 fl = ml_s[i][r8];
        sum = fmaf(fl.x, fl.y, sum);
        return fl.x;
    };
#pragma unroll
    for (int k = 0; k < kFirst; ++k) {
        const uint32_t i = part + k * kSplit;
        if (i < n) {
            const float f = weight(i);
#pragma unroll
            for (int q = 0; q < kQuads; ++q) add(f, q, v[k][q]);
        }
    }
#pragma unroll 4
    for (uint32_t i = part + kFirst * kSplit; i < n; i += kSplit) {
        const float f = weight(i);
#pragma unroll
        for (int q = 0; q < kQuads; ++q) add(f, q, __ldcg(at + (size_t)i * (step / 4) + q * kNext));
    }
    for (uint32_t i = part; i < m; i += kSplit) {
        const float f = weight(n + i);
        const float4* from = reinterpret_cast<const float4*>(own_at(i) + 2 * kGroup + h * kDim) + quad;
#pragma unroll
        for (int q = 0; q < kQuads; ++q) add(f, q, __ldcg(from + q * kLines));
    }
    if constexpr (kSplit > 1) {
        acc_s[tid] = acc[0];
        sum_s[tid] = sum;
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int k = 1; k < kSplit; ++k) {
            const float4 x = acc_s[tid + k * (kThreads / kSplit)];
            acc[0] = make_float4(acc[0].x + x.x, acc[0].y + x.y, acc[0].z + x.z, acc[0].w + x.w);
            sum += sum_s[tid + k * (kThreads / kSplit)];
        }
    }
    if (blockIdx.x * 2 + r8 / kGroup >= p.batch) return;
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum);
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        const __half2 a = __floats2half2_rn(acc[q].x * inv, acc[q].y * inv);
        const __half2 b = __floats2half2_rn(acc[q].z * inv, acc[q].w * inv);
        reinterpret_cast<uint2*>(p.out + ((size_t)own_run * kGroup + h) * kDim)[quad + q * kLines] =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

struct Geometry {
    uint32_t tiles, groups, runs;
    bool dual;
    size_t slots;  // of prefix partials
    size_t place, part, whole, total;
};
Geometry geometry(size_t batch, int heads, size_t prefix_tokens) {
    Geometry g{};
    g.tiles = (uint32_t)((prefix_tokens + kTileTokens - 1) / kTileTokens);
    const size_t mtiles = (batch + kTileSeqs - 1) / kTileSeqs;
    g.dual = mtiles == 1;
    g.groups = (uint32_t)((mtiles + 1) / 2);
    g.runs = (uint32_t)heads * g.groups;
    g.slots = std::min<size_t>((size_t)g.runs * g.tiles, kAttnMaxCtas) + g.runs;
    g.place = align256(g.slots * 2 * kRowsFloats * 4);
    g.part = g.place + align256(batch * heads * 4);
    g.whole = g.part + align256((size_t)kAttnMaxCtas * 2 * kPartFloats * 4);
    g.total = g.whole + align256(batch * heads * kPartFloats * 4);
    return g;
}

template <bool kDual>
cudaError_t launch_prefix(const PrefixParams& p, unsigned grid, cudaStream_t stream) {
    static thread_local int configured = -1;
    const int device = device_info().ordinal;
    if (configured != device) {
        cudaFuncAttributes attr{};
        cudaError_t e = cudaFuncGetAttributes(&attr, kv_prefix_kernel<kDual>);
        if (e != cudaSuccess) return e;
        // the warpgroups' shares are drawn from what the block was launched with: more would wait for ever
        if (attr.numRegs * kPrefixThreads < 128 * (2 * kSoftmaxRegs + kOtherRegs)) return cudaErrorLaunchOutOfResources;
        e = cudaFuncSetAttribute(kv_prefix_kernel<kDual>, cudaFuncAttributeMaxDynamicSharedMemorySize, Plan<kDual>::kSmem);
        if (e != cudaSuccess) return e;
        configured = device;
    }
    return launch_dependent(kv_prefix_kernel<kDual>, dim3(grid), dim3(kPrefixThreads), Plan<kDual>::kSmem, stream, false, p);
}

template <int kSplit, int kQuads, int kFirst>
cudaError_t launch_combine(const SharedCombine& c, dim3 rows, cudaStream_t stream) {
    return launch_dependent(kv_shared_combine_kernel<kSplit, kQuads, kFirst>, dim3(rows.x, rows.y, kSplit), dim3(256 / kQuads), 0,
                            stream, false, c);
}

}  // namespace
}  // namespace hsb

using namespace hsb;

extern "C" {

size_t hsb_kv_attention_shared_workspace_bytes(size_t batch, int kv_heads, size_t prefix_tokens) {
    if (!batch || batch > kMaxBatch || kv_heads < 1 || kv_heads > HSB_KV_HEADS || prefix_tokens > kMaxPrefix) return 0;
    return geometry(batch, kv_heads, prefix_tokens).total;
}

int hsb_kv_attention_shared(const hsb_kv_pages* prefix, const int32_t* d_prefix_table, size_t prefix_tokens,
                            const hsb_kv_pages* pages, const int32_t* d_table, size_t table_width,
                            const int32_t* d_lengths, size_t batch, const uint16_t* d_q, uint16_t* d_out,
                            void* d_workspace, size_t workspace_bytes, hsb_device_status* d_status, void* stream) {
    if (!kv_pages_valid(prefix) || !kv_pages_valid(pages)) return record_error(HSB_E_KV_SHAPE, "paged KV pool arguments");
    if (prefix->format != HSB_KV_F16 || prefix->kv_heads != pages->kv_heads)
        return record_error(HSB_E_KV_SHAPE, "a shared prefix is an F16 pool of the same KV heads");
    if (!d_prefix_table || !prefix_tokens || prefix_tokens > kMaxPrefix || !d_table || !table_width ||
        table_width > kMaxTableEntries || !d_lengths || !batch || batch > kMaxBatch ||
        batch * table_width > kMaxTableEntries || !d_q || !d_out)
        return record_error(HSB_E_KV_SHAPE, "paged KV attention shape");
    if (!aligned_to(16, d_q, d_out, static_cast<unsigned char*>(d_workspace)) ||
        !aligned_to(4, d_prefix_table, d_table, d_lengths) || !aligned_to(8, d_status))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention buffers are misaligned");
    const size_t bytes = batch * pages->kv_heads * kGroup * kDim * sizeof(uint16_t);
    if (!apart(d_q, bytes, d_out, bytes))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention output must not alias the query");
    const Geometry g = geometry(batch, pages->kv_heads, prefix_tokens);
    if ((unsigned long long)g.runs * (g.tiles + 4) > 0x7fffffffull)
        return record_error(HSB_E_KV_SHAPE, "paged KV attention shape");
    if (!d_workspace || workspace_bytes < g.total)
        return record_error(HSB_E_WORKSPACE, "paged KV attention workspace missing or too small");
    if (!apart(d_workspace, g.total, d_q, bytes) || !apart(d_workspace, g.total, d_out, bytes))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention workspace must not alias the query or the output");
    unsigned char* ws = static_cast<unsigned char*>(d_workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);

    PrefixParams p{};
    p.v = paged_view(*prefix, d_prefix_table, (prefix_tokens + kPageTokens - 1) / kPageTokens, 0);
    p.tokens = (uint32_t)prefix_tokens;
    p.tiles = g.tiles;
    p.q = d_q;
    p.batch = (uint32_t)batch;
    p.groups = g.groups;
    p.runs = g.runs;
    p.part = reinterpret_cast<float*>(ws);
    p.status = d_status;
    p.scale_log2 = kScaleLog2;
    // a tile for each warpgroup at least: more CTAs would only leave more partials
    const unsigned units = g.runs * g.tiles, least = g.dual ? (units + 1) / 2 : units;
    const unsigned grid = std::min<unsigned>({least, (unsigned)device_info().sms, kAttnMaxCtas});
    // idle places pay where a CTA has several times as many tiles (64 x 32768: 60.4 us without, 58.4 with;
    // 256 x 16461: 97.1 and 94.4)
    p.run_cost = units >= 6 * grid ? 2 : 0;
    cudaError_t e = g.dual ? launch_prefix<true>(p, grid, s) : launch_prefix<false>(p, grid, s);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV attention launch");

    PagedAttention a{};
    a.v = paged_view(*pages, d_table, table_width, table_width);
    a.lengths = d_lengths;
    a.batch = batch;
    a.q = d_q;
    a.place = reinterpret_cast<uint32_t*>(ws + g.place);
    a.part = reinterpret_cast<float*>(ws + g.part);
    a.whole = reinterpret_cast<float*>(ws + g.whole);
    a.status = d_status;
    a.scale_log2 = kScaleLog2;
    a.by_run = paged_by_run(batch, table_width, pages->kv_heads);
    const unsigned own = paged_attention_grid(batch, table_width, pages->kv_heads);
    e = launch_paged_partials(pages->format, a, own, s);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV attention launch");

    SharedCombine c{};
    c.prefix = p.part;
    c.split = Split(g.runs * (p.run_cost + g.tiles), grid);
    c.groups = g.groups;
    c.run_places = p.run_cost + g.tiles;
    c.prefix_cost = p.run_cost;
    c.dual = g.dual;
    c.part = a.part;
    c.whole = a.whole;
    c.place = a.place;
    c.own_grid = own;
    c.lengths = d_lengths;
    c.table_width = table_width;
    c.batch = (uint32_t)batch;
    c.heads = pages->kv_heads;
    c.out = d_out;
    const dim3 rows((unsigned)((batch + 1) / 2), pages->kv_heads);
    const unsigned ctas = rows.x * rows.y;
    e = ctas < 128 ? launch_combine<4, 1, 10>(c, rows, s)
        : ctas < 768 ? launch_combine<2, 1, 6>(c, rows, s)
                       : launch_combine<1, 4, 4>(c, rows, s);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV attention launch");
    record_error(HSB_OK, "");
    return HSB_OK;
}

}  // extern "C"
