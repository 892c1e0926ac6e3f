// kvattention.cu -- decode attention of a batch over the paged KV cache:
//   out[b][h] = softmax(q[b][h] . K_b^T / sqrt(128)) V_b,  K = codes x scales,
// one token per sequence, ragged lengths, four query heads to a KV head.
//
// Four rows of queries against every cached row is far too little arithmetic
// for the tensor cores' own pipeline to matter (4 flops a byte in F16, 8 in 8
// bits): the kernel is bound by the bytes of the pages, and is built to keep
// them coming.  K and V of a page arrive whole by bulk copies into a warp's own
// ring of shared memory; the warp turns the codes into F16 fragments in
// registers (both formats convert exactly) and runs both products with
// mma.sync.m16n8k16, tokens and channels in the wide dimension:
//
//   logits  S^T[token][col] = K[token][ch] . Q^T[ch][col]
//   output  O^T[ch][col]    = V^T[ch][token] . P^T[token][col]
//
// Of the eight columns, col h carries the F16 rounding of head h's F32 value,
// col h + 4 the remainder, so products keep ~22 bits of q and of the weights
// at no cost.  Which channel sits at which k (or row) of the MMA is free, as
// long as both operands agree: each lane owns whole 16-byte chunks, so the
// fragments are the loaded words themselves, with no ldmatrix.  The K scale
// multiplies a token's logits, the V scale its weight, both in F32; the largest
// weights are brought into F16's range by a power of two before their split into
// halves, so a weight is off by 2^-22 of itself, or 2^-32 of a head's largest.
// The running maximum is only moved when a logit passes it by 8 (in log2): until
// then no reduction across the warp and no rescaling is needed.
//
// Work is split evenly without regard to lengths: the (sequence, head, unit)
// triples in that order are one line, of which every CTA takes an equal stretch
// and each of its warps an equal part, with a ring of its own that it fills
// itself.  Warps never wait for one another inside the line, so what a run costs
// at its ends (its query, its last sums) hides behind the others' work.  A
// (sequence, head) run inside one warp's part is finished there, one that crosses
// warps is folded in shared memory at the end, and one that crosses CTAs leaves
// F32 partials that kv_combine_kernel folds in order.
//
// Measured (B200, 8 KV heads, one call in a captured graph): 64 sequences of up
// to 8192 int8 or e4m3 tokens 99 us, 5.6 TB/s, of up to 32768 360 us, 6.1; 64 x
// 32768 F16, one head, 89.3 us, 6.0 TB/s (a copy reaches 6.5); one sequence of
// 32768 int8 tokens 20.5 us, of which 10.6 are its bytes, 3.4 kv_combine_kernel
// (4 to 5 of the longer calls) and the rest the launch and the look-ups before
// the first byte.  Under the profiler (e4m3, 16 x 16384) the kernel reads 554 MB,
// the pages' bytes once, at 5.8 TB/s; 910 instructions a warp and page leave the
// issue slots two thirds idle.
#include <algorithm>
#include <cmath>

#include "kvattention.cuh"

namespace hsb {
namespace {

// Weights enter the second product times a unit.  F16: 2^7, and p is at most
// 2^kSlack, so their halves reach 2^15 at most.  8 bits: p x V scale, the unit
// a power of two that brings the largest such weight so far to 2^7 and moves when
// one would pass 2^15.  (Taken from the scales alone, it would follow rows that
// the softmax ignores: one of 6e4 among 1e-3 cost the others 14 of their 22 bits.)
constexpr float kWeightUnit = 128.0f, kTopWeight = 32768.0f;
constexpr float kSlack = 8.0f;
constexpr float kFirstUnit = 0x1p100f, kLeastWeight = 0x1p-93f;  // before any weight; kWeightUnit / kFirstUnit

// Each warp's ring holds K and V of its units in turn (K 0, V 0, K 1, ...): a
// slot is free again as soon as its product is done.  A unit is a page in 8
// bits; in F16, twice the bytes a token and no codes to convert, half a page.
// Eight warps of three slots fill the shared memory and leave a thread its 241
// registers; twelve or ten warps of two slots were slower throughout.
// The scales of both come with V (they follow it in the page: one copy), as
// the logits are first needed where the weights are made.
template <int F>
struct Ring {
    using Fmt = PageFormat<F>;
    static constexpr int kWarps = 8;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kSlots = 3;
    static constexpr int kTokens = F == HSB_KV_F16 ? kPageTokens / 2 : kPageTokens;  // of a unit
    static constexpr int kPerPage = kPageTokens / kTokens;
    static constexpr int kPanel = kTokens * 128;
    static constexpr int kPart = Fmt::kPanels * kPanel;  // K or V of a unit; the scales lie behind V
    static constexpr int kSlot = kPart + (Fmt::kScaled ? 2 * kTokens * 4 : 0);
    static constexpr int kSmem = 128 + kWarps * (kSlots * kSlot + kPartFloats * 4);
    static_assert(kSlots * kSlot >= kPartFloats * 4, "a piece fits in a warp's ring");
    // What a run costs besides its units (its query, its first rescaling, its results), in units.
    static constexpr uint32_t kRunCost = F == HSB_KV_F16 ? 2 : 1;
    __host__ __device__ static constexpr uint32_t units(uint32_t tokens) { return (tokens + kTokens - 1) / kTokens; }
    // Places of the line that a head of a sequence takes: idle ones for that cost, then its units.
    __host__ __device__ static constexpr uint32_t places(uint32_t tokens) {
        return tokens ? kRunCost + units(tokens) : 0;
    }
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8x8 transpose of F16 pairs across the warp: the logits' accumulator layout
// (row = token, columns 2t, 2t + 1) into a B fragment (column, tokens 2t, 2t + 1).
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ void prefetch_l2(const void* at) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
// The maximum over the lanes of this one's columns (t, t ^ 2), which hold all rows of a unit: two reductions by
// the warp, 0.2 us less in a run's first unit than four exchanges.
__device__ __forceinline__ float rows_max(float v, bool odd) {
    float a, b;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(a) : "f"(odd ? -INFINITY : v));
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(b) : "f"(odd ? v : -INFINITY));
    return odd ? b : a;
}
// 1 / x of a normal power of two below 2^127 (a run of 77 tokens 5.0 us, with divisions 5.5).
__device__ __forceinline__ float inverse_of_power(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
__device__ __forceinline__ float lds32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
// (a, b) as the F16 pair of this lane's columns: their roundings, or what these leave.
__device__ __forceinline__ uint32_t split_pair(float a, float b, bool low) {
    const __half2 hi = __floats2half2_rn(a, b);
    const float2 f = __half22float2(hi);
    const __half2 lo = __floats2half2_rn(a - f.x, b - f.y);
    return low ? *reinterpret_cast<const uint32_t*>(&lo) : *reinterpret_cast<const uint32_t*>(&hi);
}
__device__ __forceinline__ float4 load_q4(const float* q) { return *reinterpret_cast<const float4*>(q); }
__device__ __forceinline__ float4 load_q4(const uint16_t* q) {
    const uint2 w = *reinterpret_cast<const uint2*>(q);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

// Tokens of a sequence; a length behind the table's end counts as none.
__device__ __forceinline__ uint32_t tokens_of(const PagedAttention& p, uint32_t b, bool report) {
    const int32_t n = p.lengths[b];
    if (n < 0 || (unsigned long long)n > p.v.width * kPageTokens) {
        if (report) raise_status(p.status, HSB_E_KV_POSITION, (int)b);
        return 0;
    }
    return n;
}
// A position in the line, at a unit, up to `end`.
template <typename R>
struct Walker {
    uint32_t u, end;
    uint32_t seq, tokens, units;  // of the current run
    uint32_t run;                 // the place of its first unit
    int head;
    __device__ bool done() const { return u >= end; }
    __device__ uint32_t run_end() const { return run + units; }
    // Steps over one unit; true when that enters another run.
    __device__ bool step(const PagedAttention& p) {
        if (++u < run_end()) return false;
        run += units + R::kRunCost;
        u = run;
        if (++head == p.v.heads && !done()) {
            head = 0;
            do {
                ++seq;
                tokens = tokens_of(p, seq, false);
                units = R::units(tokens);
            } while (units == 0);
        }
        return true;
    }
};

// Finds this warp's part of CTA blockIdx.x's stretch.  Each warp scans the
// lengths by itself (a lane has every 1/32 of the batch): no barrier is needed.
template <typename R>
__device__ Walker<R> find_part(const PagedAttention& p, uint32_t* total_units, uint32_t* stretch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (p.by_run) {
        Walker<R> k{};
        k.seq = blockIdx.x / p.v.heads;
        k.head = (int)(blockIdx.x % p.v.heads);
        k.tokens = tokens_of(p, k.seq, true);
        k.units = R::units(k.tokens);
        const Split parts(k.units, R::kWarps);
        k.u = parts.begin(warp);
        k.end = parts.begin(warp + 1);
        stretch[0] = 0;
        stretch[1] = *total_units = k.units;
        return k;
    }
    const bool scribe = blockIdx.x == 0 && warp == 0;
    const uint32_t batch = (uint32_t)p.batch, per = (batch + 31) / 32;
    const uint32_t b0 = min(batch, lane * per), b1 = min(batch, b0 + per);
    uint32_t mine = 0;
#pragma unroll 4
    for (uint32_t b = b0; b < b1; ++b) mine += R::places(tokens_of(p, b, scribe));
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, upto, 31), before = upto - mine;  // places of one head
    const Split ctas(total * p.v.heads, gridDim.x);
    const uint32_t u0 = ctas.begin(blockIdx.x), u1 = ctas.begin(blockIdx.x + 1);
    const Split parts(u1 - u0, R::kWarps);
    *total_units = total * p.v.heads;
    stretch[0] = u0;
    stretch[1] = u1;
    Walker<R> k{};
    k.u = u0 + parts.begin(warp);
    k.end = u0 + parts.begin(warp + 1);
    if (k.done()) return k;
    const int shift = 31 - __clz(p.v.heads);  // heads is a power of two
    const uint32_t rank = k.u >> shift;       // among the places of one head
    const bool here = rank >= before && rank < upto;
    uint32_t b = b0, n = 0, c = before;
    if (here) {
        while (true) {
            n = tokens_of(p, b, false);
            if (rank < c + R::places(n)) break;
            c += R::places(n);
            ++b;
        }
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    k.seq = __shfl_sync(0xffffffffu, b, src);
    k.tokens = __shfl_sync(0xffffffffu, n, src);
    k.units = R::units(k.tokens);
    const uint32_t base = __shfl_sync(0xffffffffu, c, src) << shift;
    k.head = (int)((k.u - base) / R::places(k.tokens));
    k.run = base + k.head * R::places(k.tokens) + R::kRunCost;
    k.u = max(k.u, k.run);
    return k;
}

// A run's cut piece in a warp's part: [0] the run began before the part, [1] it goes on behind it.
struct Piece {
    uint32_t id, first, last;  // sequence * heads + head; its units [first, last)
    int there, ends;           // ends: within the part
};

template <int F, typename Q, bool kFinal>
__global__ void __launch_bounds__(Ring<F>::kThreads, 1) kv_attention_kernel(const __grid_constant__ PagedAttention p) {
    using Fmt = PageFormat<F>;
    using R = Ring<F>;
    constexpr int kWarps = R::kWarps, kThreads = R::kThreads, kSlots = R::kSlots, kTiles = R::kTokens / 16;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t full_s[kWarps][kSlots];
    __shared__ int bad_s[kWarps][kSlots];
    __shared__ Piece pieces[kWarps][2];
    unsigned char* const ring0 = smem_raw + ((128u - (smem_addr(smem_raw) & 127u)) & 127u);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* const heads_s = reinterpret_cast<float*>(ring0 + kWarps * kSlots * R::kSlot);  // pieces [0]
    unsigned char* const ring = ring0 + warp * kSlots * R::kSlot;
    uint64_t* const full = full_s[warp];
    int* const bad = bad_s[warp];
    if (lane == 0) {
        for (int s = 0; s < kSlots; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
        pieces[warp][0].there = pieces[warp][1].there = 0;
    }
    // Partial mode follows kv_prefix_kernel, which lets this grid start only once everything
    // before itself is complete, and whose results are not read here: only the end waits, so
    // that what follows finds both.
    pdl_trigger();
    if (kFinal) {
        // lengths and tables into L2 before the wait (hints: what the preceding grid writes, it writes there too)
        const size_t lines = (p.batch * p.v.width + 31) / 32, line = (size_t)tid * gridDim.x + blockIdx.x;
        if (line < lines) prefetch_l2(p.v.table + line * 32);
        if (line * 32 < p.batch) prefetch_l2(p.lengths + line * 32);
        pdl_wait();
    }
    uint32_t units, stretch[2];
    Walker<R> k = find_part<R>(p, &units, stretch);
    __syncwarp();  // the barriers are ready
    if (kFinal && p.by_run) {  // empty sequences: zeros
        if (stretch[1] == 0)
            for (int i = tid; i < kGroup * kDim; i += kThreads) p.out[(size_t)blockIdx.x * kGroup * kDim + i] = 0.0f;
    } else if (kFinal) {
        for (uint32_t b = blockIdx.x; b < p.batch; b += gridDim.x)
            if (tokens_of(p, b, false) == 0)
                for (int i = tid; i < p.v.heads * kGroup * kDim; i += kThreads)
                    p.out[(size_t)b * p.v.heads * kGroup * kDim + i] = 0.0f;
    }
    if (kFinal && tid == 0 && !p.by_run) {
        RunInfo info{};
        info.run = -1;
        p.info[blockIdx.x] = info;  // (a run that goes on writes its own behind the block's barrier)
    }
    if (stretch[0] >= stretch[1]) {
        if (!kFinal) pdl_wait();
        return;
    }

    const int g = lane >> 2, t = lane & 3;
    // this lane's share of a run's query head g & 3: for step ks the channels of its K words
    float4 x4[8];
    const auto load_query = [&]() {
        const Q* q = static_cast<const Q*>(p.q) + ((size_t)(k.seq * p.v.heads + k.head) * kGroup + (g & 3)) * kDim;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
            x4[ks] = load_q4(q + (Fmt::kScaled ? t * 32 + ks * 4 : (ks >> 2) * 64 + t * 16 + (ks & 3) * 4));
    };
    // ---- feeding: K (even) or V (odd) of unit feed.u into slot fed % kSlots
    Walker<R> feed = k;
    uint32_t fed = 0, ids_first = 0;
    int32_t ids = 0;  // table entries of 32 pages from ids_first
    int32_t id = 0;
    bool fresh = true;
    const auto feed_one = [&]() {
        const int s = fed % kSlots, part = fed & 1;
        if (part == 0) {
            const uint32_t page = (feed.u - feed.run) / R::kPerPage;
            if (fresh || page >= ids_first + 32) {
                ids_first = page;
                ids = (page + lane) * R::kPerPage < feed.units ? p.v.table[feed.seq * p.v.pitch + page + lane] : 0;
            }
            id = __shfl_sync(0xffffffffu, ids, (int)(page - ids_first));
        }
        if (elect_one()) {
            if (id >= 0 && (unsigned long long)id < p.v.pages) {
                const int half = (int)((feed.u - feed.run) % R::kPerPage);
                const unsigned char* src = p.v.data + ((size_t)id * p.v.heads + feed.head) * Fmt::kBytes;
                unsigned char* dst = ring + s * R::kSlot;
                bad[s] = 0;
                if constexpr (Fmt::kScaled) {
                    const uint32_t bytes = part ? R::kSlot : R::kPart;
                    mbar_arrive_expect_tx(&full[s], bytes);
                    bulk_copy_g2s(dst, src + part * R::kPart, bytes, &full[s]);
                } else {
                    mbar_arrive_expect_tx(&full[s], R::kPart);
#pragma unroll
                    for (int i = 0; i < Fmt::kPanels; ++i)
                        bulk_copy_g2s(dst + i * R::kPanel, src + (part * Fmt::kPanels + i) * kPanelBytes + half * R::kPanel,
                                      R::kPanel, &full[s]);
                }
            } else {  // no such page: its tokens are left out
                if (part == 0) raise_status(p.status, HSB_E_KV_PAGE, (int)feed.seq);
                bad[s] = 1;
                mbar_arrive(&full[s]);
            }
        }
        if (part) fresh = feed.step(p);
        ++fed;
    };
    if (!feed.done()) feed_one();
    if (!k.done()) load_query();  // on its way while the rest of the ring is fed
#pragma unroll 1
    for (int i = 1; i < kSlots; ++i)
        if (!feed.done()) feed_one();

    const bool low = t >= 2;     // this lane's accumulator columns are the remainders' (and g >= 4 in B fragments)
    const int h0 = 2 * (t & 1);  // they are heads h0 and h0 + 1 of the group
    // Of a unit's 8-token rows i (tokens 8 i + g), lanes t < 2 do the softmax of the first
    // kTiles, lanes t >= 2 of the others; both have the same heads.
    const int token0 = (low ? kTiles * 8 : 0) + g;
    uint32_t it = 0;  // K and V parts read
    bool alive = true;
    while (alive && !k.done()) {
        // ================ one run, as far as it lies in this part
        const uint32_t begin = k.u, run_begin = k.run, run_end = k.run_end(), tokens = k.tokens;
        const uint32_t stop = min(run_end, k.end), run = k.seq * p.v.heads + k.head;
        float M[2] = {-INFINITY, -INFINITY}, L[2] = {0.0f, 0.0f};
        constexpr float kUnit0 = Fmt::kScaled ? kFirstUnit : kWeightUnit;
        float unit[2] = {kUnit0, kUnit0};
        float o[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        // Q^T fragments: column g = head g & 3, its rounding or remainder (g >= 4)
        uint32_t bq[8][2];
        float sw[2];
        {
            float top = 0.0f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
                top = fmaxf(top, fmaxf(fmaxf(fabsf(x4[ks].x), fabsf(x4[ks].y)), fmaxf(fabsf(x4[ks].z), fabsf(x4[ks].w))));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // per head, 2^e brings max |q| into [2^14, 2^15): neither half leaves F16's normal range
            const int qe = (int)((__float_as_uint(top) >> 23) & 0xffu);
            const int e = (qe == 0 || qe == 0xff) ? 0 : max(-113, min(100, 141 - qe));
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                bq[ks][0] = split_pair(x4[ks].x * up, x4[ks].y * up, g >= 4);
                bq[ks][1] = split_pair(x4[ks].z * up, x4[ks].w * up, g >= 4);
            }
            const float s = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
            sw[0] = __shfl_sync(0xffffffffu, s, h0 * 4);
            sw[1] = __shfl_sync(0xffffffffu, s, (h0 + 1) * 4);
        }
        for (uint32_t u = begin; u < stop; ++u) {
            const int live = (int)min(tokens - (u - run_begin) * R::kTokens, (uint32_t)R::kTokens);
            // ---------------- K: logits
            uint32_t s = it % kSlots;
            alive = __all_sync(0xffffffffu, mbar_wait(&full[s], (it / kSlots) & 1));
            if (!alive) break;
            const bool skip = bad[s];
            uint32_t blk = smem_addr(ring + s * R::kSlot);
            float x[2][kTiles];  // [head][own row]
            {
                float acc[kTiles][4];
#pragma unroll
                for (int mt = 0; mt < kTiles; ++mt) {
                    acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.0f;
                    const uint32_t ra = blk + (mt * 16 + g) * 128;
#pragma unroll
                    for (int pl = 0; pl < Fmt::kPanels; ++pl)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t at16 = ra + pl * R::kPanel + (((2 * t + i) ^ g) << 4);
                            const uint4 va = lds128(at16), vb = lds128(at16 + 8 * 128);
                            const uint32_t a[4] = {va.x, va.y, va.z, va.w}, b[4] = {vb.x, vb.y, vb.z, vb.w};
                            if constexpr (Fmt::kScaled) {
#pragma unroll
                                for (int w = 0; w < 4; ++w) {
                                    uint32_t a0, a2, a1, a3;
                                    codes_to_half2<F>(a[w], a0, a2);
                                    codes_to_half2<F>(b[w], a1, a3);
                                    mma_f16(acc[mt], a0, a1, a2, a3, bq[i * 4 + w][0], bq[i * 4 + w][1]);
                                }
                            } else {
#pragma unroll
                                for (int w = 0; w < 2; ++w) {
                                    const int ks = pl * 4 + i * 2 + w;
                                    mma_f16(acc[mt], a[2 * w], b[2 * w], a[2 * w + 1], b[2 * w + 1], bq[ks][0], bq[ks][1]);
                                }
                            }
                        }
                }
                // rounding + remainder: each lane gives away the rows it does not own
#pragma unroll
                for (int e = 0; e < kTiles; ++e)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float a = acc[e >> 1][(e & 1) * 2 + j], b = acc[(kTiles + e) >> 1][(e & 1) * 2 + j];
                        x[j][e] = (low ? b : a) + __shfl_xor_sync(0xffffffffu, low ? a : b, 2);
                    }
            }
            __syncwarp();  // the slot is read
            if (!feed.done()) feed_one();
            ++it;
            // ---------------- V: weights and output
            s = it % kSlots;
            alive = __all_sync(0xffffffffu, mbar_wait(&full[s], (it / kSlots) & 1));
            if (!alive) break;
            if (!skip) {
                blk = smem_addr(ring + s * R::kSlot);
                float vs[kTiles];
#pragma unroll
                for (int e = 0; e < kTiles; ++e) {
                    float ks = 1.0f;
                    if constexpr (Fmt::kScaled) {
                        ks = lds32(blk + R::kPart + (token0 + 8 * e) * 4);
                        vs[e] = lds32(blk + R::kPart + (kPageTokens + token0 + 8 * e) * 4);
                    }
                    x[0][e] *= sw[0] * ks;
                    x[1][e] *= sw[1] * ks;
                }
                if (live < R::kTokens) {
#pragma unroll
                    for (int e = 0; e < kTiles; ++e)
                        if (token0 + 8 * e >= live) {
                            x[0][e] = x[1][e] = -INFINITY;
                            vs[e] = 0.0f;  // an unwritten row's scale may be anything
                        }
                }
                bool grown = false;
#pragma unroll
                for (int e = 0; e < kTiles; ++e) grown |= x[0][e] > M[0] + kSlack || x[1][e] > M[1] + kSlack;
                grown = __any_sync(0xffffffffu, grown);
                float fold[2] = {1.0f, 1.0f};
                if (grown) {  // move the maxima (of both lanes' rows)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = x[j][0];
#pragma unroll
                        for (int e = 1; e < kTiles; ++e) top = fmaxf(top, x[j][e]);
                        top = fmaxf(rows_max(top, t & 1), M[j]);
                        fold[j] = M[j] == -INFINITY ? 0.0f : exp2_ftz(M[j] - top);
                        L[j] *= fold[j];
                        M[j] = top;
                    }
                }
                const float base0 = M[0] == -INFINITY ? 0.0f : M[0], base1 = M[1] == -INFINITY ? 0.0f : M[1];
                bool over = false;
#pragma unroll
                for (int e = 0; e < kTiles; ++e) {
                    const float p0 = exp2_ftz(x[0][e] - base0), p1 = exp2_ftz(x[1][e] - base1);
                    L[0] += p0;
                    L[1] += p1;
                    x[0][e] = Fmt::kScaled ? p0 * vs[e] : p0;
                    x[1][e] = Fmt::kScaled ? p1 * vs[e] : p1;
                    if constexpr (Fmt::kScaled) over |= x[0][e] * unit[0] > kTopWeight || x[1][e] * unit[1] > kTopWeight;
                }
                if constexpr (Fmt::kScaled) over = __any_sync(0xffffffffu, over);
                if (grown || over) {
                    // the sums' new references: the maxima, and in 8 bits units for the largest weight so far
                    if constexpr (Fmt::kScaled) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float top = x[j][0];
#pragma unroll
                            for (int e = 1; e < kTiles; ++e) top = fmaxf(top, x[j][e]);
                            const float held = fold[j] * (kWeightUnit * inverse_of_power(unit[j]));
                            top = fmaxf(fmaxf(rows_max(top, t & 1), held), kLeastWeight);
                            const float up = __uint_as_float((__float_as_uint(top) + 0x7fffffu) & 0xff800000u);
                            fold[j] = held * inverse_of_power(up);
                            unit[j] = kWeightUnit * inverse_of_power(up);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        o[j][0] *= fold[0];
                        o[j][1] *= fold[1];
                        o[j][2] *= fold[0];
                        o[j][3] *= fold[1];
                    }
                }
                uint32_t bp[2 * kTiles];  // P^T fragments of rows i
#pragma unroll
                for (int e = 0; e < kTiles; ++e) {
                    const float w0 = x[0][e] * unit[0], w1 = x[1][e] * unit[1];
                    const __half2 hi = __floats2half2_rn(w0, w1);
                    const float2 f = __half22float2(hi);
                    const __half2 lo = __floats2half2_rn(w0 - f.x, w1 - f.y);
                    const uint32_t hw = *reinterpret_cast<const uint32_t*>(&hi), lw = *reinterpret_cast<const uint32_t*>(&lo);
                    const uint32_t keep = low ? lw : hw, other = __shfl_xor_sync(0xffffffffu, low ? hw : lw, 2);
                    bp[e] = transpose_8x8(low ? other : keep);
                    bp[kTiles + e] = transpose_8x8(low ? keep : other);
                }
                // The tensor cores add with truncation: a unit's products start from zero and are then
                // added with rounding (64 x 32768 F16 against 64 bits: 1.4e-6 in one chain, 0.8e-6 so;
                // the time is the same).
                float part[8][4];
#pragma unroll
                for (int j = 0; j < 8; ++j) part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0.0f;
#pragma unroll
                for (int kt = 0; kt < kTiles; ++kt) {
                    const int row = kt * 16 + 2 * t;  // and + 1, + 8, + 9
                    const uint32_t ra = blk + row * 128;
#pragma unroll
                    for (int pl = 0; pl < Fmt::kPanels; ++pl) {
                        uint4 v[4];
                        v[0] = lds128(ra + pl * R::kPanel + ((g ^ (2 * t)) << 4));
                        v[1] = lds128(ra + pl * R::kPanel + 128 + ((g ^ (2 * t + 1)) << 4));
                        v[2] = lds128(ra + pl * R::kPanel + 8 * 128 + ((g ^ (2 * t)) << 4));
                        v[3] = lds128(ra + pl * R::kPanel + 9 * 128 + ((g ^ (2 * t + 1)) << 4));
                        if (live < R::kTokens) {  // rows behind the last token may hold NaN: 0 x NaN must not enter
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (row + (i >> 1) * 8 + (i & 1) >= live) v[i] = make_uint4(0, 0, 0, 0);
                        }
                        const uint32_t A[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, B[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
                        const uint32_t C[4] = {v[2].x, v[2].y, v[2].z, v[2].w}, D[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if constexpr (Fmt::kScaled) {
                                // bytes of two tokens interleaved: channel by channel (token, token + 1)
                                uint32_t a0, a1, a2, a3;
                                codes_to_half2<F>(__byte_perm(A[w], B[w], 0x5140), a0, a1);
                                codes_to_half2<F>(__byte_perm(C[w], D[w], 0x5140), a2, a3);
                                mma_f16(part[2 * w], a0, a1, a2, a3, bp[2 * kt], bp[2 * kt + 1]);
                                codes_to_half2<F>(__byte_perm(A[w], B[w], 0x7362), a0, a1);
                                codes_to_half2<F>(__byte_perm(C[w], D[w], 0x7362), a2, a3);
                                mma_f16(part[2 * w + 1], a0, a1, a2, a3, bp[2 * kt], bp[2 * kt + 1]);
                            } else {
                                mma_f16(part[pl * 4 + w], __byte_perm(A[w], B[w], 0x5410), __byte_perm(A[w], B[w], 0x7632),
                                        __byte_perm(C[w], D[w], 0x5410), __byte_perm(C[w], D[w], 0x7632), bp[2 * kt],
                                        bp[2 * kt + 1]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[j][r] += part[j][r];
            }
            __syncwarp();
            if (!feed.done()) feed_one();
            ++it;
        }
        if (!alive) break;
        const bool begins = run_begin >= begin, ends = run_end <= k.end, whole = begins && ends;
        k.u = stop - 1;  // to the next run (or behind the part)
        k.step(p);
        if (!k.done()) load_query();
        // ---------------- the run's end here: all rows' sums, rounding + remainder.  Lanes t < 2
        // keep head h0, lanes t >= 2 head h0 + 1, and give the other's parts away.
        const int h = h0 + low;
        const float os = inverse_of_power(low ? unit[1] : unit[0]);
        const float top = low ? M[1] : M[0];
        float sum = (low ? L[1] : L[0]) + __shfl_xor_sync(0xffffffffu, low ? L[0] : L[1], 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        // a whole run's results, or a piece in shared memory: one that goes on is the part's
        // last, so the ring has no more copies in flight and keeps it
        if (!whole && lane == 0) {
            Piece& c = pieces[warp][begins];
            c.id = run;
            c.first = run_begin;
            c.last = run_end;
            c.ends = ends;
            c.there = 1;
        }
        const bool final = kFinal && whole;
        if (!kFinal && whole && lane == 0) p.place[run] = 0;
        float* slot = whole ? p.whole + (size_t)run * kPartFloats
                            : begins ? reinterpret_cast<float*>(ring) : heads_s + warp * kPartFloats;
        float* dst = final ? p.out + ((size_t)run * kGroup + h) * kDim : slot + 2 * kGroup + h * kDim;
        const float by = final ? os * (sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum)) : os;
        if (!final && g == 0) {
            slot[2 * h] = top;
            slot[2 * h + 1] = sum;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // MMA rows g, g + 8 of tile j: two neighbouring channels
            const float a = (low ? o[j][1] : o[j][0]) + __shfl_xor_sync(0xffffffffu, low ? o[j][0] : o[j][1], 2);
            const float b = (low ? o[j][3] : o[j][2]) + __shfl_xor_sync(0xffffffffu, low ? o[j][2] : o[j][3], 2);
            const int c = Fmt::kScaled ? g * 16 + 2 * j : (j >> 2) * 64 + g * 8 + (j & 3) * 2;
            *reinterpret_cast<float2*>(dst + c) = make_float2(a * by, b * by);
        }
    }
    if (!alive) {  // gave up: copies in flight land before shared memory is released
        if (lane == 0) raise_status(p.status, HSB_E_TIMEOUT, blockIdx.x);
        for (uint32_t j = it; j < fed; ++j) (void)mbar_wait(&full[j % kSlots], (j / kSlots) & 1);
    }
    __syncthreads();
    // ================ the runs that crossed warps: pieces of one run, in order, each run by one warp
    static_assert(2 * kWarps <= 32, "a lane a piece");
    const auto piece_at = [&](int i) -> const float* {
        return i & 1 ? reinterpret_cast<const float*>(ring0 + (i >> 1) * kSlots * R::kSlot) : heads_s + (i >> 1) * kPartFloats;
    };
    const Piece* const mine = lane < 2 * kWarps ? &pieces[lane >> 1][lane & 1] : nullptr;
    uint32_t there = __ballot_sync(0xffffffffu, mine && mine->there);
    const uint32_t ends_mask = __ballot_sync(0xffffffffu, mine && mine->there && mine->ends);
    for (int order = 0; there; ++order) {
        // the next run's pieces: up to the one that ends it
        const int first = __ffs(there) - 1;
        uint32_t members = there;
        // a piece that begins a run goes on; one that does not ends it or fills its warp's part
        const uint32_t stop = (first & 1 ? there & ends_mask & ~(1u << first) : there & ends_mask);
        if (stop) members &= (2u << (__ffs(stop) - 1)) - 1;
        there &= ~members;
        if (order % kWarps != warp) continue;
        const Piece c = pieces[first >> 1][first & 1];
        const bool begins = c.first >= stretch[0], ends = c.last <= stretch[1];
        const int h = lane >> 3;
        float top = -INFINITY, sum = 0.0f;
        float4 acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t left = members; left; left &= left - 1) top = fmaxf(top, piece_at(__ffs(left) - 1)[2 * h]);
        for (uint32_t left = members; left; left &= left - 1) {
            const float* part = piece_at(__ffs(left) - 1);
            // (no token under a finite maximum: sum 0; a NaN sum comes through)
            const float f = top == -INFINITY ? 1.0f : exp2_ftz(part[2 * h] - top);
            sum = fmaf(f, part[2 * h + 1], sum);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 v = reinterpret_cast<const float4*>(part + 2 * kGroup + h * kDim)[(lane & 7) + 8 * j];
                acc[j] = make_float4(fmaf(f, v.x, acc[j].x), fmaf(f, v.y, acc[j].y), fmaf(f, v.z, acc[j].z),
                                     fmaf(f, v.w, acc[j].w));
            }
        }
        const bool final = kFinal && begins && ends;
        float* slot = begins && ends ? p.whole + (size_t)c.id * kPartFloats
                                     : p.part + ((size_t)blockIdx.x * 2 + begins) * kPartFloats;
        float* dst = final ? p.out + ((size_t)c.id * kGroup + h) * kDim : slot + 2 * kGroup + h * kDim;
        const float by = final ? (sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum)) : 1.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            reinterpret_cast<float4*>(dst)[(lane & 7) + 8 * j] =
                make_float4(acc[j].x * by, acc[j].y * by, acc[j].z * by, acc[j].w * by);
        if (!final && (lane & 7) == 0) {
            slot[2 * h] = top;
            slot[2 * h + 1] = sum;
        }
        if (lane == 0 && begins && !(kFinal && ends)) {
            RunInfo info{};
            info.run = (int)c.id;
            info.last = ends ? blockIdx.x : Split(units, gridDim.x).of(c.last - 1);
            if (kFinal) p.info[blockIdx.x] = info;
            else p.place[c.id] = ends ? 0 : cut_run(blockIdx.x, info.last - blockIdx.x + 1);
        }
    }
    if (!kFinal) pdl_wait();
}

// Folds the partials of the run that begins in CTA blockIdx.x's stretch and
// does not end there, in the order of the CTAs (a run that goes on leaves no
// empty stretch before its end): head blockIdx.y, thread = channel.  Every load
// of the first 32 partials' weights and 8 outputs is on its way before the
// run's extent is known; what lies behind it is not used.  The kernel may be
// resident while its partials are written: no pointer promises constant data,
// so that no load may pass the wait.
__global__ void __launch_bounds__(kDim) kv_combine_kernel(const float* part, const RunInfo* infos, float* out) {
    constexpr int kFirst = 8;
    pdl_trigger();
    pdl_wait();
    const int h = blockIdx.y, d = threadIdx.x, lane = d & 31;
    const int room = (int)(gridDim.x - blockIdx.x);  // partials that there can be
    // the first partial is its CTA's [1], the others their CTAs' [0]
    const float* base = part + (size_t)blockIdx.x * 2 * kPartFloats;
    const auto at = [&](int i) { return base + ((size_t)i * 2 + (i == 0)) * kPartFloats; };
    const RunInfo info = infos[blockIdx.x];
    float2 ml = lane < room ? __ldcg(reinterpret_cast<const float2*>(at(lane) + 2 * h)) : make_float2(0.0f, 0.0f);
    float v[kFirst];
#pragma unroll
    for (int i = 0; i < kFirst; ++i) v[i] = i < room ? __ldcg(at(i) + 2 * kGroup + h * kDim + d) : 0.0f;
    if (info.run < 0) return;
    const int n = (int)(info.last - blockIdx.x) + 1;
    float M = -INFINITY, L = 0.0f, acc = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 32) {
        if (i0) ml = i0 + lane < n ? __ldcg(reinterpret_cast<const float2*>(at(i0 + lane) + 2 * h)) : make_float2(0.0f, 0.0f);
        const bool some = i0 + lane < n;
        const float top = fmaxf(M, warp_max(some ? ml.x : -INFINITY));
        // (all -infinity: no token, sum 0; a NaN sum comes through)
        const float old = M == -INFINITY ? 0.0f : exp2_ftz(M - top);
        const float f = !some ? 0.0f : top == -INFINITY ? 1.0f : exp2_ftz(ml.x - top);
        L = L * old + warp_sum(some ? f * ml.y : 0.0f);
        acc *= old;
        M = top;
        const int m = min(32, n - i0);
        int i = 0;
        if (i0 == 0) {
#pragma unroll
            for (i = 0; i < kFirst; ++i)
                if (i < m) acc = fmaf(__shfl_sync(0xffffffffu, f, i), v[i], acc);
        }
#pragma unroll 8
        for (; i < m; ++i)
            acc = fmaf(__shfl_sync(0xffffffffu, f, i), __ldcg(at(i0 + i) + 2 * kGroup + h * kDim + d), acc);
    }
    out[((size_t)info.run * kGroup + h) * kDim + d] = acc * (L > 0.0f ? 1.0f / L : (L == L ? 0.0f : L));
}

template <int F, typename Q, bool kFinal>
cudaError_t launch(const PagedAttention& p, unsigned grid, cudaStream_t stream) {
    static thread_local int configured = -1;
    const int device = device_info().ordinal;
    if (configured != device) {
        cudaError_t e = cudaFuncSetAttribute(kv_attention_kernel<F, Q, kFinal>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<F>::kSmem);
        if (e != cudaSuccess) return e;
        configured = device;
    }
    return launch_dependent(kv_attention_kernel<F, Q, kFinal>, dim3(grid), dim3(Ring<F>::kThreads), Ring<F>::kSmem, stream,
                            false, p);
}

template <typename Q, bool kFinal>
cudaError_t launch_format(int format, const PagedAttention& p, unsigned grid, cudaStream_t stream) {
    switch (format) {
    case HSB_KV_F16: return launch<HSB_KV_F16, Q, kFinal>(p, grid, stream);
    case HSB_KV_INT8: return launch<HSB_KV_INT8, Q, kFinal>(p, grid, stream);
    default: return launch<HSB_KV_E4M3, Q, kFinal>(p, grid, stream);
    }
}

}  // namespace

// A CTA a run needs no scan of the lengths, no partials and no second launch, but
// its eight warps are all that a run gets.  int8, 8 heads, by runs and split: one
// sequence of 77 tokens (e4m3) 4.9 and 7.4 us, 512 7.7 and 8.1, 1000 10.3 and 9.5,
// 2000 15.3 and 10.2; sixteen of up to 1000 10.8 and 14.7, 2000 17.2 and 17.8, 4000
// 27.0 and 22.5.  The host knows the tables' width, not the lengths: short
// sequences in wide tables are split too.
bool paged_by_run(size_t batch, size_t table_width, int heads) {
    const size_t runs = batch * heads, sms = device_info().sms;
    return runs <= sms && table_width <= (2 * runs >= sms ? 32 : 12);
}

unsigned paged_attention_grid(size_t batch, size_t table_width, int heads) {
    if (paged_by_run(batch, table_width, heads)) return (unsigned)(batch * heads);
    const unsigned sms = (unsigned)device_info().sms;
    const size_t units = batch * table_width * heads;
    return (unsigned)std::max<size_t>(1, std::min<size_t>(units, std::min<unsigned>(sms, kAttnMaxCtas)));
}

cudaError_t launch_paged_partials(int format, const PagedAttention& p, unsigned grid, cudaStream_t stream) {
    return launch_format<uint16_t, false>(format, p, grid, stream);
}

}  // namespace hsb

using namespace hsb;

extern "C" {

size_t hsb_kv_attention_workspace_bytes(size_t, int) {
    return align256(kAttnMaxCtas * sizeof(RunInfo)) + align256((size_t)kAttnMaxCtas * 2 * kPartFloats * sizeof(float));
}

int hsb_kv_attention(const hsb_kv_pages* pages, const int32_t* d_table, size_t table_width, const int32_t* d_lengths,
                     size_t batch, const float* d_q, float* d_out, void* d_workspace, size_t workspace_bytes,
                     hsb_device_status* d_status, void* stream) {
    if (!kv_pages_valid(pages)) return record_error(HSB_E_KV_SHAPE, "paged KV pool arguments");
    if (!d_table || !table_width || table_width > kMaxTableEntries || !d_lengths || !batch || batch > kMaxBatch ||
        batch * table_width > kMaxTableEntries || !d_q || !d_out)
        return record_error(HSB_E_KV_SHAPE, "paged KV attention shape");
    if (!aligned_to(16, d_q, d_out, static_cast<unsigned char*>(d_workspace)) || !aligned_to(4, d_table, d_lengths) ||
        !aligned_to(8, d_status))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention buffers are misaligned");
    const size_t bytes = batch * pages->kv_heads * kGroup * kDim * sizeof(float);
    if (!apart(d_q, bytes, d_out, bytes))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention output must not alias the query");
    const size_t needed = hsb_kv_attention_workspace_bytes(batch, pages->kv_heads);
    if (!d_workspace || workspace_bytes < needed)
        return record_error(HSB_E_WORKSPACE, "paged KV attention workspace missing or too small");
    if (!apart(d_workspace, needed, d_q, bytes) || !apart(d_workspace, needed, d_out, bytes))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention workspace must not alias the query or the output");
    PagedAttention p{};
    p.v = paged_view(*pages, d_table, table_width, table_width);
    p.lengths = d_lengths;
    p.batch = batch;
    p.q = d_q;
    p.out = d_out;
    p.info = static_cast<RunInfo*>(d_workspace);
    p.part = reinterpret_cast<float*>(static_cast<unsigned char*>(d_workspace) + align256(kAttnMaxCtas * sizeof(RunInfo)));
    p.status = d_status;
    p.scale_log2 = kScaleLog2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    p.by_run = paged_by_run(batch, table_width, pages->kv_heads);
    const unsigned grid = paged_attention_grid(batch, table_width, pages->kv_heads);
    cudaError_t e = launch_format<float, true>(pages->format, p, grid, s);
    if (e == cudaSuccess && !p.by_run)
        e = launch_dependent(kv_combine_kernel, dim3(grid, kGroup), dim3(kDim), 0, s, false,
                             static_cast<const float*>(p.part), static_cast<const RunInfo*>(p.info), p.out);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV attention launch");
    record_error(HSB_OK, "");
    return HSB_OK;
}

}  // extern "C"
