// kvattention.cu -- decode attention of a batch over the paged KV cache:
//   out[b][h] = softmax(q[b][h] . K_b^T / sqrt(128)) V_b,  K = codes x scales,
// one token per sequence, ragged lengths, four query heads to a KV head.
//
// Four rows of queries against every cached row is far too little arithmetic
// for the tensor cores' own pipeline to matter (4 flops a byte in F16, 8 in 8
// bits): the kernel is bound by the bytes of the pages, and is built to keep
// them coming.  Page blocks arrive whole by bulk copies into a ring of shared
// memory; warps take 32 tokens each, turn codes into F16 fragments in
// registers (both formats convert exactly) and run both products with
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
// multiplies a token's logits, the V scale its weight, both in F32; weights
// are brought to [0, 2^14] by a power of two before their split into halves.
//
// Work is split evenly without regard to lengths: the (sequence, head, page)
// units in that order are one line, of which every CTA takes an equal stretch.
// A (sequence, head) run inside one CTA is finished there; one that crosses
// CTAs leaves F32 partials that kv_combine_kernel folds in order.
#include <algorithm>
#include <cmath>

#include "kvattention.cuh"

namespace hsb {
namespace {

constexpr int kOutPitch = kDim + 4;
constexpr float kWeightTop = 16384.0f;  // 2^14: weights' F16 halves are at most this

// Warps 2 i and 2 i + 1 take the two halves of units i, i + kConsumers / 2, ...
// The ring's length is a multiple of that step, so a stage has the same two
// readers in every round: one that skipped a round could take the parity of a
// later fill for that of an earlier one.
template <int F>
struct Ring {
    static constexpr int kConsumers = F == HSB_KV_F16 ? 6 : 8;
    static constexpr int kThreads = (kConsumers + 1) * 32;
    static constexpr int kStages = F == HSB_KV_F16 ? 6 : 12;
    static_assert(kStages % (kConsumers / 2) == 0, "a stage keeps its readers");
    static constexpr int kData = kStages * PageFormat<F>::kBytes;
    static constexpr int kMerge = kConsumers * kGroup * (kOutPitch + 2) * 4;
    static constexpr int kSmem = 128 + kData + kMerge;
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
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ float lds32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ __half split_half(float x, bool low) {
    const __half hi = __float2half_rn(x);
    return low ? __float2half_rn(x - __half2float(hi)) : hi;
}
__device__ __forceinline__ uint32_t pack2(__half a, __half b) {
    return (uint32_t)__half_as_ushort(a) | ((uint32_t)__half_as_ushort(b) << 16);
}
__device__ __forceinline__ float load_q(const float* q, size_t i) { return q[i]; }
__device__ __forceinline__ float load_q(const uint16_t* q, size_t i) { return half_value(q[i]); }

// Tokens of a sequence; a length behind the table's end counts as none.
__device__ __forceinline__ unsigned long long tokens_of(const PagedAttention& p, unsigned long long b, bool report) {
    if (!p.lengths) return p.length;
    const int32_t n = p.lengths[b];
    if (n < 0 || (unsigned long long)n > p.v.width * kPageTokens) {
        if (report) raise_status(p.status, HSB_E_KV_POSITION, (int)b);
        return 0;
    }
    return n;
}

// A CTA's stretch of the line of units, one (sequence, head) run at a time.
struct Walker {
    unsigned long long u, end;      // the stretch [u, end)
    unsigned long long seq, tokens, pages;
    unsigned long long run;         // first unit of the current run
    int head;
    __device__ unsigned long long stop() const { return min(end, run + pages); }
    __device__ void next(const PagedAttention& p) {
        u = stop();
        run += pages;
        if (++head < p.v.heads || u >= end) return;
        head = 0;
        do {
            ++seq;
            tokens = tokens_of(p, seq, false);
            pages = (tokens + kPageTokens - 1) / kPageTokens;
        } while (pages == 0);
    }
};

// Finds CTA `cta`'s stretch of `ctas`.  Every thread of the block calls it.
template <int kThreads>
__device__ Walker find_stretch(const PagedAttention& p, unsigned cta, unsigned ctas, unsigned long long* total_units) {
    __shared__ unsigned long long warp_sum_s[kThreads / 32];
    __shared__ unsigned long long found[4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned long long per = (p.batch + kThreads - 1) / kThreads;
    const unsigned long long b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
    unsigned long long mine = 0;
    for (unsigned long long b = b0; b < b1; ++b)
        mine += (tokens_of(p, b, cta == 0) + kPageTokens - 1) / kPageTokens;
    unsigned long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    if (lane == 31) warp_sum_s[warp] = upto;
    __syncthreads();
    unsigned long long total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w == warp) before = total;
        total += warp_sum_s[w];
    }
    before += upto - mine;  // pages of the sequences before b0
    if (p.cum && cta == 0) {
        unsigned long long c = before;
        for (unsigned long long b = b0; b < b1; ++b) {
            p.cum[b] = c;
            c += (tokens_of(p, b, false) + kPageTokens - 1) / kPageTokens;
        }
        if (tid == 0) p.cum[p.batch] = total;
    }
    const unsigned long long units = total * p.v.heads;
    *total_units = units;
    Walker k{};
    k.u = stretch_begin(units, cta, ctas);
    k.end = stretch_begin(units, cta + 1, ctas);
    if (k.u < k.end) {
        const unsigned long long page = k.u / p.v.heads;  // the sequence whose pages hold this rank
        if (page >= before && page < before + mine) {
            unsigned long long b = b0, n, pages;
            while (true) {
                n = tokens_of(p, b, false);
                pages = (n + kPageTokens - 1) / kPageTokens;
                if (page < before + pages) break;
                before += pages;
                ++b;
            }
            found[0] = b;
            found[1] = n;
            found[2] = before;
        }
    }
    __syncthreads();
    if (k.u < k.end) {
        k.seq = found[0];
        k.tokens = found[1];
        k.pages = (k.tokens + kPageTokens - 1) / kPageTokens;
        const unsigned long long base = found[2] * p.v.heads;
        k.head = (int)((k.u - base) / k.pages);
        k.run = base + k.head * k.pages;
    }
    return k;
}

template <int F, typename Q, bool kFinal>
__global__ void __launch_bounds__(Ring<F>::kThreads, 1) kv_attention_kernel(const __grid_constant__ PagedAttention p) {
    using Fmt = PageFormat<F>;
    using R = Ring<F>;
    constexpr int kConsumers = R::kConsumers, kThreads = R::kThreads;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t full[R::kStages], empty[R::kStages];
    __shared__ int bad[R::kStages];
    __shared__ volatile int dead;
    unsigned char* ring = smem_raw + ((128u - (smem_addr(smem_raw) & 127u)) & 127u);
    float* merge = reinterpret_cast<float*>(ring + R::kData);  // [warp][head][kOutPitch], then [warp][head][2]
    float* merge_ml = merge + kConsumers * kGroup * kOutPitch;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < R::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 2);
        }
        mbar_fence_init();
        dead = 0;
    }
    pdl_wait();
    pdl_trigger();
    unsigned long long units;
    Walker k = find_stretch<kThreads>(p, blockIdx.x, gridDim.x, &units);  // syncs: the barriers are ready
    if (kFinal) {  // empty sequences: zeros
        for (unsigned long long b = blockIdx.x; b < p.batch; b += gridDim.x)
            if (tokens_of(p, b, false) == 0)
                for (int i = tid; i < p.v.heads * kGroup * kDim; i += kThreads)
                    p.out[b * p.v.heads * kGroup * kDim + i] = 0.0f;
    }
    if (tid == 0) {
        RunInfo info{};
        info.run = -1;
        info.units = units;
        p.info[blockIdx.x] = info;
    }
    if (k.u >= k.end) return;
    const unsigned long long begin = k.u;

    if (warp == kConsumers) {
        // ---------------- producer: one block per unit
        uint32_t it = 0;
        bool ok = true;
        for (; ok && k.u < k.end; k.next(p)) {
            const unsigned long long stop = k.stop();
            for (unsigned long long u = k.u; ok && u < stop; u += 32) {
                const unsigned long long mine = u + lane;
                const int32_t page = mine < stop ? p.v.table[k.seq * p.v.pitch + (mine - k.run)] : 0;
                const int n = (int)min(stop - u, 32ull);
                for (int i = 0; i < n; ++i, ++it) {
                    const uint32_t s = it % R::kStages;
                    if (it >= R::kStages) ok = mbar_wait(&empty[s], ((it / R::kStages) - 1) & 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const int32_t id = __shfl_sync(0xffffffffu, page, i);
                    if (lane == 0) {
                        const bool have = id >= 0 && (unsigned long long)id < p.v.pages;
                        bad[s] = !have;
                        if (have) {
                            mbar_arrive_expect_tx(&full[s], Fmt::kBytes);
                            bulk_copy_g2s(ring + s * Fmt::kBytes,
                                          p.v.data + ((size_t)id * p.v.heads + k.head) * Fmt::kBytes, Fmt::kBytes,
                                          &full[s]);
                        } else {  // no such page: its tokens are left out
                            raise_status(p.status, HSB_E_KV_PAGE, (int)k.seq);
                            mbar_arrive(&full[s]);
                        }
                    }
                }
            }
        }
        if (!ok) {  // give up, once the copies in flight have landed
            if (lane == 0) {
                raise_status(p.status, HSB_E_TIMEOUT, blockIdx.x);
                dead = 1;
            }
            const uint32_t first = it > R::kStages ? it - R::kStages : 0;
            for (uint32_t j = first; j < it; ++j) (void)mbar_wait(&full[j % R::kStages], (j / R::kStages) & 1);
        }
        return;
    }

    // ---------------- consumers
    const int g = lane >> 2, t = lane & 3;
    const bool low = t >= 2;        // this lane's accumulator columns are the remainders' (and g >= 4 in B fragments)
    const int h0 = 2 * (t & 1);     // they are heads h0 and h0 + 1 of the group
    uint32_t hp0 = 0;               // half pages of the stretch before the current segment
    for (; k.u < k.end; k.next(p)) {
        const unsigned long long stop = k.stop();
        const uint32_t hp1 = hp0 + 2 * (uint32_t)(stop - k.u);
        float M[2] = {-INFINITY, -INFINITY}, L[2] = {0.0f, 0.0f}, vref = 0.0f;
        float o[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        uint32_t hp = hp0 + (warp + kConsumers - hp0 % kConsumers) % kConsumers;
        if (hp < hp1) {
            // Q^T fragments: column g = head g & 3, its rounding or remainder (g >= 4)
            uint32_t bq[8][2];
            float sw[2];
            {
                const Q* q = static_cast<const Q*>(p.q) + ((k.seq * p.v.heads + k.head) * kGroup + (g & 3)) * kDim;
                float x[8][4], top = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const int c = Fmt::kScaled ? t * 32 + ks * 4 : (ks >> 2) * 64 + t * 16 + (ks & 3) * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[ks][i] = load_q(q, c + i);
                }
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[ks][i]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // per head, 2^e brings max |q| into [2^14, 2^15): neither half leaves F16's normal range
                const int qe = (int)((__float_as_uint(top) >> 23) & 0xffu);
                const int e = (qe == 0 || qe == 0xff) ? 0 : max(-100, min(100, 141 - qe));
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        bq[ks][i] = pack2(split_half(x[ks][2 * i] * up, g >= 4), split_half(x[ks][2 * i + 1] * up, g >= 4));
                const float s = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
                sw[0] = __shfl_sync(0xffffffffu, s, h0 * 4);
                sw[1] = __shfl_sync(0xffffffffu, s, (h0 + 1) * 4);
            }
            for (; hp < hp1; hp += kConsumers) {
                const uint32_t unit = hp >> 1;  // of the stretch
                const uint32_t s = unit % R::kStages;
                if (!__all_sync(0xffffffffu, !dead && mbar_wait(&full[s], (unit / R::kStages) & 1))) {
                    if (lane == 0) {
                        raise_status(p.status, HSB_E_TIMEOUT, blockIdx.x);
                        dead = 1;
                    }
                    break;
                }
                const int r0 = (int)(hp & 1) * 32;
                const unsigned long long at = (begin + unit - k.run) * kPageTokens + r0;
                const int live = bad[s] || at >= k.tokens ? 0 : (int)min(k.tokens - at, 32ull);
                if (live) {
                    const uint32_t blk = smem_addr(ring + s * Fmt::kBytes);
                    // ---- logits
                    float acc[2][4];
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.0f;
                        const uint32_t ra = blk + (r0 + mt * 16 + g) * 128;
#pragma unroll
                        for (int pl = 0; pl < Fmt::kPanels; ++pl)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint32_t at16 = ra + pl * kPanelBytes + (((2 * t + i) ^ g) << 4);
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
                    // ---- online softmax: this lane has tokens g + 8 i of heads h0, h0 + 1
                    float vs[4] = {kWeightTop, kWeightTop, kWeightTop, kWeightTop};
                    float x[2][4];  // [head][i]
                    float vfold = 1.0f;
                    if constexpr (Fmt::kScaled) {
                        const uint32_t sc = blk + Fmt::kScaleOffset + (r0 + g) * 4;
                        float vtop = 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            vs[i] = lds32(sc + kPageTokens * 4 + i * 32);
                            if (8 * i + g < live) vtop = fmaxf(vtop, vs[i]);
                        }
                        vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 4));
                        vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 8));
                        vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 16));
                        // the next power of two: weight x scale stays within kWeightTop
                        const float up = __uint_as_float((__float_as_uint(vtop) + 0x7fffffu) & 0xff800000u);
                        if (up > vref) {
                            vfold = vref / up;
                            vref = up;
                        }
                        const float inv = vref > 0.0f ? kWeightTop / vref : 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) vs[i] *= inv;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float ks = lds32(sc + i * 32);
                            const int mt = i >> 1, r = (i & 1) * 2;
                            x[0][i] = (acc[mt][r] + __shfl_xor_sync(0xffffffffu, acc[mt][r], 2)) * (sw[0] * ks);
                            x[1][i] = (acc[mt][r + 1] + __shfl_xor_sync(0xffffffffu, acc[mt][r + 1], 2)) * (sw[1] * ks);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int mt = i >> 1, r = (i & 1) * 2;
                            x[0][i] = (acc[mt][r] + __shfl_xor_sync(0xffffffffu, acc[mt][r], 2)) * sw[0];
                            x[1][i] = (acc[mt][r + 1] + __shfl_xor_sync(0xffffffffu, acc[mt][r + 1], 2)) * sw[1];
                        }
                    }
                    if (live < 32) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (8 * i + g >= live) {
                                x[0][i] = x[1][i] = -INFINITY;
                                vs[i] = 0.0f;  // an unwritten row's scale may be anything
                            }
                    }
                    float mx[2], fold[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mx[j] = fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3]));
                        mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 4));
                        mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 8));
                        mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 16));
                        mx[j] = fmaxf(M[j], mx[j]);
                    }
                    // the accumulators change scale only where a maximum (or the V reference) grew
                    if (__any_sync(0xffffffffu, mx[0] > M[0] || mx[1] > M[1] || vfold != 1.0f)) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            fold[j] = M[j] == -INFINITY ? 0.0f : exp2f(M[j] - mx[j]);
                            L[j] *= fold[j];
                            fold[j] *= vfold;
                            M[j] = mx[j];
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            o[j][0] *= fold[0];
                            o[j][1] *= fold[1];
                            o[j][2] *= fold[0];
                            o[j][3] *= fold[1];
                        }
                    }
                    const float base0 = M[0] == -INFINITY ? 0.0f : M[0], base1 = M[1] == -INFINITY ? 0.0f : M[1];
                    uint32_t bp[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p0 = exp2f(x[0][i] - base0), p1 = exp2f(x[1][i] - base1);
                        L[0] += p0;
                        L[1] += p1;
                        bp[i] = transpose_8x8(pack2(split_half(p0 * vs[i], low), split_half(p1 * vs[i], low)));
                    }
                    // ---- output
                    const uint32_t vb = blk + Fmt::kPanels * kPanelBytes;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
                        const int row = kt * 16 + 2 * t;  // and + 1, + 8, + 9
                        const uint32_t ra = vb + (r0 + row) * 128;
#pragma unroll
                        for (int pl = 0; pl < Fmt::kPanels; ++pl) {
                            uint4 v[4];
                            v[0] = lds128(ra + pl * kPanelBytes + ((g ^ (2 * t)) << 4));
                            v[1] = lds128(ra + pl * kPanelBytes + 128 + ((g ^ (2 * t + 1)) << 4));
                            v[2] = lds128(ra + pl * kPanelBytes + 8 * 128 + ((g ^ (2 * t)) << 4));
                            v[3] = lds128(ra + pl * kPanelBytes + 9 * 128 + ((g ^ (2 * t + 1)) << 4));
                            if (live < 32) {  // rows behind the last token may hold NaN: 0 x NaN must not enter
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
                                    mma_f16(o[2 * w], a0, a1, a2, a3, bp[2 * kt], bp[2 * kt + 1]);
                                    codes_to_half2<F>(__byte_perm(A[w], B[w], 0x7362), a0, a1);
                                    codes_to_half2<F>(__byte_perm(C[w], D[w], 0x7362), a2, a3);
                                    mma_f16(o[2 * w + 1], a0, a1, a2, a3, bp[2 * kt], bp[2 * kt + 1]);
                                } else {
                                    mma_f16(o[pl * 4 + w], __byte_perm(A[w], B[w], 0x5410), __byte_perm(A[w], B[w], 0x7632),
                                            __byte_perm(C[w], D[w], 0x5410), __byte_perm(C[w], D[w], 0x7632), bp[2 * kt],
                                            bp[2 * kt + 1]);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
        }
        // ---- the segment's end: rounding + remainder, then the warps together
        const float os = Fmt::kScaled ? vref / kWeightTop : 1.0f / kWeightTop;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            L[j] += __shfl_xor_sync(0xffffffffu, L[j], 4);
            L[j] += __shfl_xor_sync(0xffffffffu, L[j], 8);
            L[j] += __shfl_xor_sync(0xffffffffu, L[j], 16);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[j][r] = (o[j][r] + __shfl_xor_sync(0xffffffffu, o[j][r], 2)) * os;
        if (!low) {
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int slot = warp * kGroup + h0 + hh;
                if (g == 0) {
                    merge_ml[slot * 2] = M[hh];
                    merge_ml[slot * 2 + 1] = L[hh];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {  // MMA rows g, g + 8 of tile j: two neighbouring channels
                    const int c = Fmt::kScaled ? g * 16 + 2 * j : (j >> 2) * 64 + g * 8 + (j & 3) * 2;
                    *reinterpret_cast<float2*>(merge + slot * kOutPitch + c) = make_float2(o[j][hh], o[j][hh + 2]);
                }
            }
        }
        named_sync(1, kConsumers * 32);
        for (int i = tid; i < kGroup * kDim / 2; i += kConsumers * 32) {
            const int h = i >> 6, c = (i & 63) * 2;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) top = fmaxf(top, merge_ml[(w * kGroup + h) * 2]);
            float sum = 0.0f, a = 0.0f, b = 0.0f;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) {
                // (a warp without tokens has sum 0; a NaN sum must come through)
                const float f = top == -INFINITY ? 1.0f : exp2f(merge_ml[(w * kGroup + h) * 2] - top);
                const float2 v = *reinterpret_cast<const float2*>(merge + (w * kGroup + h) * kOutPitch + c);
                sum = fmaf(f, merge_ml[(w * kGroup + h) * 2 + 1], sum);
                a = fmaf(f, v.x, a);
                b = fmaf(f, v.y, b);
            }
            const bool begins = k.run >= begin, ends = k.run + k.pages <= k.end;
            const unsigned long long run = k.seq * p.v.heads + k.head;
            if (kFinal && begins && ends) {
                const float inv = sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum);
                *reinterpret_cast<float2*>(p.out + (run * kGroup + h) * kDim + c) = make_float2(a * inv, b * inv);
            } else {
                float* slot = begins && ends ? p.whole + run * kPartFloats
                                             : p.part + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * kPartFloats;
                *reinterpret_cast<float2*>(slot + 2 * kGroup + h * kDim + c) = make_float2(a, b);
                if (c == 0) {
                    slot[2 * h] = top;
                    slot[2 * h + 1] = sum;
                }
                if (i == 0 && begins && !ends) {
                    RunInfo info{};
                    info.run = (long long)run;
                    info.units = units;
                    info.last = stretch_of(units, k.run + k.pages - 1, gridDim.x);
                    p.info[blockIdx.x] = info;
                }
            }
        }
        named_sync(1, kConsumers * 32);  // before the next segment writes the merge area
        hp0 = hp1;
    }
}

// Folds the partials of the run that begins in CTA blockIdx.x's stretch and
// does not end there, in the order of the CTAs.  Thread = (head, channel).
__global__ void __launch_bounds__(kGroup* kDim) kv_combine_kernel(const float* __restrict__ part,
                                                                 const RunInfo* __restrict__ infos,
                                                                 float* __restrict__ out) {
    __shared__ float weight[kGroup][kAttnMaxCtas];
    __shared__ float inv[kGroup];
    pdl_wait();
    pdl_trigger();
    const RunInfo info = infos[blockIdx.x];
    if (info.run < 0) return;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned first = blockIdx.x, ctas = gridDim.x;
    const int n = (int)(info.last - first) + 1;
    if (warp < kGroup) {  // weights of the partials of head `warp`
        float top = -INFINITY;
        for (int i = lane; i < n; i += 32) {
            const unsigned c = first + i;
            const bool some = stretch_begin(info.units, c, ctas) < stretch_begin(info.units, c + 1, ctas);
            const float m = some ? part[((size_t)c * 2 + (i == 0)) * kPartFloats + 2 * warp] : INFINITY;
            weight[warp][i] = m;
            if (some) top = fmaxf(top, m);
        }
        top = warp_max(top);
        float sum = 0.0f;
        for (int i = lane; i < n; i += 32) {
            const float m = weight[warp][i];
            // -1: an empty stretch, which left nothing
            const float f = m == INFINITY ? -1.0f : top == -INFINITY ? 1.0f : exp2f(m - top);
            weight[warp][i] = f;
            if (f >= 0.0f) sum = fmaf(f, part[((size_t)(first + i) * 2 + (i == 0)) * kPartFloats + 2 * warp + 1], sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) inv[warp] = sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum);
    }
    __syncthreads();
    const int h = tid / kDim;
    float acc = 0.0f;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
        const float f = weight[h][i];
        if (f >= 0.0f) acc = fmaf(f, part[((size_t)(first + i) * 2 + (i == 0)) * kPartFloats + 2 * kGroup + tid], acc);
    }
    out[(size_t)info.run * kGroup * kDim + tid] = acc * inv[h];
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

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
    return launch_dependent(kv_attention_kernel<F, Q, kFinal>, dim3(grid), dim3(Ring<F>::kThreads), Ring<F>::kSmem, stream, false, p);
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

unsigned paged_attention_grid(size_t units) {
    const unsigned sms = (unsigned)device_info().sms;
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
    if ((reinterpret_cast<uintptr_t>(d_q) & 3u) || (reinterpret_cast<uintptr_t>(d_out) & 7u) ||
        (reinterpret_cast<uintptr_t>(d_workspace) & 15u))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention buffers are misaligned");
    if (!d_workspace || workspace_bytes < hsb_kv_attention_workspace_bytes(batch, pages->kv_heads))
        return record_error(HSB_E_WORKSPACE, "paged KV attention workspace missing or too small");
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
    const unsigned grid = paged_attention_grid(batch * table_width * pages->kv_heads);
    cudaError_t e = launch_format<float, true>(pages->format, p, grid, s);
    if (e == cudaSuccess)
        e = launch_dependent(kv_combine_kernel, dim3(grid), dim3(kGroup * kDim), 0, s, false,
                             static_cast<const float*>(p.part), static_cast<const RunInfo*>(p.info), p.out);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV attention launch");
    record_error(HSB_OK, "");
    return HSB_OK;
}

}  // extern "C"
