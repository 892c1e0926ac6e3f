// kvpages.cu -- writing K/V rows into the paged cache (quantised as they are
// written) and reading them back as F16 rows.
#include <cuda_fp8.h>

#include <algorithm>

#include "kvpages.cuh"

namespace hsb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// ------------------------------------------------------------------- write
// Of each (token, K or V, head) vector of 128 channels, with top = 127 (int8)
// or 448 (e4m3): scale = max|x| / top, code = round(x * (top / max|x|)), both
// quotients and the product rounded once in F32, codes to nearest even.
struct AppendParams {
    PagedView v;
    const int32_t* starts;   // [batch]
    const int32_t* offsets;  // [batch + 1], or null: row i is sequence i's
    const uint16_t* k;
    const uint16_t* x;       // V
    unsigned long long row_stride, head_stride;  // words
    unsigned long long batch, rows;
    hsb_device_status* status;
};

// The last sequence whose first row is <= row; -1 for a row of none.
__device__ __forceinline__ long long sequence_of(const int32_t* offsets, unsigned long long batch, long long row) {
    if (row >= offsets[batch] || row < offsets[0]) return -1;
    unsigned long long first = 0, n = batch;
    while (n > 1) {
        const unsigned long long half = n / 2;
        if (offsets[first + half] <= row) {
            first += half;
            n -= half;
        } else {
            n = half;
        }
    }
    return (long long)first;
}

// Eight F16 values (four words) as codes; `inv` = top / max|x|.  Finite: the
// products lie within the range up to one rounding, which the conversions end.
template <int F>
__device__ __forceinline__ uint2 codes_of(const uint32_t (&w)[4], float inv) {
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w[2 * i]));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w[2 * i + 1]));
        const float y[4] = {__fmul_rn(a.x, inv), __fmul_rn(a.y, inv), __fmul_rn(b.x, inv), __fmul_rn(b.y, inv)};
        if constexpr (F == HSB_KV_INT8) {
            // adding 1.5 2^23 rounds to the nearest integer, ties to even, in the low byte
            constexpr float kRound = 12582912.0f;
            uint32_t r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = __float_as_uint(__fadd_rn(y[j], kRound));
            c[i] = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
        } else {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
            c[i] = lo | (hi << 16);
        }
    }
    return make_uint2(c[0], c[1]);
}
// The same with NaN (code 0) or infinities (the end of the range) among the values.
template <int F>
__device__ uint2 codes_of_nonfinite(const uint32_t (&w)[4], float inv) {
    constexpr float kTop = PageFormat<F>::kTop;
    uint32_t c[2] = {0, 0};
    for (int i = 0; i < 8; ++i) {
        const float x = half_value((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
        float y = __fmul_rn(x, inv);
        y = y == y ? fminf(fmaxf(y, -kTop), kTop) : 0.0f;
        uint32_t code;
        if constexpr (F == HSB_KV_INT8) code = (uint32_t)__float2int_rn(y) & 0xffu;
        else code = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
        c[i >> 2] |= code << (8 * (i & 3));
    }
    return make_uint2(c[0], c[1]);
}

// A CTA takes `per` rows: one lane a row looks its page up while the first
// rows are already being loaded.  A warp then takes U heads of a row at a
// time: half-warp 0 the K vector, half-warp 1 the V vector, a lane 8 channels.
// Bound by memory and, in 8 bits, by the issue slots (71 % busy): 32768 e4m3 rows of
// 8 heads, 134 MB read and 69 MB written, take 33 us, 6.2 TB/s.  Look-ups by every
// warp for itself (four dependent loads before each store) took 73 us.
constexpr int kMostRows = 32;
template <int F, int U>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ AppendParams p, const int per) {
    using Fmt = PageFormat<F>;
    __shared__ long long place[kMostRows];  // page x 64 + row in it; -1: nowhere
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = lane >> 4, l = lane & 15;
    const int shift = 31 - __clz(p.v.heads / U), mask = (1 << shift) - 1;  // of a row's groups of heads
    const unsigned long long row0 = (unsigned long long)blockIdx.x * per;
    const int items = (int)min((unsigned long long)per, p.rows - row0) << shift;
    const uint16_t* const src = (part ? p.x : p.k) + l * 8;
    uint4 next[U];
    const auto load = [&](int item) {
        const uint16_t* at = src + (row0 + (item >> shift)) * p.row_stride + (item & mask) * U * p.head_stride;
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = __ldcs(reinterpret_cast<const uint4*>(at + u * p.head_stride));
    };
    if (warp < items) load(warp);
    if (threadIdx.x < per && row0 + threadIdx.x < p.rows) {
        const long long row = (long long)(row0 + threadIdx.x);
        long long seq = row, first = row, at = -1;
        if (p.offsets) {
            seq = sequence_of(p.offsets, p.batch, row);
            if (seq >= 0) first = p.offsets[seq];
        }
        const int32_t start = seq >= 0 ? p.starts[seq] : 0;
        if (start < 0) {  // (no position at all, however wide the table)
            raise_status(p.status, HSB_E_KV_POSITION, (int)row);
        } else if (seq >= 0) {
            const unsigned long long pos = (unsigned long long)start + (unsigned long long)(row - first);
            const long long page = page_of(p.v, seq, pos, p.status, (int)row);
            if (page >= 0) at = page * kPageTokens + (long long)(pos % kPageTokens);
        }
        place[threadIdx.x] = at;
    }
    __syncthreads();
    for (int item = warp; item < items; item += kWarps) {
        uint32_t w[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            w[u][0] = next[u].x;
            w[u][1] = next[u].y;
            w[u][2] = next[u].z;
            w[u][3] = next[u].w;
        }
        if (item + kWarps < items) load(item + kWarps);
        const long long at = place[item >> shift];
        if (at < 0) continue;
        const int r = (int)(at % kPageTokens), h0 = (item & mask) * U;
        unsigned char* const block = p.v.data + ((size_t)(at / kPageTokens) * p.v.heads + h0) * Fmt::kBytes;
        uint32_t top[U], most = 0;  // the largest magnitudes' bits (F16 orders as integers)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t m2 = __vmaxu2(__vmaxu2(w[u][0] & 0x7fff7fffu, w[u][1] & 0x7fff7fffu),
                                         __vmaxu2(w[u][2] & 0x7fff7fffu, w[u][3] & 0x7fff7fffu));
            top[u] = max(m2 & 0xffffu, m2 >> 16);
            most = max(most, top[u]);
        }
        const bool odd = __any_sync(0xffffffffu, most >= 0x7c00u);
        if (odd) {
            if (lane == 0) raise_status(p.status, HSB_E_EXECUTOR_NONFINITE_KV, (int)(row0 + (item >> shift)));
            // the largest finite magnitude: NaN and infinity do not set the scale
#pragma unroll
            for (int u = 0; u < U; ++u) {
                top[u] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a = w[u][i] & 0x7fffu, b = (w[u][i] >> 16) & 0x7fffu;
                    top[u] = max(top[u], max(a < 0x7c00u ? a : 0u, b < 0x7c00u ? b : 0u));
                }
            }
        }
        if constexpr (!Fmt::kScaled) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                unsigned char* panel = block + (size_t)u * Fmt::kBytes + (part * 2 + (l >> 3)) * kPanelBytes;
                *reinterpret_cast<uint4*>(panel + r * 128 + (((l & 7) ^ (r & 7)) << 4)) =
                    make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
            }
        } else {
            // a vector's maximum over its 16 lanes; of four vectors, lanes 4 u .. 4 u + 3 of the half-warp end
            // with vector u's, so each quotient is formed once
            static_assert(U == 1 || U == 4, "one vector a half-warp, or four");
            uint32_t mine;
            if constexpr (U == 4) {
                const bool b3 = l & 8, b2 = l & 4;
                const uint32_t x0 = max(b3 ? top[2] : top[0], __shfl_xor_sync(0xffffffffu, b3 ? top[0] : top[2], 8));
                const uint32_t x1 = max(b3 ? top[3] : top[1], __shfl_xor_sync(0xffffffffu, b3 ? top[1] : top[3], 8));
                mine = max(b2 ? x1 : x0, __shfl_xor_sync(0xffffffffu, b2 ? x0 : x1, 4));
            } else {
                mine = max(top[0], __shfl_xor_sync(0xffffffffu, top[0], 8));
                mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 4));
            }
            mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
            mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
            const float amax = half_value((uint16_t)mine);
            const float inv = mine ? __fdiv_rn(Fmt::kTop, amax) : 0.0f;
            const int owner = U == 4 ? l >> 2 : 0;
            if ((U == 4 ? l & 3 : l) == 0)
                reinterpret_cast<float*>(block + (size_t)owner * Fmt::kBytes + Fmt::kScaleOffset)[part * kPageTokens + r] =
                    __fdiv_rn(amax, Fmt::kTop);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float by = __shfl_sync(0xffffffffu, inv, (lane & 16) + 4 * u);
                const uint2 code = odd ? codes_of_nonfinite<F>(w[u], by) : codes_of<F>(w[u], by);
                unsigned char* panel = block + (size_t)u * Fmt::kBytes + part * kPanelBytes;
                *reinterpret_cast<uint2*>(panel + r * 128 + (((l >> 1) ^ (r & 7)) << 4) + (l & 1) * 8) = code;
            }
        }
    }
}

// -------------------------------------------------------------------- read
struct ReadParams {
    PagedView v;
    const int32_t* seqs;       // or null: sequence 0
    const uint32_t* positions;
    const uint32_t* count;     // device, or null: max_rows
    unsigned long long batch, max_rows;
    uint16_t* out;             // [max_rows][2][heads][128]
    hsb_device_status* status;
};

// A warp takes U heads of a row, half-warp 0 their K, half-warp 1 their V, a lane 8
// channels.  Bound by memory: 32768 e4m3 rows, 69 MB read and 134 MB written, 33 us,
// 6.1 TB/s; 6553 int8 rows 6.9 us, 5.9 TB/s; 77 rows 1.7 us, the launch.
template <int F, int U>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadParams p) {
    using Fmt = PageFormat<F>;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, part = lane >> 4, l = lane & 15;
    const unsigned groups = p.v.heads / U;
    const unsigned long long item = (unsigned long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const unsigned long long i = item / groups;
    const int h0 = (int)(item % groups) * U;
    if (i >= p.max_rows || (p.count && i >= *p.count)) return;
    const unsigned long long seq = p.seqs ? (uint32_t)p.seqs[i] : 0;
    const unsigned long long pos = p.positions[i];
    long long page = -1;
    if (seq >= p.batch) raise_status(p.status, HSB_E_KV_POSITION, (int)i);
    else page = page_of(p.v, seq, pos, p.status, (int)i);
    uint16_t* dst = p.out + ((i * 2 + part) * p.v.heads + h0) * kDim + l * 8;
    if (page < 0) {  // no such row: zeros
#pragma unroll
        for (int u = 0; u < U; ++u) *reinterpret_cast<uint4*>(dst + u * kDim) = make_uint4(0, 0, 0, 0);
        return;
    }
    const int r = (int)(pos % kPageTokens);
    const unsigned char* block = p.v.data + ((size_t)page * p.v.heads + h0) * Fmt::kBytes;
    if constexpr (!Fmt::kScaled) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            w[u] = __ldcs(reinterpret_cast<const uint4*>(block + (size_t)u * Fmt::kBytes +
                                                         (part * 2 + (l >> 3)) * kPanelBytes + r * 128 +
                                                         (((l & 7) ^ (r & 7)) << 4)));
#pragma unroll
        for (int u = 0; u < U; ++u) *reinterpret_cast<uint4*>(dst + u * kDim) = w[u];
    } else {
        uint2 c[U];
        float scale[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned char* b = block + (size_t)u * Fmt::kBytes;
            c[u] = __ldcs(reinterpret_cast<const uint2*>(b + part * kPanelBytes + r * 128 +
                                                         (((l >> 1) ^ (r & 7)) << 4) + (l & 1) * 8));
            scale[u] = reinterpret_cast<const float*>(b + Fmt::kScaleOffset)[part * kPageTokens + r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t h[4], o[4];
            codes_to_half2<F>(c[u].x, h[0], h[1]);
            codes_to_half2<F>(c[u].y, h[2], h[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
                const __half2 v = __floats2half2_rn(f.x * scale[u], f.y * scale[u]);
                o[e] = *reinterpret_cast<const uint32_t*>(&v);
            }
            *reinterpret_cast<uint4*>(dst + u * kDim) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// Four heads a warp keep more loads in flight; one head a warp spreads a few
// rows over more SMs.  Of 8 heads, four and one a warp: 256 e4m3 rows written in
// 2.6 and 2.5 us, read in 2.1 and 2.0; 1024 in 3.6 and 3.9, 3.0 and 3.5; 4096 in
// 7.5 and 9.4, 6.3 and 8.5 (F16 alike, but for 1024 written in 3.7 and 3.3).
constexpr unsigned long long kWideRows = 1024;

template <int F>
cudaError_t run_append(const AppendParams& p, cudaStream_t stream) {
    const bool wide = p.v.heads % 4 == 0 && p.rows >= kWideRows;
    // as many rows a CTA as still leave eight CTAs to each SM, of the 8 warps' worth at least
    const unsigned long long fill = p.rows / (8ull * device_info().sms);
    const int least = std::max(1, kWarps / (p.v.heads / (wide ? 4 : 1)));
    const int per = (int)std::min<unsigned long long>(kMostRows, std::max<unsigned long long>(least, fill));
    const dim3 grid((unsigned)((p.rows + per - 1) / per));
    return wide ? launch_dependent(kv_append_kernel<F, 4>, grid, dim3(kThreads), 0, stream, false, p, per)
                : launch_dependent(kv_append_kernel<F, 1>, grid, dim3(kThreads), 0, stream, false, p, per);
}
template <int F>
cudaError_t run_read(const ReadParams& p, cudaStream_t stream) {
    const bool wide = p.v.heads % 4 == 0 && p.max_rows >= kWideRows;
    const unsigned long long items = p.max_rows * (p.v.heads / (wide ? 4 : 1));
    const dim3 grid((unsigned)((items + kWarps - 1) / kWarps));
    return wide ? launch_dependent(kv_read_kernel<F, 4>, grid, dim3(kThreads), 0, stream, false, p)
                : launch_dependent(kv_read_kernel<F, 1>, grid, dim3(kThreads), 0, stream, false, p);
}

// Grid limit: 2^31 - 1 blocks of 8 warps, at most 8 warps (heads) a row.
constexpr size_t kMaxRows = 0x7fffffffull;

}  // namespace

bool kv_pages_valid(const hsb_kv_pages* p) {
    return p && p->data && p->pages && p->pages <= 0x7fffffffull && hsb_kv_page_bytes(p->format) &&
           (p->kv_heads == 1 || p->kv_heads == 2 || p->kv_heads == 4 || p->kv_heads == 8) &&
           (reinterpret_cast<uintptr_t>(p->data) & 15u) == 0;
}

PagedView paged_view(const hsb_kv_pages& p, const int32_t* table, size_t width, size_t pitch) {
    PagedView v{};
    v.data = static_cast<unsigned char*>(p.data);
    v.pages = p.pages;
    v.heads = p.kv_heads;
    v.table = table;
    v.width = width;
    v.pitch = pitch;
    return v;
}

}  // namespace hsb

using namespace hsb;

extern "C" {

size_t hsb_kv_page_bytes(int format) {
    switch (format) {
    case HSB_KV_F16: return PageFormat<HSB_KV_F16>::kBytes;
    case HSB_KV_INT8: return PageFormat<HSB_KV_INT8>::kBytes;
    case HSB_KV_E4M3: return PageFormat<HSB_KV_E4M3>::kBytes;
    default: return 0;
    }
}

int hsb_kv_append(const hsb_kv_pages* pages, const int32_t* d_table, size_t table_width, size_t batch,
                  const int32_t* d_starts, const int32_t* d_offsets, const uint16_t* d_k, const uint16_t* d_v,
                  size_t rows, size_t row_stride, size_t head_stride, hsb_device_status* d_status, void* stream) {
    if (!kv_pages_valid(pages)) return record_error(HSB_E_KV_SHAPE, "paged KV pool arguments");
    if (!d_table || !table_width || !batch || !d_starts || !d_k || !d_v || !rows || rows > kMaxRows ||
        (!d_offsets && rows != batch))
        return record_error(HSB_E_KV_SHAPE, "paged KV append shape");
    if (!aligned_to(16, d_k, d_v) || row_stride % 8 || head_stride % 8)
        return record_error(HSB_E_KV_SHAPE, "paged KV rows must be 16-byte aligned");
    if (!aligned_to(4, d_table, d_starts, d_offsets) || !aligned_to(8, d_status))
        return record_error(HSB_E_KV_SHAPE, "paged KV tables are misaligned");
    AppendParams p{};
    p.v = paged_view(*pages, d_table, table_width, table_width);
    p.starts = d_starts;
    p.offsets = d_offsets;
    p.k = d_k;
    p.x = d_v;
    p.row_stride = row_stride;
    p.head_stride = head_stride;
    p.batch = batch;
    p.rows = rows;
    p.status = d_status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = pages->format == HSB_KV_F16    ? run_append<HSB_KV_F16>(p, s)
                    : pages->format == HSB_KV_INT8 ? run_append<HSB_KV_INT8>(p, s)
                                                   : run_append<HSB_KV_E4M3>(p, s);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV append launch");
    record_error(HSB_OK, "");
    return HSB_OK;
}

int hsb_kv_read(const hsb_kv_pages* pages, const int32_t* d_table, size_t table_width, size_t batch,
                const int32_t* d_seqs, const uint32_t* d_positions, const uint32_t* d_count, size_t max_rows,
                uint16_t* d_out, hsb_device_status* d_status, void* stream) {
    if (!kv_pages_valid(pages)) return record_error(HSB_E_KV_SHAPE, "paged KV pool arguments");
    if (!d_table || !table_width || !batch || !d_positions || !d_out || !max_rows || max_rows > kMaxRows)
        return record_error(HSB_E_KV_SHAPE, "paged KV read shape");
    if (!aligned_to(16, d_out)) return record_error(HSB_E_KV_SHAPE, "paged KV rows must be 16-byte aligned");
    if (!aligned_to(4, d_table, d_seqs, d_positions, d_count) || !aligned_to(8, d_status))
        return record_error(HSB_E_KV_SHAPE, "paged KV tables are misaligned");
    ReadParams p{};
    p.v = paged_view(*pages, d_table, table_width, table_width);
    p.seqs = d_seqs;
    p.positions = d_positions;
    p.count = d_count;
    p.batch = batch;
    p.max_rows = max_rows;
    p.out = d_out;
    p.status = d_status;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = pages->format == HSB_KV_F16    ? run_read<HSB_KV_F16>(p, s)
                    : pages->format == HSB_KV_INT8 ? run_read<HSB_KV_INT8>(p, s)
                                                   : run_read<HSB_KV_E4M3>(p, s);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV read launch");
    record_error(HSB_OK, "");
    return HSB_OK;
}

}  // extern "C"
