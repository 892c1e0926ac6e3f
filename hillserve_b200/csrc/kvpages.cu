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

// The last sequence whose first row is <= row; -1 for a row of none.  The
// lanes probe 32 places at once: two rounds for 1024 sequences.
__device__ __forceinline__ long long sequence_of(const int32_t* offsets, unsigned long long batch, long long row) {
    const int lane = threadIdx.x & 31;
    if (row >= offsets[batch]) return -1;
    unsigned long long first = 0, n = batch;
    while (true) {
        const unsigned long long step = (n + 31) / 32;
        const unsigned long long at = lane * step;
        const unsigned under = __ballot_sync(0xffffffffu, at < n && offsets[first + at] <= row);
        if (!under) return -1;
        const unsigned long long skip = (31 - __clz(under)) * step;
        first += skip;
        n = min(step, n - skip);
        if (step == 1) return (long long)first;
    }
}

// A warp takes U heads of a row; half-warp 0 the K vector, half-warp 1 the V
// vector, a lane 8 channels (one 16-byte load).
template <int F, int U>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ AppendParams p) {
    using Fmt = PageFormat<F>;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, part = lane >> 4, l = lane & 15;
    const unsigned groups = p.v.heads / U;
    const unsigned long long item = (unsigned long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const unsigned long long row = item / groups;
    const int h0 = (int)(item % groups) * U;
    if (row >= p.rows) return;
    uint4 w[U];
    const uint16_t* src = (part ? p.x : p.k) + row * p.row_stride + l * 8;
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = __ldcs(reinterpret_cast<const uint4*>(src + (h0 + u) * p.head_stride));
    long long seq = (long long)row, first = seq;
    if (p.offsets) {
        seq = sequence_of(p.offsets, p.batch, (long long)row);
        if (seq < 0) return;  // a row of no sequence
        first = p.offsets[seq];
    }
    const unsigned long long pos = (unsigned long long)(uint32_t)p.starts[seq] + (unsigned long long)(row - first);
    const long long page = page_of(p.v, seq, pos, p.status, (int)row);
    if (page < 0) return;
    const int r = (int)(pos % kPageTokens);
    bool finite = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        unsigned char* block = p.v.data + ((size_t)page * p.v.heads + h0 + u) * Fmt::kBytes;
        const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            finite &= ((words[i] & 0x7c00u) != 0x7c00u) && ((words[i] & 0x7c000000u) != 0x7c000000u);
        if constexpr (!Fmt::kScaled) {
            unsigned char* panel = block + (part * 2 + (l >> 3)) * kPanelBytes;
            *reinterpret_cast<uint4*>(panel + r * 128 + (((l & 7) ^ (r & 7)) << 4)) = w[u];
        } else {
            float f[8], top = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&words[i]));
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
                // the largest finite magnitude: NaN and infinity do not set the scale
                top = fmaxf(top, fabsf(t.x) < INFINITY ? fabsf(t.x) : 0.0f);
                top = fmaxf(top, fabsf(t.y) < INFINITY ? fabsf(t.y) : 0.0f);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float inv = top > 0.0f ? __fdiv_rn(Fmt::kTop, top) : 0.0f;
            uint32_t code[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float y = __fmul_rn(f[i], inv);
                y = y == y ? fminf(fmaxf(y, -Fmt::kTop), Fmt::kTop) : 0.0f;  // NaN: 0, infinity: the end of the range
                uint32_t c;
                if constexpr (F == HSB_KV_INT8) c = (uint32_t)__float2int_rn(y) & 0xffu;
                else c = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
                code[i >> 2] |= c << (8 * (i & 3));
            }
            unsigned char* panel = block + part * kPanelBytes;
            *reinterpret_cast<uint2*>(panel + r * 128 + (((l >> 1) ^ (r & 7)) << 4) + (l & 1) * 8) =
                make_uint2(code[0], code[1]);
            if (l == 0)
                reinterpret_cast<float*>(block + Fmt::kScaleOffset)[part * kPageTokens + r] = __fdiv_rn(top, Fmt::kTop);
        }
    }
    if (!__all_sync(0xffffffffu, finite) && lane == 0) raise_status(p.status, HSB_E_EXECUTOR_NONFINITE_KV, (int)row);
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

template <int F, int U>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadParams p) {
    using Fmt = PageFormat<F>;
    pdl_wait();
    pdl_trigger();
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
// rows over more SMs.
constexpr unsigned long long kWideRows = 2048;

template <int F>
cudaError_t run_append(const AppendParams& p, cudaStream_t stream) {
    const bool wide = p.v.heads % 4 == 0 && p.rows >= kWideRows;
    const unsigned long long items = p.rows * (p.v.heads / (wide ? 4 : 1));
    const dim3 grid((unsigned)((items + kWarps - 1) / kWarps));
    return wide ? launch_dependent(kv_append_kernel<F, 4>, grid, dim3(kThreads), 0, stream, false, p)
                : launch_dependent(kv_append_kernel<F, 1>, grid, dim3(kThreads), 0, stream, false, p);
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
    if (((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v)) & 15u) || row_stride % 8 ||
        head_stride % 8)
        return record_error(HSB_E_KV_SHAPE, "paged KV rows must be 16-byte aligned");
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
    if (reinterpret_cast<uintptr_t>(d_out) & 15u)
        return record_error(HSB_E_KV_SHAPE, "paged KV rows must be 16-byte aligned");
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
