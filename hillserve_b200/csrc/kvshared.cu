// kvshared.cu -- decode attention of a batch whose sequences share a prefix.
#include <algorithm>

#include "kvattention.cuh"

namespace hsb {
namespace {

// Partial results of one run: `n` of them, from the stretches first, first + 1, ...
struct Source {
    const float* part;
    const float* whole;
    uint32_t units;
    unsigned ctas;
};

struct SharedCombine {
    Source prefix, own;
    uint32_t prefix_units;
    const uint32_t* cum;
    unsigned long long batch;
    int heads;
    uint16_t* out;
};

__device__ __forceinline__ void fold(const Source& s, unsigned long long run, unsigned long long begin,
                                     unsigned long long pages, int h, int d, float& M, float& L, float& acc) {
    if (!pages) return;
    const Split split(s.units, s.ctas);
    const unsigned first = split.of((uint32_t)begin), last = split.of((uint32_t)(begin + pages - 1));
    for (unsigned c = first; c <= last; ++c) {
        const float* slot = first == last ? s.whole + run * kPartFloats
                                          : s.part + ((size_t)c * 2 + (c == first)) * kPartFloats;
        const float m = __ldcg(slot + 2 * h), l = __ldcg(slot + 2 * h + 1);
        const float v = __ldcg(slot + 2 * kGroup + h * kDim + d);
        if (m == -INFINITY && l == l) continue;
        const float top = fmaxf(M, m), a = M == -INFINITY ? 0.0f : exp2f(M - top), b = top == -INFINITY ? 1.0f : exp2f(m - top);
        L = L * a + l * b;
        acc = acc * a + v * b;
        M = top;
    }
}

__global__ void __launch_bounds__(kGroup* kDim) kv_shared_combine_kernel(const __grid_constant__ SharedCombine p) {
    pdl_wait();
    pdl_trigger();
    const unsigned long long run = blockIdx.x, seq = run / p.heads;
    const int head = (int)(run % p.heads), h = threadIdx.x / kDim, d = threadIdx.x % kDim;
    float M = -INFINITY, L = 0.0f, acc = 0.0f;
    Source p_own = p.own;
    fold(p.prefix, run, run * p.prefix_units, p.prefix_units, h, d, M, L, acc);
    const unsigned long long pages = p.cum[seq + 1] - p.cum[seq];
    p_own.units = p.cum[p.batch] * p.heads;
    fold(p_own, run, p.cum[seq] * p.heads + head * pages, pages, h, d, M, L, acc);
    p.out[(run * kGroup + h) * kDim + d] = __half_as_ushort(__float2half_rn(L > 0.0f ? acc / L : (L == L ? 0.0f : L)));
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }
struct Layout {
    size_t info, part, whole, total;
};
Layout layout_of(size_t batch, int heads) {
    Layout l{};
    l.info = align256((batch + 1) * 8);
    l.part = l.info + align256(kAttnMaxCtas * sizeof(RunInfo));
    l.whole = l.part + align256((size_t)kAttnMaxCtas * 2 * kPartFloats * 4);
    l.total = l.whole + align256(batch * heads * kPartFloats * 4);
    return l;
}

}  // namespace
}  // namespace hsb

using namespace hsb;

extern "C" {

size_t hsb_kv_attention_shared_workspace_bytes(size_t batch, int kv_heads, size_t) {
    return 2 * layout_of(batch, kv_heads).total;
}

int hsb_kv_attention_shared(const hsb_kv_pages* prefix, const int32_t* d_prefix_table, size_t prefix_tokens,
                            const hsb_kv_pages* pages, const int32_t* d_table, size_t table_width,
                            const int32_t* d_lengths, size_t batch, const uint16_t* d_q, uint16_t* d_out,
                            void* d_workspace, size_t workspace_bytes, hsb_device_status* d_status, void* stream) {
    if (!kv_pages_valid(prefix) || !kv_pages_valid(pages)) return record_error(HSB_E_KV_SHAPE, "paged KV pool arguments");
    if (prefix->format != HSB_KV_F16 || prefix->kv_heads != pages->kv_heads)
        return record_error(HSB_E_KV_SHAPE, "a shared prefix is an F16 pool of the same KV heads");
    if (!d_prefix_table || !prefix_tokens || prefix_tokens > kMaxTableEntries || !d_table || !table_width ||
        table_width > kMaxTableEntries || !d_lengths || !batch || batch > kMaxBatch ||
        batch * table_width > kMaxTableEntries || !d_q || !d_out)
        return record_error(HSB_E_KV_SHAPE, "paged KV attention shape");
    if (((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_workspace)) & 15u) ||
        (reinterpret_cast<uintptr_t>(d_out) & 7u))
        return record_error(HSB_E_KV_SHAPE, "paged KV attention buffers are misaligned");
    if (!d_workspace || workspace_bytes < hsb_kv_attention_shared_workspace_bytes(batch, pages->kv_heads, prefix_tokens))
        return record_error(HSB_E_WORKSPACE, "paged KV attention workspace missing or too small");
    const Layout l = layout_of(batch, pages->kv_heads);
    const size_t prefix_pages = (prefix_tokens + kPageTokens - 1) / kPageTokens;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    SharedCombine c{};
    for (int which = 0; which < 2; ++which) {
        unsigned char* ws = static_cast<unsigned char*>(d_workspace) + which * l.total;
        PagedAttention p{};
        p.v = which ? paged_view(*pages, d_table, table_width, table_width)
                    : paged_view(*prefix, d_prefix_table, prefix_pages, 0);
        p.lengths = which ? d_lengths : nullptr;
        p.length = prefix_tokens;
        p.batch = batch;
        p.q = d_q;
        p.cum = reinterpret_cast<uint32_t*>(ws);
        p.info = reinterpret_cast<RunInfo*>(ws + l.info);
        p.part = reinterpret_cast<float*>(ws + l.part);
        p.whole = reinterpret_cast<float*>(ws + l.whole);
        p.status = d_status;
        p.scale_log2 = kScaleLog2;
        const unsigned grid = paged_attention_grid(2 * batch * pages->kv_heads * p.v.width);
        cudaError_t e = launch_paged_partials(which ? pages->format : HSB_KV_F16, p, grid, s);
        if (e != cudaSuccess) return record_cuda_error(e, "paged KV attention launch");
        Source& src = which ? c.own : c.prefix;
        src.part = p.part;
        src.whole = p.whole;
        src.units = which ? 0 : batch * pages->kv_heads * ((prefix_tokens + 31) / 32);
        src.ctas = grid;
        c.cum = p.cum;
    }
    c.prefix_units = (prefix_tokens + 31) / 32;
    c.batch = batch;
    c.heads = pages->kv_heads;
    c.out = d_out;
    cudaError_t e = launch_dependent(kv_shared_combine_kernel, dim3((unsigned)(batch * pages->kv_heads)),
                                     dim3(kGroup * kDim), 0, s, false, c);
    if (e != cudaSuccess) return record_cuda_error(e, "paged KV attention launch");
    record_error(HSB_OK, "");
    return HSB_OK;
}

}  // extern "C"
