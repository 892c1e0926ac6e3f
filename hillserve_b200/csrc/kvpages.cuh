// kvpages.cuh -- the paged KV cache's layout, shared by the kernels that
// write, read and attend over it.
//
// A pool is [pages][kv_heads] blocks.  A block holds 64 tokens of one KV head:
// K panels, V panels, and in the 8-bit formats the F32 scales K[64], V[64].  A
// panel is 64 rows (tokens) of 128 bytes whose 16-byte chunk c lies at place
// c ^ (row & 7): F16 needs two panels (channels 0-63, 64-127), 8 bits one.
//
// The order is the tensor core's 128-byte swizzle, so one untiled bulk copy of
// a panel is an MMA operand, and fragment loads from a staged block touch all
// 32 banks (8 lanes = 2 rows x 4 chunks, or 4 rows x 2 chunks, never share a
// 16-byte place modulo 128 bytes).  One block is one contiguous copy, whatever
// the page's place: no tensor map, no gather inside a page.
#pragma once
#include "common.cuh"
#include "internal.h"

namespace hsb {

constexpr int kPageTokens = 64;
constexpr int kPanelBytes = kPageTokens * 128;

template <int F>
struct PageFormat {
    static constexpr bool kScaled = F != HSB_KV_F16;
    static constexpr int kPanels = kScaled ? 1 : 2;  // per K or V
    static constexpr int kScaleOffset = 2 * kPanels * kPanelBytes;
    static constexpr int kBytes = kScaleOffset + (kScaled ? 2 * kPageTokens * 4 : 0);
    static constexpr float kTop = F == HSB_KV_INT8 ? 127.0f : 448.0f;  // the largest code
};

// Kernel-side view of a pool and its page tables.
struct PagedView {
    unsigned char* data;
    unsigned long long pages;
    int heads;
    const int32_t* table;           // [batch][pitch]
    unsigned long long width;       // entries of a sequence
    unsigned long long pitch;       // entries from one sequence to the next
};

// The pool page of a sequence's position, -1 (with a status) where the table
// has none: a position behind the table's end or an entry outside the pool.
__device__ __forceinline__ long long page_of(const PagedView& v, unsigned long long seq, unsigned long long pos,
                                             hsb_device_status* status, int index) {
    if (pos / kPageTokens >= v.width) {
        raise_status(status, HSB_E_KV_POSITION, index);
        return -1;
    }
    const int32_t page = v.table[seq * v.pitch + pos / kPageTokens];
    if (page < 0 || (unsigned long long)page >= v.pages) {
        raise_status(status, HSB_E_KV_PAGE, index);
        return -1;
    }
    return page;
}

// Two e4m3 codes (low 16 bits) as two F16 values, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((unsigned short)codes));
    return d;
}
// The same for int8 codes: byte b ^ 0x80 = b + 128 in the low mantissa bits
// under 0x64 is the F16 number 1024 + 128 + b, so one subtraction is exact.
__device__ __forceinline__ uint32_t biased_to_half2(uint32_t biased, uint32_t select) {
    const uint32_t h = __byte_perm(biased, 0x64646464u, select);
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&d);
}
// Four codes of one word as F16 pairs (bytes 0, 1) and (2, 3).
template <int F>
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (F == HSB_KV_E4M3) {
        lo = e4m3x2_to_half2(w & 0xffffu);
        hi = e4m3x2_to_half2(w >> 16);
    } else {
        const uint32_t b = w ^ 0x80808080u;
        lo = biased_to_half2(b, 0x4140);
        hi = biased_to_half2(b, 0x4342);
    }
}

bool kv_pages_valid(const hsb_kv_pages* p);
// Whether each of these addresses (null ones too) is a multiple of `by`.
template <typename... P>
bool aligned_to(uintptr_t by, const P*... at) {
    return ((... | reinterpret_cast<uintptr_t>(at)) & (by - 1)) == 0;
}
// Whether two ranges have no byte in common.
inline bool apart(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y ? y - x >= a_bytes : x - y >= b_bytes;
}
PagedView paged_view(const hsb_kv_pages& p, const int32_t* table, size_t width, size_t pitch);

}  // namespace hsb
