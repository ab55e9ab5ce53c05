// What the kernels of attention over pages share: a document's queries and keys,
// clamped to the tensors whatever the device arrays hold; blocks of 16 keys of a
// page as buffers; matrix core operands from them.
//
// Products here run on 16 x 16 tiles: of C[row][col], lane l holds column l % 16,
// rows 4 (l / 16) + r. An operand's lane has row (A) or column (B) l % 16 and,
// of the contraction, a quarter's share: quarter c = l / 16. Which elements a
// quarter has is free as long as A and B agree, and so is which channel or key
// has which row, so nothing moves between lanes:
//   S^T = K Q^T    A: a key's channels as loaded, B: the same channels of a query
//   O^T += V^T P^T B: the probabilities as S^T leaves them, a quarter's keys
//                  being 4 c + r of each block of 16; A: those keys' rows, each
//                  lane's neighbouring channels one to a product.
#pragma once

#include "packed_device.hpp"

namespace bl {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// ---- documents ----

struct PagedDocument {
    int q0, n_q;
    int n_k, shift;  // query i stands at key i + shift
    int index;
};

__device__ __forceinline__ PagedDocument paged_document(const bl_paged_attention_args &a, int d) {
    PagedDocument doc;
    const int rows = (int)a.q_rows;
    doc.index = d;
    doc.q0 = uniform(a.q_offsets ? min(max(a.q_offsets[d], 0), rows) : 0);
    doc.n_q = uniform(max((a.q_offsets ? min(max(a.q_offsets[d + 1], 0), rows) : rows) - doc.q0, 0));
    doc.n_k = uniform(min(max(a.cache.lengths[d], 0), (int)(a.cache.max_pages * a.cache.page_rows)));
    doc.shift = doc.n_k - doc.n_q;
    return doc;
}
// Query i sees keys [from, to).
__device__ __forceinline__ int keys_to(const bl_paged_attention_args &a, const PagedDocument &doc, int i) {
    return a.mask == BL_MASK_NONE ? doc.n_k : min(doc.n_k, max(i + doc.shift + 1, 0));
}
__device__ __forceinline__ int keys_from(const bl_paged_attention_args &a, const PagedDocument &doc, int i) {
    return a.window ? (int)max((int64_t)0, (int64_t)i + doc.shift + 1 - (int64_t)a.window) : 0;
}

// ---- blocks of 16 keys ----

// The keys j .. j + 15 of a document (j a multiple of 16, so of one page) and a
// key head: what is there of them, 0 to 16, and of k's or v's rows a buffer that
// ends behind the last: the rest, and channels a lane puts outside, arrive as
// zeros.
struct KeyBlock {
    int page, row, there;
    __device__ __forceinline__ KeyBlock(const bl_paged_cache &cache, const int32_t *table, uint32_t magic, int j, int end) {
        const int n = (int)__umulhi((uint32_t)j, magic);  // j / page_rows
        row = j - n * (int)cache.page_rows;
        there = min(max(end - j, 0), 16);
        page = there > 0 ? uniform(table[n]) : -1;
        if ((uint32_t)page >= cache.pages) there = 0;
    }
    __device__ __forceinline__ uint64_t address(const bl_pages &p, uint32_t head) const {
        return (uint64_t)p.data + (uint64_t)(there > 0 ? page : 0) * p.page_stride + (uint64_t)row * p.row_stride + (uint64_t)head * p.head_stride;
    }
    __device__ __forceinline__ int bytes(const bl_pages &p, int width) const { return there > 0 ? (there - 1) * (int)p.row_stride + width : 0; }
};

constexpr uint32_t OUTSIDE = 0x7ffffff0u;

#ifdef __HIP_DEVICE_COMPILE__  // the host pass knows no buffers
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(uint64_t address, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)uniform64(address), 0, uniform(bytes), 0x00020000);
}
__device__ __forceinline__ u32x4 fetch16(Buffer b, uint32_t offset) { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0)); }
__device__ __forceinline__ u32x2 fetch8(Buffer b, uint32_t offset) { return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(b, offset, 0, 0)); }
__device__ __forceinline__ uint32_t fetch4(Buffer b, uint32_t offset) { return __builtin_amdgcn_raw_buffer_load_b32(b, offset, 0, 0); }
#else
typedef int Buffer;
__device__ inline Buffer buffer_of(uint64_t, int) { return 0; }
__device__ inline u32x4 fetch16(Buffer, uint32_t) { return u32x4{}; }
__device__ inline u32x2 fetch8(Buffer, uint32_t) { return u32x2{}; }
__device__ inline uint32_t fetch4(Buffer, uint32_t) { return 0; }
#endif

// ---- operands ----

__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// The low (N 0) or high halves of a and b side by side.
template <int N> __device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, N == 0 ? 0x05040100u : 0x07060302u); }

// Four pairs of codes, one of each half of w: f16 1024 + code and 64 + code are a
// code under an exponent whose last place is 1, or 1/16 for the code's place in
// bits 4 .. 7; less 1024 or 64 they are the code, exactly, and low + code step
// rounds once.
__device__ __forceinline__ f16x2 value_of(uint32_t w, uint32_t mask, uint32_t under, f16x2 less, f16x2 step, f16x2 low) {
    const f16x2 code = __builtin_bit_cast(f16x2, (w & mask) | under) - less;
    return __builtin_elementwise_fma(code, step, low);
}
template <int N> __device__ __forceinline__ void values_of(uint32_t w, f16x2 step, f16x2 low, f16x2 (&v)[N]) {
    const f16x2 kilo = {(_Float16)1024.0f, (_Float16)1024.0f}, some = {(_Float16)64.0f, (_Float16)64.0f};
#pragma unroll
    for (int n = 0; n < N; n += 2) {
        v[n] = value_of(w >> (4 * n), 0x000f000fu, 0x64006400u, kilo, step, low);
        v[n + 1] = value_of(w >> (4 * n), 0x00f000f0u, 0x54005400u, some, step, low);
    }
}

__device__ __forceinline__ f16x2 both(uint32_t bits) { return __builtin_bit_cast(f16x2, bits); }

}  // namespace bl
