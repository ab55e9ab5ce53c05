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
    int n_k;    // keys that the table's row has room for
    int shift;  // query i stands at key i + shift, by the whole length, as it was appended
    int index;
};

// A document's first row, rows, length and keys, whatever the arrays hold; any
// lane's own.
__device__ __forceinline__ void bounds_of(const bl_paged_attention_args &a, int d, int &q0, int &n_q, int &length, int &n_k) {
    const int rows = (int)a.q_rows;
    q0 = a.q_offsets ? min(max(a.q_offsets[d], 0), rows) : 0;
    n_q = max((a.q_offsets ? min(max(a.q_offsets[d + 1], 0), rows) : rows) - q0, 0);
    length = max(a.cache.lengths[d], 0);
    n_k = min(length, (int)(a.cache.max_pages * a.cache.page_rows));
}

// Which document and which of its tiles of `tile` places a workgroup has; tile
// -1: none. Up to 64 documents are looked at in one load, a lane each, and go in
// the order of their keys, the longest first, so that the last workgroups to
// start are short ones; more of them keep theirs, from the last.
struct Assignment {
    PagedDocument doc;
    int tile;
    __device__ __forceinline__ Assignment(const bl_paged_attention_args &a, int group, int tile_places, int slot) {
        const int documents = (int)a.documents;
        if (documents <= 64) {
            const int lane = threadIdx.x % 64;
            int q0, n_q, length, n_k;
            bounds_of(a, min(lane, documents - 1), q0, n_q, length, n_k);
            const int tiles = lane < documents ? (int)(((int64_t)n_q * group + tile_places - 1) / tile_places) : 0;
            const int cost = a.window ? (int)min((int64_t)n_k, (int64_t)n_q + a.window) : n_k;
            int first = 0;  // tiles of the documents that go before the lane's
            for (int d = 0; d < documents; d++) {
                const int other = __builtin_amdgcn_readlane(cost, d);
                first += other > cost || (other == cost && d < lane) ? __builtin_amdgcn_readlane(tiles, d) : 0;
            }
            const uint64_t found = __ballot(slot >= first && slot - first < tiles);
            const int at = found ? __builtin_ctzll(found) : 0;
            doc.index = at;
            doc.q0 = __builtin_amdgcn_readlane(q0, at);
            doc.n_q = __builtin_amdgcn_readlane(n_q, at);
            doc.n_k = __builtin_amdgcn_readlane(n_k, at);
            doc.shift = __builtin_amdgcn_readlane(length - n_q, at);
            // A causal document's last places see the most keys.
            tile = found ? __builtin_amdgcn_readlane(tiles, at) - 1 - (slot - __builtin_amdgcn_readlane(first, at)) : -1;
        } else {
            const int back = (int)slots(a.q_rows, group, tile_places, documents) - 1 - slot;
            doc.index = document_of_slot(a.q_offsets, documents, a.q_rows, group, tile_places, back);
            int length;
            bounds_of(a, doc.index, doc.q0, doc.n_q, length, doc.n_k);
            doc.q0 = uniform(doc.q0);
            doc.n_q = uniform(doc.n_q);
            doc.n_k = uniform(doc.n_k);
            doc.shift = uniform(length) - doc.n_q;
            tile = back - ((int)((int64_t)doc.q0 * group / tile_places) + doc.index);
            if ((int64_t)tile * tile_places >= (int64_t)doc.n_q * group) tile = -1;
        }
    }
};
// Query i sees keys [from, to), both within the keys that there are.
__device__ __forceinline__ int keys_to(const bl_paged_attention_args &a, const PagedDocument &doc, int i) {
    return a.mask == BL_MASK_NONE ? doc.n_k : min(doc.n_k, max(i + doc.shift + 1, 0));
}
__device__ __forceinline__ int keys_from(const bl_paged_attention_args &a, const PagedDocument &doc, int i) {
    return a.window ? (int)min((int64_t)doc.n_k, max((int64_t)0, (int64_t)i + doc.shift + 1 - (int64_t)a.window)) : 0;
}

// A workgroup's share of the tiles that its places see: equal ones, so that a
// batch of unequal documents fills the chip, and the last has what is left. A
// place has as many splits as hold some of it; one alone is the whole.
struct Share {
    int begin, end, used;
    bool mine;
    __device__ __forceinline__ Share(int tiles, int each, int split, int splits) {
        used = uniform(min(max((tiles + each - 1) / each, 1), splits));
        mine = split < used;
        begin = uniform(split * each);
        end = uniform(split == used - 1 ? tiles : begin + each);
    }
};

// ---- blocks of 16 keys ----

// Keys come in blocks of 16, j .. j + 15 of a document and a key head (j a
// multiple of 16, so of one page), k's and v's rows each a buffer that ends
// behind the last that is there: the rest, and channels that a lane puts
// outside, arrive as zeros. A block that is not there at all has no bytes.
struct BlockOf {  // of one block, in scalar registers
    uint32_t k[2], v[2];  // addresses, low and high
    int k_bytes, v_bytes;
};

// A wave's next blocks, a lane's each: table entries are loaded 64 at a time and
// 64 ahead (a step that waited for its own would take several times as long as
// its keys: 8 documents, four of 1024 queries over 1641 to 6837 keys, 566 -> 474
// us), and their addresses are made in all lanes at once, so a step reads them
// from lanes instead of multiplying strides in scalar registers.
struct BlocksAhead {
    uint64_t k, v;
    int k_bytes, v_bytes;
    int page;       // of the blocks behind those
    int taken = 0;

    // key(n): the first key of the wave's block n; none at or beyond `end`.
    template <typename Key> static __device__ __forceinline__ int load(const int32_t *table, uint32_t magic, int end, int from, Key key) {
        const int j = key(from + (int)(threadIdx.x % 64));
        return j < end ? table[__umulhi((uint32_t)j, magic)] : -1;
    }
    template <typename Key>
    __device__ __forceinline__ void make(const bl_paged_cache &c, uint32_t magic, int end, uint32_t head, int width, int of, int from, Key key) {
        const int j = key(from + (int)(threadIdx.x % 64));
        const int row = j - (int)(__umulhi((uint32_t)j, magic) * c.page_rows);
        const int there = (uint32_t)of < c.pages ? min(max(end - j, 0), 16) : 0;
        k = v = 0;
        k_bytes = v_bytes = 0;
        if (there > 0) {
            k = (uint64_t)c.k.data + (uint64_t)(uint32_t)of * c.k.page_stride + (uint64_t)(uint32_t)row * c.k.row_stride + (uint64_t)head * c.k.head_stride;
            v = (uint64_t)c.v.data + (uint64_t)(uint32_t)of * c.v.page_stride + (uint64_t)(uint32_t)row * c.v.row_stride + (uint64_t)head * c.v.head_stride;
            k_bytes = (there - 1) * (int)c.k.row_stride + width;
            v_bytes = (there - 1) * (int)c.v.row_stride + width;
        }
    }
    // `width`: bytes of a row.
    template <typename Key>
    __device__ __forceinline__ BlocksAhead(const bl_paged_cache &c, const int32_t *table, uint32_t magic, int end, uint32_t head, int width, Key key) {
        page = load(table, magic, end, 64, key);
        make(c, magic, end, head, width, load(table, magic, end, 0, key), 0, key);
    }
    // The next N blocks, N a divisor of 64.
    template <int N, typename Key>
    __device__ __forceinline__ void take(BlockOf (&b)[N], const bl_paged_cache &c, const int32_t *table, uint32_t magic, int end, uint32_t head, int width, Key key) {
        if (taken % 64 == 0 && taken) {
            make(c, magic, end, head, width, page, taken, key);
            page = load(table, magic, end, taken + 64, key);
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int at = (taken + n) % 64;
            b[n].k[0] = __builtin_amdgcn_readlane((int)(uint32_t)k, at);
            b[n].k[1] = __builtin_amdgcn_readlane((int)(uint32_t)(k >> 32), at);
            b[n].v[0] = __builtin_amdgcn_readlane((int)(uint32_t)v, at);
            b[n].v[1] = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), at);
            b[n].k_bytes = __builtin_amdgcn_readlane(k_bytes, at);
            b[n].v_bytes = __builtin_amdgcn_readlane(v_bytes, at);
        }
        taken += N;
    }
};

constexpr uint32_t OUTSIDE = 0x7ffffff0u;

#ifdef __HIP_DEVICE_COMPILE__  // the host pass knows no buffers
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const uint32_t (&address)[2], int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)((uint64_t)address[1] << 32 | address[0]), 0, bytes, 0x00020000);
}
__device__ __forceinline__ u32x4 fetch16(Buffer b, uint32_t offset) { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0)); }
__device__ __forceinline__ u32x2 fetch8(Buffer b, uint32_t offset) { return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(b, offset, 0, 0)); }
__device__ __forceinline__ uint32_t fetch4(Buffer b, uint32_t offset) { return __builtin_amdgcn_raw_buffer_load_b32(b, offset, 0, 0); }
#else
typedef int Buffer;
__device__ inline Buffer buffer_of(const uint32_t (&)[2], int) { return 0; }
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

// Whether some code of a group stands for an infinity or NaN: the last one does
// then, as what codes stand for rises or falls from low to it.
__device__ __forceinline__ bool infinite_codes(uint32_t params) {
    const f16x2 p = both(params);
    return !(__builtin_fabsf16(__builtin_fmaf16((_Float16)15.0f, p[0], p[1])) < (_Float16)INFINITY);
}

}  // namespace bl
