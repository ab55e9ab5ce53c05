// What the packed attention kernels share: a document's bounds, clamped to
// the tensors whatever the offset arrays hold, and the score of a (query,
// key) pair.
#pragma once

#include "ops_device.hpp"

namespace bl {

struct Document {
    int q0, n_q;     // first query row, query rows
    int k0, n_k;     // first key row, key rows
    int shift;       // n_k - n_q: query i stands at key i + shift
    int prefix;      // keys every query sees
};

__device__ __forceinline__ Document document_of(const bl_packed_attention_args &a, int d) {
    Document doc;
    const int q_rows = (int)a.q_rows, k_rows = (int)a.k_rows;
    doc.q0 = a.q_offsets ? min(max(a.q_offsets[d], 0), q_rows) : 0;
    const int q1 = a.q_offsets ? min(max(a.q_offsets[d + 1], 0), q_rows) : q_rows;
    doc.n_q = max(q1 - doc.q0, 0);
    doc.k0 = a.k_begin ? min(max(a.k_begin[d], 0), k_rows) : 0;
    const int k1 = a.k_begin ? min(max(a.k_end[d], 0), k_rows) : k_rows;
    doc.n_k = max(k1 - doc.k0, 0);
    doc.shift = doc.n_k - doc.n_q;
    doc.prefix = a.mask == BL_MASK_PREFIX ? max(a.prefix[d], 0) : 0;
    return doc;
}

// The document that holds row `row` by `offsets` (documents + 1 of them, or
// null: one), or -1.
__device__ __forceinline__ int document_at(const int32_t *offsets, uint32_t documents, int row) {
    if (!offsets) return 0;
    int lo = 0, hi = (int)documents;  // the first offset beyond row lies in (lo, hi]
    if (row < offsets[0] || row >= offsets[documents]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (offsets[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ bool visible(const bl_packed_attention_args &a, const Document &doc, int i, int j) {
    return a.mask == BL_MASK_NONE || j <= i + doc.shift || j < doc.prefix;
}

__device__ __forceinline__ float distance_of(const bl_packed_attention_args &a, const Document &doc, int i, int j) {
    if (!a.axes) return (float)abs(i + doc.shift - j);
    int sum = 0;
    for (uint32_t x = 0; x < a.axes; x++)
        sum += abs(a.q_positions[(int64_t)(doc.q0 + i) * a.axes + x] - a.k_positions[(int64_t)(doc.k0 + j) * a.axes + x]);
    return (float)sum;
}

}  // namespace bl
