// What the packed attention kernels share: a document's bounds, clamped to
// the tensors whatever the offset arrays hold; which document and tile a
// workgroup has; matrix core operands of the three element types; tiles of
// rows staged through LDS; scores.
#pragma once

#include "ops_device.hpp"

namespace bl {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// ---- documents ----

// What every lane holds alike, in a scalar register: buffer descriptors and
// branches want it there, and the compiler cannot always tell.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    return (uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v);
}

struct Document {
    int q0, n_q;     // first query row, query rows
    int k0, n_k;     // first key row, key rows
    int shift;       // n_k - n_q: query i stands at key i + shift
    int prefix;      // keys every query sees
};

__device__ __forceinline__ Document document_of(const bl_packed_attention_args &a, int d) {
    Document doc;
    const int q_rows = (int)a.q_rows, k_rows = (int)a.k_rows;
    doc.q0 = uniform(a.q_offsets ? min(max(a.q_offsets[d], 0), q_rows) : 0);
    const int q1 = a.q_offsets ? min(max(a.q_offsets[d + 1], 0), q_rows) : q_rows;
    doc.n_q = uniform(max(q1 - doc.q0, 0));
    doc.k0 = uniform(a.k_begin ? min(max(a.k_begin[d], 0), k_rows) : 0);
    const int k1 = a.k_begin ? min(max(a.k_end[d], 0), k_rows) : k_rows;
    doc.n_k = uniform(max(k1 - doc.k0, 0));
    doc.shift = doc.n_k - doc.n_q;
    doc.prefix = uniform(a.mask == BL_MASK_PREFIX ? max(a.prefix[d], 0) : 0);
    return doc;
}

// Keys [0, limit) of the document are what its query i sees.
__device__ __forceinline__ int limit_of(const bl_packed_attention_args &a, const Document &doc, int i) {
    return a.mask == BL_MASK_NONE ? doc.n_k : min(doc.n_k, max(i + doc.shift + 1, doc.prefix));
}

// The tiles of all documents have one grid: document d's tiles of `tile`
// places (its rows times `times`) start at slot first * times / tile + d,
// which leaves room for each document's last, partial tile whatever the
// lengths are. slots() is the grid; document_of_slot finds the document whose
// first slot is the last one not beyond `slot` (64 candidates a step, one
// load), or 0.
__host__ __device__ __forceinline__ uint32_t slots(uint32_t rows, uint32_t times, uint32_t tile, uint32_t documents) {
    return (uint32_t)((uint64_t)rows * times / tile) + documents;
}
__device__ __forceinline__ int first_slot(const int32_t *offsets, int d, int rows, int times, int tile) {
    return (int)((int64_t)min(max(offsets[d], 0), rows) * times / tile) + d;
}
__device__ __forceinline__ int document_of_slot(const int32_t *offsets, int documents, int rows, int times, int tile, int slot) {
    if (!offsets || documents == 1) return 0;
    const int lane = threadIdx.x % 64;
    int lo = 0, count = documents;  // the answer is in [lo, lo + count)
    while (count > 1) {
        const int step = (count + 63) / 64;
        const int d = lo + lane * step;
        const bool before = lane * step < count && first_slot(offsets, d, rows, times, tile) <= slot;
        const int last = __popcll(__ballot(before)) - 1;  // first slots rise with d
        const int at = max(last, 0) * step;
        lo += at;
        count = min(step, count - at);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// Nothing is scheduled across this: it bounds how many operands are in
// registers at once where the compiler would fetch all of a loop's first.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// ---- matrix core operands ----
//
// Every product here runs on 32 x 32 tiles: C[row][col] is held by lane
// (half h = lane / 32, col = lane % 32), register r at row
// 8 (r / 4) + 4 h + r % 4. An operand is a 16-byte chunk a lane: KS / 2
// elements of the contraction for its row (A) or column (B), the two halves
// sharing a step of KS. Which of the step's elements a half holds is free as
// long as A and B agree:
//  - for operands read along their rows, half h has elements KS/2 h + [0, KS/2);
//  - for a product over a tile's rows or columns just computed (probabilities),
//    half h has those its registers hold: 8 (j / 4) + 4 h + j % 4 of 16 for the
//    16-bit types, 4 h + j of 8 for f32. The other operand is read transposed
//    in the same order, so no value changes lanes.

template <typename T> struct Mma;
template <> struct Mma<_Float16> {
    typedef f16x8 Frag;
    static constexpr int KS = 16;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<__bf16> {
    typedef bf16x8 Frag;
    static constexpr int KS = 16;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> {
    typedef f32x4 Frag;
    static constexpr int KS = 8;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

// KS values of a tile's registers (16-bit: registers 8 t .. 8 t + 7, f32:
// 4 t .. 4 t + 3) as an operand of step t: the one rounding of probabilities
// and scores' gradients to the tensors' type, which the matrix cores ask for. It
// averages out over keys: 2.1e-3 of the output's 2-norm where the output's own
// rounding is 1.6e-3 (bf16, one token over 16326 keys), 3.0e-4 of d_q's where that is
// 2.1e-4 (f16, 700 tokens). f32 is not rounded.
template <typename T>
__device__ __forceinline__ typename Mma<T>::Frag operand_of(const f32x16 &v, int t) {
    typename Mma<T>::Frag f;
    constexpr int N = Mma<T>::KS / 2;
#pragma unroll
    for (int j = 0; j < N; j++) f[j] = (T)v[N * t + j];
    return f;
}

// ---- tiles of rows in LDS ----
//
// ROWS rows of D channels, 16-byte chunks, brought by buffer loads straight
// into LDS. The buffer ends with the last row the document owns and a lane
// beyond head_dim points outside, and what lies outside arrives as zeros: no
// row of another document is read, and no padding is left to chance. Chunks
// lie in LDS in the loads' order, which is linear in the lane, so a row's
// chunks are permuted on the global side: position x holds chunk
// x ^ swizzle(row), which spreads both the reads along rows (16 rows, one
// chunk each) and the transposed ones (8 rows, 4 neighbouring chunks each)
// over all 64 banks.

template <typename T, int D, int ROWS, int THREADS = 256> struct Tile {
    typedef typename Mma<T>::Frag Frag;
    static constexpr int CHUNKS = D * (int)sizeof(T) / 16;  // of a row: 8, 16 or 32
    static constexpr int ROW = D * (int)sizeof(T);
    static constexpr int BYTES = ROWS * ROW;
    static constexpr int LOADS = ROWS * CHUNKS / THREADS;    // a thread's, of the workgroup's
    static constexpr int STEPS = D / Mma<T>::KS;             // of a product over channels

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (CHUNKS == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
        else if constexpr (sizeof(T) == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
        else return row & 7;
    }

    // Byte offsets of this thread's chunks from the tile's first row.
    uint32_t offset[LOADS];
    int stride, end;  // bytes from a row to the next; of the last row

    __device__ __forceinline__ Tile(uint64_t row_stride, uint32_t head_dim) {
        stride = uniform((int)(row_stride * sizeof(T)));
        end = uniform((int)(head_dim * sizeof(T)));
#pragma unroll
        for (int n = 0; n < LOADS; n++) {
            const int i = n * THREADS + threadIdx.x % THREADS;
            const int row = i / CHUNKS, chunk = (i % CHUNKS) ^ swizzle(row);
            offset[n] = chunk * 16 < end ? (uint32_t)row * stride + chunk * 16 : 0x7ffffff0u;
        }
    }
    // Starts the loads of up to `left` rows from `base` (a scalar address)
    // into `lds`, zeros where there are none; `own`: bytes on, where the loading threads
    // are one wave of several with a tile each.
    __device__ __forceinline__ void load(uint64_t base, int left, char *lds, int own = 0) const {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass knows no 16-byte loads to LDS
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)uniform64(base), 0, uniform(left > 0 ? (min(left, ROWS) - 1) * stride + end : 0), 0x00020000);
        const int wave = uniform(threadIdx.x % THREADS / 64);
#pragma unroll
        for (int n = 0; n < LOADS; n++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)(lds + own + (n * THREADS + wave * 64) * 16), 16,
                                                     offset[n], 0, 0, 0);
#endif
    }
    static __device__ __forceinline__ T *element(char *lds, int row, int c) {
        constexpr int PER = 16 / sizeof(T);
        return (T *)(lds + row * ROW + ((c / PER) ^ swizzle(row)) * 16) + c % PER;
    }
};

// A lane's places in a tile, found once: all that is left for a read is a
// constant (LDS instructions take it) and one of a few registers.
template <typename T, int D, int ROWS, int BLOCKS = D / 32> struct Reader {
    typedef Tile<T, D, ROWS> S;
    typedef typename Mma<T>::Frag Frag;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int STEPS = F32 ? 4 : S::STEPS;       // steps until the places along a row repeat, 128 bytes on
    static constexpr int PIECES = F32 ? 4 : BLOCKS * 2;
    int a[STEPS], b[PIECES];

    // `first`: the first of the BLOCKS blocks of 32 channels that are read transposed.
    __device__ __forceinline__ explicit Reader(int lane, int first = 0) {
        const int half = lane / 32, row = lane % 32;
#pragma unroll
        for (int t = 0; t < STEPS; t++) a[t] = row * S::ROW + ((2 * t + half) ^ S::swizzle(row)) * 16;
#pragma unroll
        for (int n = 0; n < PIECES; n++) {
            if constexpr (F32) {
                const int r = 4 * half + n;
                b[n] = r * S::ROW + ((lane % 32 / 4) ^ S::swizzle(r)) * 16 + lane % 4 * 4 + first * 128;
            } else {
                // 16 lanes bring a 4 x 16 piece: lane i row i / 4, channels 4 (i % 4) ..; each gets its column.
                const int i = lane % 16, chunk = 4 * (first + n / 2) + 2 * (lane / 16 % 2) + i % 4 / 2;
                const int r = 4 * half + i / 4 + n % 2 * 8;
                b[n] = r * S::ROW + (chunk ^ S::swizzle(r)) * 16 + i % 2 * 8;
            }
        }
    }
    // The operand of rows r0 + lane % 32 (r0 a multiple of 32) and step t along the channels.
    __device__ __forceinline__ Frag along(const char *lds, int r0, int t) const {
        return *(const Frag *)(lds + a[t % STEPS] + (r0 * S::ROW + t / STEPS * 128));
    }
    // The transposed operand: channel 32 (first + block) + lane % 32, rows of step t.
    __device__ __forceinline__ Frag across(const char *lds, int t, int block) const {
        if constexpr (F32) {
            Frag f;
#pragma unroll
            for (int j = 0; j < 4; j++) f[j] = *(const float *)(lds + b[j] + (8 * t * S::ROW + block * 128));
            return f;
        } else {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            const auto piece = [&](int n) {
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + b[2 * block + n] + 16 * t * S::ROW));
            };
            return __builtin_bit_cast(Frag, __builtin_shufflevector(piece(0), piece(1), 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// The address of a (row, head) of a tensor, scalar.
template <typename T> __device__ __forceinline__ uint64_t address_of(const bl_heads &h, int64_t row, int64_t head) {
    return uniform64((uint64_t)h.data + (uint64_t)(row * (int64_t)h.row_stride + head * (int64_t)h.head_stride) * sizeof(T));
}

// A lane's row of a tensor as operands along the channels, zeros beyond
// head_dim and where the lane has none (`row` is then any row there is).
template <typename T, int D>
__device__ __forceinline__ void load_row(const bl_heads &h, bool there, int64_t row, int64_t head, int half, uint32_t head_dim,
                                         typename Mma<T>::Frag (&f)[D / Mma<T>::KS]) {
    typedef typename Mma<T>::Frag Frag;
    constexpr int KS = Mma<T>::KS;
    const T *at = (const T *)h.data + row * (int64_t)h.row_stride + head * (int64_t)h.head_stride;
#pragma unroll
    for (int t = 0; t < D / KS; t++) {
        const uint32_t c = t * KS + half * (KS / 2);
        const bool in = c < head_dim;
        const Frag v = *(const Frag *)(at + (in ? c : 0));
        f[t] = there && in ? v : Frag{};
    }
}

// Accumulators C[channel][the lane's row] of N blocks of 32 channels from
// block `first` on, times `by`, to the lane's row of a tensor.
template <typename T, int N>
__device__ __forceinline__ void store_row(const bl_heads &h, int64_t row, int64_t head, int half, uint32_t head_dim, const f32x16 (&acc)[N], int first,
                                          float by) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T *at = (T *)h.data + row * (int64_t)h.row_stride + head * (int64_t)h.head_stride;
#pragma unroll
    for (int b = 0; b < N; b++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const uint32_t c = 32 * (first + b) + 2 * r + 4 * half;
            T4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = (T)(acc[b][r + e] * by);
            if (c < head_dim) *(T4 *)(at + c) = v;  // head_dim is a multiple of 8
        }
}
// The same to a row of a split's partial sums.
template <int N>
__device__ __forceinline__ void store_partial(float *at, int half, const f32x16 (&acc)[N], int first, float by) {
#pragma unroll
    for (int b = 0; b < N; b++)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *(f32x4 *)(at + 32 * (first + b) + 2 * r + 4 * half) = f32x4{acc[b][r], acc[b][r + 1], acc[b][r + 2], acc[b][r + 3]} * by;
}

// ---- scores ----
//
// In base two: x = log2(e) s, so probabilities are exp2(x - .), by the hardware's
// exponential in every type: off by a step of f32, as its argument's own rounding
// is from |x| = 1 on. With a cap, s = cap tanh(u), u = scale qk / cap. `factor` is
// what x is of a product, or of its tanh.

// tanh(u) for |u| < TANH_NEAR: a polynomial in u^2 (fitted to tanh(u) / u at
// Chebyshev points) that is off by less than a step of f32.
template <bool F32> constexpr float TANH_NEAR = F32 ? 1.0f : 0.5f;
template <bool F32> __device__ __forceinline__ float tanh_near_zero(float u) {
    const float w = u * u;
    float v;
    if constexpr (F32) {
        v = 0.00228764559f + w * -0.000354883407f;
        v = 0.0214699805f + w * (-0.00792494603f + w * v);
        v = 0.133321911f + w * (-0.053872738f + w * v);
        v = 1.0f + w * (-0.333332807f + w * v);
    } else {
        v = 0.133248284f + w * (-0.0529892407f + w * 0.0171413198f);
        v = 1.0f + w * (-0.333330721f + w * v);
    }
    return u * v;
}

template <typename T, bool CAP> struct Scores {
    float factor;  // log2(e) scale, or log2(e) cap
    float inner;   // scale / cap
    Scores() = default;
    // `ordered`: for q whose sign the caller has changed where scale is
    // negative, so that x grows with the product (and a scale of zero keeps a
    // hidden -inf what it is).
    __device__ __forceinline__ explicit Scores(const bl_packed_attention_args &a, bool ordered = false) {
        const float scale = ordered ? fmaxf(fabsf(a.scale), 1e-37f) : a.scale;
        factor = (CAP ? a.softcap : scale) * LOG2E;
        inner = CAP ? scale / a.softcap : 0.0f;
    }
    // With a cap, products to their tanh u. Where a wave's tile has no |u| of
    // LIMIT or more, the usual case as caps are wide, the polynomial: 4 or 7
    // multiplications more than the product itself, 28 cycles a wave for the
    // 16-bit types. Any other tile: 1 - 2 / (e^2u + 1), off by a few steps of
    // 1, 44 cycles with its two quarter-rate instructions; f32 takes tanhf, some
    // ten times that.
    __device__ __forceinline__ void caps(f32x16 &s) const {
        if constexpr (!CAP) return;
        constexpr bool F32 = sizeof(T) == 4;
        constexpr float LIMIT = TANH_NEAR<F32>;
        float top = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) top = fmaxf(fmaxf(fabsf(s[r]), fabsf(s[r + 1])), top);
        if (__all(top * fabsf(inner) < LIMIT)) {  // a NaN is no maximum, and stays one in either form
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = tanh_near_zero<F32>(s[r] * inner);
        } else if constexpr (F32) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = tanhf(s[r] * inner);
        } else {
            const float twice = 2.0f * LOG2E * inner;
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[r] * twice) + 1.0f);
        }
    }
};

// |a - b| + c of values whose order is that of unsigned numbers: one v_sad_u32.
__device__ __forceinline__ uint32_t apart(uint32_t a, uint32_t b, uint32_t c) { return (max(a, b) - min(a, b)) + c; }

}  // namespace bl
