// New keys and values into a cache of pages, with the keys' norm and rotary
// positions on the way and the queries' beside them, and the way back to packed
// rows (include/beatlm_cache.h).
//
// First a few threads a row find its document, its place and its page, then the
// workgroup makes the rows' sines once, then every head is a few threads' as in
// k_heads.hip: queries to their tensor, keys and values to their page's row. For
// 4 bits a key is made in 64 bits and goes through LDS in f32, since its groups
// of 32 channels lie across the threads that hold its pairs; then, as values do,
// four threads have a group, 8 channels each. The bound is HBM for chunks of
// prompts and the chain of dependent loads (offsets, lengths, table) for a
// step's few tokens, beside which the first heads are on their way: 32 tokens of
// 16 + 4 heads of 128, bf16, 6.6 us. 8192 tokens of them into 4-bit pages 27 us,
// 3.3 TB/s: the keys' 64 bits leave a SIMD three or four waves, whose vector
// instructions are half of the cycles (codes found in 64 bits throughout,
// sines in LDS as large as any call needs and two heads a row at once: 35).
#include "heads_device.hpp"

namespace bl {

namespace {

// The last of `documents` whose offset is not beyond the row, by `width` threads
// of a wave (a power of two from 4 on) that ask for the same row.
__device__ __forceinline__ int document_of_row(const int32_t *offsets, int documents, int64_t row, uint32_t width) {
    if (!offsets) return 0;
    const int sub = (int)(threadIdx.x % width), shift = (int)(threadIdx.x % 64 / width * width);
    const uint64_t mine = width == 64 ? ~0ull : ((1ull << width) - 1) << shift;
    int lo = 0, count = documents;  // the answer is in [lo, lo + count)
    while (count > 1) {
        const int step = (count + (int)width - 1) / (int)width, at = sub * step;
        const bool before = at < count && offsets[lo + at] <= row;
        const int last = __popcll(__ballot(before) & mine) - 1;  // offsets do not fall
        const int skip = max(last, 0) * step;
        lo += skip;
        count = min(step, count - skip);
    }
    return lo;
}

// Where a row of the call belongs.
struct Home {
    int place;  // its key index; of no document: NOBODY
    int page;   // -1: not in the cache
    int row;    // of the page
};
constexpr int NOBODY = INT32_MIN;

__device__ __forceinline__ Home page_of(const bl_paged_cache &cache, int document, int64_t place) {
    Home h{(int)max((int64_t)(NOBODY + 1), min(place, (int64_t)INT32_MAX)), -1, 0};
    const int64_t most = (int64_t)cache.max_pages * cache.page_rows;
    if (place < 0 || place >= most) return h;
    const uint32_t n = (uint32_t)place / cache.page_rows;
    h.row = (int)((uint32_t)place - n * cache.page_rows);
    const int page = cache.table[(uint64_t)document * cache.max_pages + n];
    h.page = (uint32_t)page < cache.pages ? page : -1;
    return h;
}

// The homes of a workgroup's rows, to LDS: `find` gives a (document, row)'s.
template <typename Find>
__device__ __forceinline__ void find_homes(const int32_t *offsets, int documents, uint32_t rows, uint64_t first, uint64_t all, Home *homes, Find find) {
    const uint32_t each = 256 / rows, width = each > 64 ? 64 : each < 4 ? 4 : each, at_once = 256 / width;
    for (uint32_t slot = threadIdx.x / width; slot < rows; slot += at_once) {
        const int64_t row = (int64_t)(first + slot);
        if (row >= (int64_t)all) continue;
        const int d = document_of_row(offsets, documents, row, width);
        if (threadIdx.x % width) continue;
        const int64_t from = offsets ? offsets[d] : 0, to = offsets ? offsets[d + 1] : (int64_t)all;
        homes[slot] = row >= from && row < to ? find(d, row - from, to - from) : Home{NOBODY, -1, 0};
    }
}

__device__ __forceinline__ char *row_of(const bl_pages &pages, const Home &h) {
    return (char *)pages.data + (int64_t)h.page * (int64_t)pages.page_stride + (int64_t)h.row * (int64_t)pages.row_stride;
}

// Extremes of a quad's lanes, in each of them.
__device__ __forceinline__ float quad_min(float v) {
    v = fminf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, false)));
    return fminf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, false)));
}
__device__ __forceinline__ uint32_t half_bits(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
// To f32: a rounding that the compiler would otherwise join with one to f16 behind it.
__device__ __forceinline__ float rounded_once(double v) {
#pragma clang fp contract(off)
    return (float)v;
}

// 8 channels of a group that the lane's quad shares, to their codes, and from
// the quad's first lane the group's step and low. A value's distance to low is
// exact in 64 bits: a tie between two codes is one on every path.
__device__ __forceinline__ void store_codes(const float (&x)[8], char *row, uint32_t head_dim, uint32_t chunk) {
    float least = x[0], most = x[0], bad = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        least = fminf(least, x[e]);
        most = fmaxf(most, x[e]);
        bad = fabsf(x[e]) <= 65504.0f ? bad : 1.0f;
    }
    least = quad_min(least);
    most = -quad_min(-most);
    bad = -quad_min(-bad);
    const uint32_t low_bits = half_bits(least), step_bits = bad != 0.0f ? 0x7e00u : half_bits(rounded_once(((double)most - (double)least) / 15.0));
    const float low = (float)__builtin_bit_cast(_Float16, (uint16_t)low_bits), step = (float)__builtin_bit_cast(_Float16, (uint16_t)step_bits);
    // In f32 a code's place is off by some 2^-20: only where that might cross the
    // middle between two codes is it found in 64 bits. A step of zero or NaN:
    // whatever the code, the value is low or NaN.
    const float per = __builtin_amdgcn_rcpf(step);
    uint32_t codes = 0, close = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float place = (x[e] - low) * per, code = rintf(place);
        close |= (fabsf(place - code) > 0.4999f ? 1u : 0u) << e;
        codes |= (step > 0.0f ? (uint32_t)fminf(fmaxf(code, 0.0f), 15.0f) : 0u) << (e / 2 * 4 + e % 2 * 16);
    }
    if (close && step > 0.0f) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (close >> e & 1) {
                const double code = fmin(fmax(rint(((double)x[e] - (double)low) / (double)step), 0.0), 15.0);
                const int at = e / 2 * 4 + e % 2 * 16;
                codes = (codes & ~(15u << at)) | (uint32_t)code << at;
            }
    }
    *(uint32_t *)(row + chunk * 4) = codes;
    if (chunk % 4 == 0) *(uint32_t *)(row + head_dim / 2 + chunk) = step_bits | low_bits << 16;
}

// 8 channels at p, in accesses of VEC elements.
template <typename T, int VEC>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    constexpr int N = VEC > 8 ? 8 : VEC;
#pragma unroll
    for (int e = 0; e < 8; e += N) {
        float v[N];
        load_vec<T, N>(p + e, v);
#pragma unroll
        for (int i = 0; i < N; i++) x[e + i] = v[i];
    }
}

template <typename T, int VEC, bool INT4>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p, HeadsGeometry g) {
    constexpr int UP = UNITS<VEC>;
    typedef std::conditional_t<INT4, double, float> F;
    extern __shared__ __attribute__((aligned(16))) char turns[];  // of the rows' pairs, as many as there are
    F *const cosines = (F *)turns, *const sines = cosines + g.rows * p.h.table.pairs;
    __shared__ __attribute__((aligned(16))) float staged[INT4 ? 2 * 256 * UP * VEC : 1];  // a head's channels for each of the seats' lanes
    __shared__ Home homes[256];
    __shared__ __attribute__((aligned(16))) float weights[2][BL_ATTENTION_MAX_HEAD_DIM];
    const HeadsParams &a = p.h;
    const Seat seat(g);
    const uint64_t first = g.first + (uint64_t)blockIdx.x * g.rows, row = first + seat.slot;
    Chunk<VEC> c[UP];
    chunks_of<VEC>(g, a.table, seat.lane, c);
    // The first heads are on their way while the rows' homes are looked up.
    const T *const q = (const T *)a.q_in.data + row * a.q_in.row_stride, *const k = (const T *)a.k_in.data + row * a.k_in.row_stride;
    Raw<T, VEC> next_q, next_k;
    const bool has_q = row < a.rows && seat.group < a.q_heads, has_k = row < a.rows && seat.group < a.k_heads;
    if (has_q) next_q.load(q + (uint64_t)seat.group * a.q_in.head_stride, c);
    if (has_k) next_k.load(k + (uint64_t)seat.group * a.k_in.head_stride, c);
    if (a.norm != BL_HEAD_NORM_NONE) put_weights<T>(a, weights);
    find_homes(p.q_offsets, (int)p.documents, g.rows, first, a.rows, homes,
               [&](int d, int64_t i, int64_t n) { return page_of(p.cache, d, (int64_t)p.cache.lengths[d] - n + i); });
    __syncthreads();
    make_sines(a.table, g.rows, first, a.rows, cosines, sines, [&](uint32_t slot, uint64_t r, uint32_t axis) {
        return a.positions ? a.positions[r * a.table.axes + axis] : homes[slot].place;
    });
    __syncthreads();
    if (row >= a.rows) return;
    const Home home = homes[seat.slot];
    if (home.place == NOBODY) return;
    const F *const co = cosines + seat.slot * a.table.pairs, *const si = sines + seat.slot * a.table.pairs;
    if (has_q) {
        T *dst = (T *)a.q_out.data + row * a.q_out.row_stride;
        for (uint32_t h = seat.group; h < a.q_heads; h += g.head_groups) {
            Channels<VEC, float> x;
            next_q.to(x);
            if (h + g.head_groups < a.q_heads) next_q.load(q + (uint64_t)(h + g.head_groups) * a.q_in.head_stride, c);
            if (a.norm != BL_HEAD_NORM_NONE) {
                x.normalise(a.norm, a.epsilon, a.head_dim, g.lanes, c);
                weigh_by<VEC>(x, weights[0], c);
            }
            turn_by<VEC>(x, co, si, a.table.layout, 1.0f, c);
            x.store(dst + (uint64_t)h * a.q_out.head_stride, c);
        }
    }
    if (home.page < 0 || !has_k) return;
    const T *const v = (const T *)p.v_in.data + row * p.v_in.row_stride;
    char *const k_row = row_of(p.cache.k, home), *const v_row = row_of(p.cache.v, home);
    for (uint32_t h = seat.group; h < a.k_heads; h += g.head_groups) {
        Channels<VEC, F> x;
        next_k.to(x);
        if (h + g.head_groups < a.k_heads) next_k.load(k + (uint64_t)(h + g.head_groups) * a.k_in.head_stride, c);
        if (a.norm != BL_HEAD_NORM_NONE) {
            x.normalise(a.norm, a.epsilon, a.head_dim, g.lanes, c);
            weigh_by<VEC>(x, weights[1], c);
        }
        turn_by<VEC>(x, co, si, a.table.layout, F(1), c);
        const T *value = v + (uint64_t)h * p.v_in.head_stride;
        char *const to_k = k_row + (uint64_t)h * p.cache.k.head_stride, *const to_v = v_row + (uint64_t)h * p.cache.v.head_stride;
        if constexpr (INT4) {
            // Through LDS within the head's lanes, which are of one wave.
            float *const mine = staged + threadIdx.x / g.lanes * g.lanes * UP * 2 * VEC;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            x.store(mine, c);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            for (uint32_t n = seat.lane; n < a.head_dim / 8; n += g.lanes) {
                float z[8];
                load8<float, 4>(mine + n * 8, z);
                store_codes(z, to_k, a.head_dim, n);
                load8<T, VEC>(value + n * 8, z);
                store_codes(z, to_v, a.head_dim, n);
            }
        } else {
            x.store((T *)to_k, c);
            for (uint32_t n = seat.lane * VEC; n < a.head_dim; n += g.lanes * VEC) {
                float z[VEC];
                load_vec<T, VEC>(value + n, z);
                store_vec<T, VEC>((T *)to_v + n, z);
            }
        }
    }
}

// The f16 values of 8 codes, in channels' order.
__device__ __forceinline__ void values_of(uint32_t codes, uint32_t params, float (&x)[8]) {
    const _Float16 step = __builtin_bit_cast(_Float16, (uint16_t)params), low = __builtin_bit_cast(_Float16, (uint16_t)(params >> 16));
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (float)__builtin_fmaf16((_Float16)(float)(codes >> (e / 2 * 4 + e % 2 * 16) & 15), step, low);
}

// 8 channels a thread of a row and head, k's and then v's.
template <typename T, bool INT4>
__global__ __launch_bounds__(256) void read_kernel(bl_cache_read_args a, HeadsGeometry g) {
    __shared__ Home homes[256];
    const Seat seat(g);
    const uint64_t first = g.first + (uint64_t)blockIdx.x * g.rows, row = first + seat.slot;
    find_homes(a.offsets, (int)a.documents, g.rows, first, a.rows, homes, [&](int d, int64_t i, int64_t) {
        const int64_t j = (a.first ? a.first[d] : 0) + i;
        if (j < 0 || j >= min((int64_t)a.cache.lengths[d], (int64_t)a.cache.max_pages * a.cache.page_rows)) return Home{NOBODY, -1, 0};
        return page_of(a.cache, d, j);
    });
    __syncthreads();
    const uint32_t c = seat.lane * 8;
    if (row >= a.rows || c >= a.head_dim) return;
    const Home home = homes[seat.slot];
    if (home.place == NOBODY) return;
    for (uint32_t h = seat.group; h < a.kv_heads; h += g.head_groups) {
        T *const out[2] = {(T *)a.k_out.data + row * a.k_out.row_stride + (uint64_t)h * a.k_out.head_stride + c,
                           (T *)a.v_out.data + row * a.v_out.row_stride + (uint64_t)h * a.v_out.head_stride + c};
        float x[2][8] = {};
        if (home.page >= 0)
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const bl_pages &pages = n == 0 ? a.cache.k : a.cache.v;
                const char *from = row_of(pages, home) + (uint64_t)h * pages.head_stride;
                if constexpr (INT4) values_of(*(const uint32_t *)(from + c / 2), *(const uint32_t *)(from + a.head_dim / 2 + c / 32 * 4), x[n]);
                else load8<T, 16 / sizeof(T)>((const T *)from + c, x[n]);
            }
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 8; e += N) {
                float v[N];
#pragma unroll
                for (int i = 0; i < N; i++) v[i] = x[n][e + i];
                store_vec<T, N>(out[n] + e, v);
            }
    }
}

// Rows in launches of fewer than 2^32 threads.
template <typename Launch>
hipError_t in_parts(HeadsGeometry &g, uint64_t rows, Launch launch) {
    const uint64_t most = 1u << 23, groups = (rows + g.rows - 1) / g.rows;
    for (uint64_t done = 0; done < groups; done += most) {
        g.first = (uint32_t)(done * g.rows);
        if (const hipError_t e = launch((uint32_t)(groups - done < most ? groups - done : most)); e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename T, int VEC>
hipError_t append(const AppendParams &p, uint32_t compute_units, hipStream_t s) {
    const HeadsParams &a = p.h;
    const bool int4 = p.cache.kind == BL_CACHE_INT4;
    HeadsGeometry g = heads_geometry(VEC, a.table.pairs, a.head_dim, a.q_heads > a.k_heads ? a.q_heads : a.k_heads, a.rows, int4 ? 4 : 1, 4ull * compute_units);
    return in_parts(g, a.rows, [&](uint32_t grid) {
        const uint32_t held = 2 * g.rows * a.table.pairs;
        return int4 ? run_kernel_with(held * sizeof(double), append_kernel<T, VEC, true>, grid, 256, s, p, g)
                    : run_kernel_with(held * sizeof(float), append_kernel<T, VEC, false>, grid, 256, s, p, g);
    });
}

template <typename T>
hipError_t read(const bl_cache_read_args &a, uint32_t compute_units, hipStream_t s) {
    HeadsGeometry g = heads_geometry(8, 0, a.head_dim, a.kv_heads, a.rows, 1, 2ull * compute_units);
    return in_parts(g, a.rows, [&](uint32_t grid) {
        return a.cache.kind == BL_CACHE_INT4 ? run_kernel(read_kernel<T, true>, grid, 256, s, a, g) : run_kernel(read_kernel<T, false>, grid, 256, s, a, g);
    });
}

}  // namespace

hipError_t launch_cache_append(const AppendParams &p, uint32_t dtype, uint32_t compute_units, hipStream_t s) {
    const uint32_t vec = p.h.vec;
    switch (dtype) {
    case BL_F32: return vec == 4 ? append<float, 4>(p, compute_units, s) : append<float, 1>(p, compute_units, s);
    case BL_F16:
        return vec == 8 ? append<_Float16, 8>(p, compute_units, s) : vec == 4 ? append<_Float16, 4>(p, compute_units, s) : append<_Float16, 1>(p, compute_units, s);
    default:
        return vec == 8 ? append<__bf16, 8>(p, compute_units, s) : vec == 4 ? append<__bf16, 4>(p, compute_units, s) : append<__bf16, 1>(p, compute_units, s);
    }
}

hipError_t launch_cache_read(const bl_cache_read_args &a, uint32_t compute_units, hipStream_t s) {
    switch (a.dtype) {
    case BL_F32: return read<float>(a, compute_units, s);
    case BL_F16: return read<_Float16>(a, compute_units, s);
    default: return read<__bf16>(a, compute_units, s);
    }
}

}  // namespace bl
