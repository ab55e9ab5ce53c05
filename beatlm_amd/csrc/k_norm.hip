// LayerNorm over strided rows and its gradients (include/beatlm_ops.h).
//
// Both directions read each row once: TPR threads (a quarter of a wave to
// sixteen waves) keep it in registers, 16 values each, so the variance is the
// mean of squares about the mean (two passes over registers, no cancellation)
// and nothing is read twice. The bound is HBM: forward x in, y out; backward x
// and dy in, dx out. Rows come and go in 16-byte pieces wherever they start
// (the memory system takes them at any element's address; 4097 x 1003 f32
// forward and backward: 23 us, an element at a time 43), their last few values
// one by one. What the sums do not need is loaded before them, and the backward
// loads its next row while it finishes the last, so one latency is paid a row.
// 21920 x 768 bf16: forward 15.9 us, 4.2 TB/s, backward 21.5, 4.7 TB/s, and
// 4.5 for the weights' gradients' second launch.
//
// The weights' gradients are sums over rows: a workgroup of the backward walks
// rows with a stride of the grid and keeps its columns' two sums in registers;
// its partial sums go to the workspace and a second launch adds the groups'
// in order. No atomics, so the order of the sums is fixed.
#include "ops_device.hpp"

namespace bl {

namespace {

constexpr int EPT = 16;  // values of a row a thread holds
template <int TPR> constexpr int norm_threads = TPR <= 64 ? 256 : TPR;  // of a workgroup

// Sum over the wave, in every lane, without LDS: 16 lanes by DPP, then the
// two exchanges of rows of 16 and of 32.
__device__ __forceinline__ float wave_sum_dpp(float v) {
    v = row16_sum(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return sum_xor32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Sums of K values over the TPR threads of a row, in every one of them.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float *lds) {
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = TPR == 16 ? row16_sum(v[k]) : wave_sum_dpp(v[k]);
    if constexpr (TPR > 64) {
        constexpr int WAVES = TPR / 64;
        const int wave = threadIdx.x / 64;
        __syncthreads();  // the last sums have been read
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int k = 0; k < K; k++) lds[k * WAVES + wave] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) s += lds[k * WAVES + w];
            v[k] = s;
        }
    }
}

// A thread's pieces of a row: N of VEC values, piece n from column
// (n * TPR + lane) * VEC on.
template <typename T, int TPR> struct Pieces {
    static constexpr int VEC = 16 / sizeof(T), N = EPT / VEC;
    typedef T V __attribute__((ext_vector_type(VEC)));
    typedef V Anywhere __attribute__((aligned(sizeof(T))));  // at any element's address
    V v[N];
    static __device__ __forceinline__ uint32_t col(int lane, int n) { return (uint32_t)(n * TPR + lane) * VEC; }
    // Values beyond the row are `other`.
    __device__ __forceinline__ void load(const T *row, uint32_t cols, int lane, T other) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const uint32_t c = col(lane, n);
            if (c + VEC <= cols) {
                v[n] = *(const Anywhere *)(row + c);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++) v[n][e] = c + e < cols ? row[c + e] : other;
            }
        }
    }
    static __device__ __forceinline__ void store(T *row, uint32_t cols, int lane, int n, V x) {
        const uint32_t c = col(lane, n);
        if (c + VEC <= cols) {
            *(Anywhere *)(row + c) = x;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (c + e < cols) row[c + e] = x[e];
        }
    }
};

template <typename T, int TPR>
__global__ __launch_bounds__(norm_threads<TPR>) void norm_forward_kernel(NormParams p) {
    typedef Pieces<T, TPR> P;
    constexpr int VEC = P::VEC, N = P::N, ROWS = norm_threads<TPR> / TPR;
    __shared__ float lds[TPR / 64 + 1];
    const int lane = threadIdx.x % TPR;
    uint32_t row = blockIdx.x * ROWS + threadIdx.x / TPR;
    if (row >= p.rows) return;  // all threads of a row; with rows of a wave or less no barrier follows
    P x, gamma, beta;
    x.load((const T *)p.x + (uint64_t)row * p.x_stride, p.cols, lane, (T)0.0f);
    gamma.load((const T *)p.gamma, p.cols, lane, (T)0.0f);
    beta.load((const T *)p.beta, p.cols, lane, (T)0.0f);
    while (row < p.rows) {
        float v[N][VEC];
        float sum[1] = {0.0f};
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < VEC; e++) sum[0] += v[n][e] = (float)x.v[n][e];
        const uint32_t now = row;
        row += gridDim.x * ROWS;
        if (row < p.rows) x.load((const T *)p.x + (uint64_t)row * p.x_stride, p.cols, lane, (T)0.0f);
        row_sums<TPR, 1>(sum, lds);
        const float mean = sum[0] / (float)p.cols;
        float square[1] = {0.0f};
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                v[n][e] -= mean;
                square[0] += P::col(lane, n) + e < p.cols ? v[n][e] * v[n][e] : 0.0f;
            }
        row_sums<TPR, 1>(square, lds);
        const float rstd = 1.0f / sqrtf(square[0] / (float)p.cols + p.epsilon);
        if (lane == 0) {
            if (p.mean) p.mean[now] = mean;
            if (p.rstd) p.rstd[now] = rstd;
        }
        T *y = (T *)p.y + (uint64_t)now * p.y_stride;
#pragma unroll
        for (int n = 0; n < N; n++) {
            typename P::V out;
#pragma unroll
            for (int e = 0; e < VEC; e++) out[e] = (T)(v[n][e] * rstd * (float)gamma.v[n][e] + (float)beta.v[n][e]);
            P::store(y, p.cols, lane, n, out);
        }
    }
}

template <typename T, int TPR>
__global__ __launch_bounds__(norm_threads<TPR>) void norm_backward_kernel(NormParams p) {
    typedef Pieces<T, TPR> P;
    constexpr int VEC = P::VEC, N = P::N, ROWS = norm_threads<TPR> / TPR, WIDTH = TPR * EPT;
    __shared__ float lds[TPR <= 64 ? 2 * ROWS * WIDTH : 2 * (TPR / 64)];
    const int lane = threadIdx.x % TPR;
    P gamma, x, dy;
    gamma.load((const T *)p.gamma, p.cols, lane, (T)0.0f);
    float dg[N][VEC], db[N][VEC];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int e = 0; e < VEC; e++) dg[n][e] = db[n][e] = 0.0f;
    const float each = 1.0f / (float)p.cols;
    uint32_t row = blockIdx.x * ROWS + threadIdx.x / TPR;
    float mean = 0.0f, rstd = 0.0f;
    const auto fetch = [&](uint32_t r) {
        x.load((const T *)p.x + (uint64_t)r * p.x_stride, p.cols, lane, (T)0.0f);
        dy.load((const T *)p.dy + (uint64_t)r * p.dy_stride, p.cols, lane, (T)0.0f);
        mean = p.mean[r];
        rstd = p.rstd[r];
    };
    constexpr bool AHEAD = TPR < 1024;  // sixteen waves of a workgroup have no registers for the next row
    if (AHEAD && row < p.rows) fetch(row);
    while (row < p.rows) {
        if constexpr (!AHEAD) fetch(row);
        float n_[N][VEC], d[N][VEC];
        float sums[2] = {0.0f, 0.0f};  // of g and of g n
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                // dy is 0 beyond the row; n has to be finite there, as mean * rstd need not be
                n_[n][e] = P::col(lane, n) + e < p.cols ? ((float)x.v[n][e] - mean) * rstd : 0.0f;
                d[n][e] = (float)dy.v[n][e];
                dg[n][e] += d[n][e] * n_[n][e];
                db[n][e] += d[n][e];
                d[n][e] *= (float)gamma.v[n][e];
                sums[0] += d[n][e];
                sums[1] += d[n][e] * n_[n][e];
            }
        const float scale = rstd;
        T *dx = (T *)p.dx + (uint64_t)row * p.dx_stride;
        row += gridDim.x * ROWS;
        if (AHEAD && row < p.rows) fetch(row);
        row_sums<TPR, 2>(sums, lds);
        const float m0 = sums[0] * each, m1 = sums[1] * each;
#pragma unroll
        for (int n = 0; n < N; n++) {
            typename P::V out;
#pragma unroll
            for (int e = 0; e < VEC; e++) out[e] = (T)((d[n][e] - m0 - n_[n][e] * m1) * scale);
            P::store(dx, p.cols, lane, n, out);
        }
    }
    // The workgroup's partial sums; where it has several rows at once, theirs added first.
    float *out = p.partial + (uint64_t)blockIdx.x * 2 * p.cols;
    if constexpr (TPR <= 64) {
        const int which_row = threadIdx.x / TPR;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                lds[(which_row * 2 + 0) * WIDTH + P::col(lane, n) + e] = dg[n][e];
                lds[(which_row * 2 + 1) * WIDTH + P::col(lane, n) + e] = db[n][e];
            }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2 * p.cols; i += 256) {
            const uint32_t which = i >= p.cols, c = i - which * p.cols;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < ROWS; w++) s += lds[(w * 2 + which) * WIDTH + c];
            out[i] = s;
        }
    } else {
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const uint32_t c = P::col(lane, n) + e;
                if (c < p.cols) {
                    out[c] = dg[n][e];
                    out[p.cols + c] = db[n][e];
                }
            }
    }
}

// d_gamma and d_beta from the groups' partial sums: 16 columns a workgroup (64
// bytes of each partial), 64 threads a column, each with several groups at once.
__global__ __launch_bounds__(1024) void norm_reduce_kernel(NormParams p) {
    __shared__ float lds[64][17];
    const uint32_t i = blockIdx.x * 16 + threadIdx.x % 16;  // of 2 * cols
    const uint32_t first = threadIdx.x / 16;
    float s = 0.0f;
    if (i < 2 * p.cols) {
        uint32_t group = first;
        for (; group + 192 < p.groups; group += 256) {
            float v[4];
#pragma unroll
            for (int n = 0; n < 4; n++) v[n] = p.partial[(uint64_t)(group + 64 * n) * 2 * p.cols + i];
            s += (v[0] + v[1]) + (v[2] + v[3]);
        }
        for (; group < p.groups; group += 64) s += p.partial[(uint64_t)group * 2 * p.cols + i];
    }
    lds[first][threadIdx.x % 16] = s;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    // 16 rows each, then across the four sixteens of the wave.
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w++) s += lds[first * 16 + w][threadIdx.x % 16];
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(s), false, false);
    s = sum_xor32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
    if (threadIdx.x >= 16 || i >= 2 * p.cols) return;
    if (i < p.cols) p.d_gamma[i] = s;
    else p.d_beta[i - p.cols] = s;
}

// The threads a row of `cols` gets: a quarter of a wave for up to 256 columns
// (forward and backward of 8353 x 128 bf16 12.5 us, with a wave 20.8), a wave
// for up to 1024, four for up to 4096, sixteen for the rest.
uint32_t threads_per_row(uint32_t cols) { return cols <= 16 * EPT ? 16 : cols <= 64 * EPT ? 64 : cols <= 256 * EPT ? 256 : 1024; }

template <typename T>
hipError_t forward(const NormParams &p, hipStream_t s) {
    switch (threads_per_row(p.cols)) {
    case 16: return run_kernel(norm_forward_kernel<T, 16>, p.groups, 256, s, p);
    case 64: return run_kernel(norm_forward_kernel<T, 64>, p.groups, 256, s, p);
    case 256: return run_kernel(norm_forward_kernel<T, 256>, p.groups, 256, s, p);
    default: return run_kernel(norm_forward_kernel<T, 1024>, p.groups, 1024, s, p);
    }
}

template <typename T>
hipError_t backward(const NormParams &p, hipStream_t s) {
    if (p.groups) {
        hipError_t e;
        switch (threads_per_row(p.cols)) {
        case 16: e = run_kernel(norm_backward_kernel<T, 16>, p.groups, 256, s, p); break;
        case 64: e = run_kernel(norm_backward_kernel<T, 64>, p.groups, 256, s, p); break;
        case 256: e = run_kernel(norm_backward_kernel<T, 256>, p.groups, 256, s, p); break;
        default: e = run_kernel(norm_backward_kernel<T, 1024>, p.groups, 1024, s, p); break;
        }
        if (e != hipSuccess) return e;
    }
    return run_kernel(norm_reduce_kernel, (2 * p.cols + 15) / 16, 1024, s, p);
}

}  // namespace

uint32_t norm_groups(uint32_t rows, uint32_t cols, uint32_t compute_units, uint32_t each) {
    const uint32_t threads = threads_per_row(cols), at_once = threads <= 64 ? 256 / threads : 1;
    const uint64_t most = (uint64_t)compute_units * (threads == 1024 ? (each + 3) / 4 : each), need = ((uint64_t)rows + at_once - 1) / at_once;
    return (uint32_t)(need < most ? need : most);
}

hipError_t launch_norm_forward(const NormParams &p, uint32_t dtype, hipStream_t s) {
    return dtype == BL_F32 ? forward<float>(p, s) : dtype == BL_F16 ? forward<_Float16>(p, s) : forward<__bf16>(p, s);
}

hipError_t launch_norm_backward(const NormParams &p, uint32_t dtype, hipStream_t s) {
    return dtype == BL_F32 ? backward<float>(p, s) : dtype == BL_F16 ? backward<_Float16>(p, s) : backward<__bf16>(p, s);
}

}  // namespace bl
