// LayerNorm over strided rows and its gradients (include/beatlm_ops.h).
//
// Both directions read each row once: TPR threads (one wave, four or sixteen)
// keep it in registers, so the variance is the mean of squares about the mean
// (two passes over registers, no cancellation) and nothing is read twice. The
// bound is HBM: forward x in, y out; backward x and dy in, dx out.
//
// The weights' gradients are sums over rows: a workgroup of the backward walks
// rows with a stride of the grid and keeps its columns' two sums in registers;
// its partial sums go to the workspace and a second launch adds the groups'
// in order. No atomics, so the order of the sums is fixed.
#include "ops_device.hpp"

namespace bl {

namespace {

template <int TPR> constexpr int norm_threads = TPR == 64 ? 256 : TPR;  // of a workgroup

template <int TPR, int VEC, int EPT> struct NormShape {
    static constexpr int N = EPT / VEC;                     // chunks a thread holds
    static constexpr int THREADS = norm_threads<TPR>;
    static constexpr int ROWS = THREADS / TPR;              // rows at once
    static constexpr int WAVES = TPR / 64;                  // waves of one row
    static __device__ __forceinline__ uint32_t col(int lane, int n) { return (uint32_t)(n * TPR + lane) * VEC; }
};

// Sums of K values over the TPR threads of a row, in every one of them.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float *lds) {
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = wave_sum(v[k]);
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

template <typename T, int TPR, int VEC, int EPT>
__global__ __launch_bounds__(norm_threads<TPR>) void norm_forward_kernel(NormParams p) {
    using S = NormShape<TPR, VEC, EPT>;
    __shared__ float lds[S::WAVES];
    const int lane = threadIdx.x % TPR;
    const uint32_t row = blockIdx.x * S::ROWS + threadIdx.x / TPR;
    if (row >= p.rows) return;  // whole waves of a one-wave row; no barrier follows for those
    const T *x = (const T *)p.x + (uint64_t)row * p.x_stride;
    float v[S::N][VEC];
    float sum[1] = {0.0f};
#pragma unroll
    for (int n = 0; n < S::N; n++) {
        const uint32_t c = S::col(lane, n);
        if (c < p.cols) {
            load_vec<T, VEC>(x + c, v[n]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) v[n][e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) sum[0] += v[n][e];
    }
    row_sums<TPR, 1>(sum, lds);
    const float mean = sum[0] / (float)p.cols;
    float square[1] = {0.0f};
#pragma unroll
    for (int n = 0; n < S::N; n++) {
        const bool in = S::col(lane, n) < p.cols;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            v[n][e] -= mean;
            if (in) square[0] += v[n][e] * v[n][e];
        }
    }
    row_sums<TPR, 1>(square, lds);
    const float rstd = 1.0f / sqrtf(square[0] / (float)p.cols + p.epsilon);
    if (lane == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
    }
    T *y = (T *)p.y + (uint64_t)row * p.y_stride;
#pragma unroll
    for (int n = 0; n < S::N; n++) {
        const uint32_t c = S::col(lane, n);
        if (c >= p.cols) continue;
        float g[VEC], b[VEC];
        load_vec<T, VEC>((const T *)p.gamma + c, g);
        load_vec<T, VEC>((const T *)p.beta + c, b);
#pragma unroll
        for (int e = 0; e < VEC; e++) v[n][e] = v[n][e] * rstd * g[e] + b[e];
        store_vec<T, VEC>(y + c, v[n]);
    }
}

template <typename T, int TPR, int VEC, int EPT>
__global__ __launch_bounds__(norm_threads<TPR>) void norm_backward_kernel(NormParams p) {
    using S = NormShape<TPR, VEC, EPT>;
    __shared__ float lds[TPR == 64 ? 2 * S::ROWS * 64 * EPT : 2 * S::WAVES];
    const int lane = threadIdx.x % TPR;
    float g[S::N][VEC], dg[S::N][VEC], db[S::N][VEC];
#pragma unroll
    for (int n = 0; n < S::N; n++) {
        const uint32_t c = S::col(lane, n);
#pragma unroll
        for (int e = 0; e < VEC; e++) g[n][e] = dg[n][e] = db[n][e] = 0.0f;
        if (c < p.cols) load_vec<T, VEC>((const T *)p.gamma + c, g[n]);
    }
    const float each = 1.0f / (float)p.cols;
    for (uint32_t row = blockIdx.x * S::ROWS + threadIdx.x / TPR; row < p.rows; row += gridDim.x * S::ROWS) {
        const T *x = (const T *)p.x + (uint64_t)row * p.x_stride;
        const T *dy = (const T *)p.dy + (uint64_t)row * p.dy_stride;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float n_[S::N][VEC], d[S::N][VEC];
        float sums[2] = {0.0f, 0.0f};  // of g and of g n
#pragma unroll
        for (int n = 0; n < S::N; n++) {
            const uint32_t c = S::col(lane, n);
            if (c < p.cols) {
                load_vec<T, VEC>(x + c, n_[n]);
                load_vec<T, VEC>(dy + c, d[n]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++) n_[n][e] = mean, d[n][e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                n_[n][e] = (n_[n][e] - mean) * rstd;
                dg[n][e] += d[n][e] * n_[n][e];
                db[n][e] += d[n][e];
                d[n][e] *= g[n][e];
                sums[0] += d[n][e];
                sums[1] += d[n][e] * n_[n][e];
            }
        }
        row_sums<TPR, 2>(sums, lds);
        const float m0 = sums[0] * each, m1 = sums[1] * each;
        T *dx = (T *)p.dx + (uint64_t)row * p.dx_stride;
#pragma unroll
        for (int n = 0; n < S::N; n++) {
            const uint32_t c = S::col(lane, n);
            if (c >= p.cols) continue;
#pragma unroll
            for (int e = 0; e < VEC; e++) d[n][e] = (d[n][e] - m0 - n_[n][e] * m1) * rstd;
            store_vec<T, VEC>(dx + c, d[n]);
        }
    }
    // The workgroup's partial sums; of one-wave rows, the waves' added first.
    float *out = p.partial + (uint64_t)blockIdx.x * 2 * p.cols;
    if constexpr (TPR == 64) {
        const int wave = threadIdx.x / 64;
#pragma unroll
        for (int n = 0; n < S::N; n++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                lds[(wave * 2 + 0) * 64 * EPT + S::col(lane, n) + e] = dg[n][e];
                lds[(wave * 2 + 1) * 64 * EPT + S::col(lane, n) + e] = db[n][e];
            }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < 2 * 64 * EPT; i += S::THREADS) {
            const uint32_t which = i / (64 * EPT), c = i % (64 * EPT);
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < S::ROWS; w++) s += lds[(w * 2 + which) * 64 * EPT + c];
            if (c < p.cols) out[which * p.cols + c] = s;
        }
    } else {
#pragma unroll
        for (int n = 0; n < S::N; n++) {
            const uint32_t c = S::col(lane, n);
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (c < p.cols) {
                    out[c + e] = dg[n][e];
                    out[p.cols + c + e] = db[n][e];
                }
        }
    }
}

// d_gamma and d_beta from the groups' partial sums: 64 columns a workgroup,
// its 16 waves taking every 16th group.
__global__ __launch_bounds__(1024) void norm_reduce_kernel(NormParams p) {
    __shared__ float lds[16][64];
    const uint32_t i = blockIdx.x * 64 + threadIdx.x % 64;  // of 2 * cols
    const int wave = threadIdx.x / 64;
    float s = 0.0f;
    if (i < 2 * p.cols)
        for (uint32_t group = wave; group < p.groups; group += 16) s += p.partial[(uint64_t)group * 2 * p.cols + i];
    lds[wave][threadIdx.x % 64] = s;
    __syncthreads();
    if (wave || i >= 2 * p.cols) return;
#pragma unroll
    for (int w = 1; w < 16; w++) s += lds[w][threadIdx.x];
    if (i < p.cols) p.d_gamma[i] = s;
    else p.d_beta[i - p.cols] = s;
}

// The threads a row of `cols` gets: a wave for up to 1024 columns (16 values a
// thread), four for up to 4096, sixteen for the rest.
uint32_t threads_per_row(uint32_t cols) { return cols <= 1024 ? 64 : cols <= 4096 ? 256 : 1024; }

template <typename T, int VEC>
hipError_t forward(const NormParams &p, hipStream_t s) {
    const uint32_t tpr = threads_per_row(p.cols);
    if (tpr == 64) {
        const uint32_t grid = (p.rows + 3) / 4;
        if (p.cols <= 512) norm_forward_kernel<T, 64, VEC, 8><<<grid, 256, 0, s>>>(p);
        else norm_forward_kernel<T, 64, VEC, 16><<<grid, 256, 0, s>>>(p);
    } else if (tpr == 256) {
        norm_forward_kernel<T, 256, VEC, 16><<<p.rows, 256, 0, s>>>(p);
    } else {
        norm_forward_kernel<T, 1024, VEC, 16><<<p.rows, 1024, 0, s>>>(p);
    }
    return hipGetLastError();
}

template <typename T, int VEC>
hipError_t backward(const NormParams &p, hipStream_t s) {
    const uint32_t tpr = threads_per_row(p.cols);
    if (p.groups) {
        if (tpr == 64) {
            if (p.cols <= 512) norm_backward_kernel<T, 64, VEC, 8><<<p.groups, 256, 0, s>>>(p);
            else norm_backward_kernel<T, 64, VEC, 16><<<p.groups, 256, 0, s>>>(p);
        } else if (tpr == 256) {
            norm_backward_kernel<T, 256, VEC, 16><<<p.groups, 256, 0, s>>>(p);
        } else {
            norm_backward_kernel<T, 1024, VEC, 16><<<p.groups, 1024, 0, s>>>(p);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    norm_reduce_kernel<<<(2 * p.cols + 63) / 64, 1024, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace

uint32_t norm_groups(uint32_t rows, uint32_t cols, uint32_t compute_units) {
    const uint32_t at_once = threads_per_row(cols) == 64 ? 4 : 1;
    const uint32_t most = threads_per_row(cols) == 1024 ? compute_units : 2 * compute_units;
    const uint32_t need = (uint32_t)(((uint64_t)rows + at_once - 1) / at_once);
    return need < most ? need : most;
}

hipError_t launch_norm_forward(const NormParams &p, uint32_t dtype, hipStream_t s) {
    switch (dtype) {
    case BL_F32: return p.vector ? forward<float, 4>(p, s) : forward<float, 1>(p, s);
    case BL_F16: return p.vector ? forward<_Float16, 8>(p, s) : forward<_Float16, 1>(p, s);
    default: return p.vector ? forward<__bf16, 8>(p, s) : forward<__bf16, 1>(p, s);
    }
}

hipError_t launch_norm_backward(const NormParams &p, uint32_t dtype, hipStream_t s) {
    switch (dtype) {
    case BL_F32: return p.vector ? backward<float, 4>(p, s) : backward<float, 1>(p, s);
    case BL_F16: return p.vector ? backward<_Float16, 8>(p, s) : backward<_Float16, 1>(p, s);
    default: return p.vector ? backward<__bf16, 8>(p, s) : backward<__bf16, 1>(p, s);
    }
}

}  // namespace bl
