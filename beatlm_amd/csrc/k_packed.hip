// Attention over packed documents and its gradients (include/beatlm_ops.h).
//
// The plain form of the kernels: one workgroup per (query row, head), keys in
// chunks of a workgroup's threads, all arithmetic f32.
#include "packed_device.hpp"

namespace bl {

namespace {

constexpr int THREADS = 128;
constexpr int MAX_D = BL_ATTENTION_MAX_HEAD_DIM;
constexpr float LOWEST = -INFINITY;

__device__ __forceinline__ float block_sum(float v, float *lds) {
    v = wave_sum(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    return lds[0] + lds[1];
}
__device__ __forceinline__ float block_max(float v, float *lds) {
    v = wave_max(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    return fmaxf(lds[0], lds[1]);
}

template <typename T>
__device__ __forceinline__ const T *at(const bl_heads &h, int64_t row, int64_t head) {
    return (const T *)h.data + row * (int64_t)h.row_stride + head * (int64_t)h.head_stride;
}

template <typename T>
__device__ __forceinline__ float dot(const float *q, const T *k, int d) {
    float s = 0.0f;
    for (int c = 0; c < d; c++) s += q[c] * (float)k[c];
    return s;
}

// The score of a pair, and tanh of the capped one.
__device__ __forceinline__ float score(const bl_packed_attention_args &a, const Document &doc, int head, int i, int j, float qk, float &th) {
    float s = qk * a.scale;
    th = 0.0f;
    if (a.softcap > 0.0f) {
        th = tanhf(s / a.softcap);
        s = a.softcap * th;
    }
    if (a.slopes) s -= a.slopes[head] * distance_of(a, doc, i, j);
    return s;
}

template <typename T>
__global__ __launch_bounds__(THREADS) void forward_kernel(PackedParams p) {
    const bl_packed_attention_args &a = p.a;
    __shared__ float q[MAX_D], prob[THREADS], red[2];
    const int row = blockIdx.x, head = blockIdx.y, d = a.head_dim, t = threadIdx.x;
    const int index = document_at(a.q_offsets, a.documents, row);
    if (index < 0) return;
    const Document doc = document_of(a, index);
    const int i = row - doc.q0;
    const int kv = head / (a.q_heads / a.kv_heads);
    if (t < d) q[t] = (float)at<T>(a.q, row, head)[t];
    __syncthreads();
    float m = LOWEST, l = 0.0f, o = 0.0f;
    for (int j0 = 0; j0 < doc.n_k; j0 += THREADS) {
        const int j = j0 + t;
        float s = LOWEST, th;
        if (j < doc.n_k && visible(a, doc, i, j)) s = score(a, doc, head, i, j, dot<T>(q, at<T>(a.k, doc.k0 + j, kv), d), th);
        // A chunk that is hidden whole leaves the maximum where it was; a NaN
        // is no maximum, but its probability is NaN and so is the row's.
        const float top = fmaxf(m, block_max(s, red));
        const float base = top == LOWEST ? 0.0f : top;
        const float e = s == LOWEST ? 0.0f : expf(s - base);
        const float carry = m == LOWEST ? 1.0f : expf(m - base);
        prob[t] = e;
        l = l * carry + block_sum(e, red);
        m = top;
        if (t < d) {
            o *= carry;
            for (int x = 0; x < THREADS && j0 + x < doc.n_k; x++)
                if (prob[x] != 0.0f) o += prob[x] * (float)at<T>(a.v, doc.k0 + j0 + x, kv)[t];
        }
        __syncthreads();
    }
    if (t < d) ((T *)at<T>(a.out, row, head))[t] = (T)(l == 0.0f ? 0.0f : o / l);
    if (t == 0 && a.lse) a.lse[(int64_t)head * a.q_rows + row] = l == 0.0f ? LOWEST : m + logf(l);
}

// d_q, and each row's delta (sum_j P_ij dP_ij) and part of d_slopes.
template <typename T>
__global__ __launch_bounds__(THREADS) void backward_q_kernel(PackedParams p) {
    const bl_packed_attention_args &a = p.a;
    __shared__ float q[MAX_D], g[MAX_D], ds[THREADS], red[2];
    const int row = blockIdx.x, head = blockIdx.y, d = a.head_dim, t = threadIdx.x;
    const int64_t stat = (int64_t)head * a.q_rows + row;
    const int index = document_at(a.q_offsets, a.documents, row);
    if (index < 0) {
        if (t == 0 && p.d_slope) p.d_slope[stat] = 0.0f;
        return;
    }
    const Document doc = document_of(a, index);
    const int i = row - doc.q0;
    const int kv = head / (a.q_heads / a.kv_heads);
    if (t < d) {
        q[t] = (float)at<T>(a.q, row, head)[t];
        g[t] = (float)at<T>(p.g.d_out, row, head)[t];
    }
    __syncthreads();
    const float lse = a.lse[stat];
    float delta = 0.0f, slope = 0.0f, dq = 0.0f;
    for (int pass = 0; pass < 2; pass++) {
        float part = 0.0f;
        for (int j0 = 0; j0 < doc.n_k; j0 += THREADS) {
            const int j = j0 + t;
            float v = 0.0f;
            if (j < doc.n_k && lse != LOWEST && visible(a, doc, i, j)) {
                float th;
                const float s = score(a, doc, head, i, j, dot<T>(q, at<T>(a.k, doc.k0 + j, kv), d), th);
                const float pr = expf(s - lse), dp = dot<T>(g, at<T>(a.v, doc.k0 + j, kv), d);
                if (pass == 0) part += pr * dp;
                else {
                    v = pr * (dp - delta);
                    if (a.slopes) part -= v * distance_of(a, doc, i, j);
                    if (a.softcap > 0.0f) v *= 1.0f - th * th;
                    v *= a.scale;
                }
            }
            if (pass == 0) continue;
            ds[t] = v;
            __syncthreads();
            if (t < d)
                for (int x = 0; x < THREADS && j0 + x < doc.n_k; x++)
                    if (ds[x] != 0.0f) dq += ds[x] * (float)at<T>(a.k, doc.k0 + j0 + x, kv)[t];
            __syncthreads();
        }
        if (pass == 0) delta = block_sum(part, red);
        else slope = block_sum(part, red);
    }
    if (t < d) ((T *)at<T>(p.g.d_q, row, head))[t] = (T)dq;
    if (t == 0) {
        p.delta[stat] = delta;
        if (p.d_slope) p.d_slope[stat] = slope;
    }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void backward_kv_kernel(PackedParams p) {
    const bl_packed_attention_args &a = p.a;
    __shared__ float k[MAX_D], v[MAX_D], ds[THREADS], pr[THREADS];
    const int row = blockIdx.x, kv = blockIdx.y, d = a.head_dim, t = threadIdx.x;
    const int index = document_at(a.k_begin, a.documents, row);
    if (index < 0) return;
    const Document doc = document_of(a, index);
    const int j = row - doc.k0, group = a.q_heads / a.kv_heads;
    if (t < d) {
        k[t] = (float)at<T>(a.k, row, kv)[t];
        v[t] = (float)at<T>(a.v, row, kv)[t];
    }
    __syncthreads();
    float dk = 0.0f, dv = 0.0f;
    for (int head = kv * group; head < (kv + 1) * group; head++)
        for (int i0 = 0; i0 < doc.n_q; i0 += THREADS) {
            const int i = i0 + t;
            const int64_t stat = (int64_t)head * a.q_rows + doc.q0 + i;
            float x = 0.0f, y = 0.0f;
            if (i < doc.n_q && visible(a, doc, i, j) && a.lse[stat] != LOWEST) {
                float th;
                const float s = score(a, doc, head, i, j, dot<T>(k, at<T>(a.q, doc.q0 + i, head), d), th);
                y = expf(s - a.lse[stat]);
                x = y * (dot<T>(v, at<T>(p.g.d_out, doc.q0 + i, head), d) - p.delta[stat]) * a.scale;
                if (a.softcap > 0.0f) x *= 1.0f - th * th;
            }
            ds[t] = x;
            pr[t] = y;
            __syncthreads();
            if (t < d)
                for (int n = 0; n < THREADS && i0 + n < doc.n_q; n++)
                    if (pr[n] != 0.0f) {
                        dk += ds[n] * (float)at<T>(a.q, doc.q0 + i0 + n, head)[t];
                        dv += pr[n] * (float)at<T>(p.g.d_out, doc.q0 + i0 + n, head)[t];
                    }
            __syncthreads();
        }
    if (t < d) {
        ((T *)at<T>(p.g.d_k, row, kv))[t] = (T)dk;
        ((T *)at<T>(p.g.d_v, row, kv))[t] = (T)dv;
    }
}

// d_slopes: a head's rows added by one workgroup, in a fixed order.
__global__ __launch_bounds__(THREADS) void slopes_kernel(PackedParams p) {
    __shared__ float red[2];
    const int64_t head = blockIdx.x;
    float s = 0.0f;
    for (int row = threadIdx.x; row < (int)p.a.q_rows; row += THREADS) s += p.d_slope[head * p.a.q_rows + row];
    s = block_sum(s, red);
    if (threadIdx.x == 0) p.g.d_slopes[head] = s;
}

template <typename T>
hipError_t forward(const PackedParams &p, hipStream_t s) {
    forward_kernel<T><<<dim3(p.a.q_rows, p.a.q_heads), THREADS, 0, s>>>(p);
    return hipGetLastError();
}

template <typename T>
hipError_t backward(const PackedParams &p, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (p.a.q_rows) {
        backward_q_kernel<T><<<dim3(p.a.q_rows, p.a.q_heads), THREADS, 0, s>>>(p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (p.a.k_rows) {
        backward_kv_kernel<T><<<dim3(p.a.k_rows, p.a.kv_heads), THREADS, 0, s>>>(p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (p.g.d_slopes) {
        slopes_kernel<<<p.a.q_heads, THREADS, 0, s>>>(p);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

PackedPlan plan_packed(const bl_packed_attention_args &a, uint32_t compute_units) {
    (void)compute_units;
    PackedPlan plan;
    plan.forward_bytes = 0;
    plan.backward_bytes = 2ull * a.q_heads * a.q_rows * sizeof(float);
    return plan;
}

hipError_t launch_packed_forward(const PackedParams &p, const PackedPlan &, hipStream_t s) {
    switch (p.a.dtype) {
    case BL_F32: return forward<float>(p, s);
    case BL_F16: return forward<_Float16>(p, s);
    default: return forward<__bf16>(p, s);
    }
}

hipError_t launch_packed_backward(const PackedParams &q, const PackedPlan &, hipStream_t s) {
    PackedParams p = q;
    p.delta = (float *)p.a.workspace;
    p.d_slope = p.g.d_slopes ? p.delta + (uint64_t)p.a.q_heads * p.a.q_rows : nullptr;
    switch (p.a.dtype) {
    case BL_F32: return backward<float>(p, s);
    case BL_F16: return backward<_Float16>(p, s);
    default: return backward<__bf16>(p, s);
    }
}

}  // namespace bl
