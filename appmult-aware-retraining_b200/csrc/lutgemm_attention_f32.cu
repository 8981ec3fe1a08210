// Attention of fp32 operands on the fp32 pipes: heads of 72 to 128 values, whose three planes of 16 bits would not fit shared memory.
//
// A block has 64 packed rows (or 64 keys, for grad_k and grad_v) and goes over tiles of 64 keys (rows), 16 x 16 threads with 4 x 4 scores
// each: S = Q K^T from shared memory, mask, maximum and sum over the 16 threads of a row by shuffles, P to shared memory, O += P V
// in registers.  Gradients in two kernels like those on the tensor cores, scores formed once more in each, so that no sum is
// atomic.  The fp32 pipes bound it: per value of a product two reads from shared memory serve sixteen multiply-adds.
// 2 x 1024 tokens, 16 / 4 heads of 128: 1276 us forward (13.5 TFLOP/s), 5638 backward; as planes, heads of 64 take 79 and 330.
#include "lutgemm.h"
#include "lutgemm_attention.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

constexpr int kT = 64;        // rows and keys of a tile
constexpr int kThreads = 256; // 16 x 16, each with 4 x 4 scores

__device__ __forceinline__ const float *row_ptr(const AttnTensor &t, int b, int i, int h) {
    return reinterpret_cast<const float *>(t.p) + b * t.sb + i * t.st + h * t.sh;
}

// the 64 rows from m0 on (packed rows of key head g) of a query-side operand, as fp32, rows DP + 4 apart; zeros beyond the end
// and for padding
template <int DP>
__device__ __forceinline__ void load_rows(float *dst, const AttnProblem &p, const AttnTensor &t, int b, int g, int m0) {
    for (int idx = threadIdx.x; idx < kT * DP; idx += kThreads) {
        const int r = idx / DP, d = idx - r * DP, m = m0 + r;
        float x = 0.f;
        if (m < p.M && d < p.D) {
            const int i = m / p.R, h = g * p.R + m - i * p.R;
            if (!p.doc_q || p.doc_q[b * p.doc_q_sb + i] >= 0) x = row_ptr(t, b, i, h)[d];
        }
        dst[r * (DP + 4) + d] = x;
    }
}
template <int DP>
__device__ __forceinline__ void load_keys(float *dst, const AttnProblem &p, const AttnTensor &t, int b, int g, int j0) {
    for (int idx = threadIdx.x; idx < kT * DP; idx += kThreads) {
        const int r = idx / DP, d = idx - r * DP, j = j0 + r;
        float x = 0.f;
        if (j < p.Tk && d < p.D && (!p.doc_k || p.doc_k[b * p.doc_k_sb + j] >= 0)) x = row_ptr(t, b, j, g)[d];
        dst[r * (DP + 4) + d] = x;
    }
}

// acc[i][j] = sum_d A[ty*4 + i][d] * B[tx + 16*j][d]
template <int DP>
__device__ __forceinline__ void products(float (&acc)[4][4], const float *A, const float *B, int ty, int tx) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        float4 a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4 *>(A + (ty * 4 + i) * (DP + 4) + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4 *>(B + (tx + 16 * j) * (DP + 4) + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] += a[i].x * b[j].x + a[i].y * b[j].y + a[i].z * b[j].z + a[i].w * b[j].w;
    }
}

// acc[i][c] += sum_n P[ty*4 + i][n] * V[n][tx*4 + 64*c ..]
template <int DP>
__device__ __forceinline__ void mix(float4 (&acc)[4][DP / 64], const float *P, const float *V, int ty, int tx) {
#pragma unroll 2
    for (int n = 0; n < kT; n += 4) {
        float4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float4 *>(P + (ty * 4 + i) * (kT + 4) + n);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const float4 v = *reinterpret_cast<const float4 *>(V + (n + e) * (DP + 4) + tx * 4 + 64 * c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float s = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
                    acc[i][c].x += s * v.x; acc[i][c].y += s * v.y; acc[i][c].z += s * v.z; acc[i][c].w += s * v.w;
                }
            }
    }
}
// acc[i][c] += sum_m P[m][ty*4 + i] * X[m][tx*4 + 64*c ..]
template <int DP>
__device__ __forceinline__ void mix_transposed(float4 (&acc)[4][DP / 64], const float *P, const float *X, int ty, int tx) {
#pragma unroll 4
    for (int m = 0; m < kT; ++m) {
        const float4 w = *reinterpret_cast<const float4 *>(P + m * (kT + 4) + ty * 4);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float4 x = *reinterpret_cast<const float4 *>(X + m * (DP + 4) + tx * 4 + 64 * c);
            const float s[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[i][c].x += s[i] * x.x; acc[i][c].y += s[i] * x.y; acc[i][c].z += s[i] * x.z; acc[i][c].w += s[i] * x.w;
            }
        }
    }
}

// keys that any row of a tile can see, causal masks only: [0, end)
__device__ __forceinline__ int key_end(const AttnProblem &p, int b, int m0) {
    if (!p.causal) return p.Tk;
    const int last = min(m0 + kT, p.M) - 1;
    int end = last / p.R + p.shift + 1;
    if (p.prefix) end = max(end, p.prefix[b]);
    return max(0, min(end, p.Tk));
}

struct RowInfo {
    int place, doc;
    float slope;
    bool in;
};
__device__ __forceinline__ RowInfo row_info(const AttnProblem &p, int b, int g, int m) {
    RowInfo r{0, -1, 0.f, m < p.M};
    if (r.in) {
        const int i = m / p.R, h = g * p.R + m - i * p.R;
        r.place = i + p.shift;
        if (p.doc_q) r.doc = p.doc_q[b * p.doc_q_sb + i];
        if (p.slopes) r.slope = p.slopes[h] * kLog2e;
    }
    return r;
}
// the score in units of log 2, and by `bend` the derivative of the cap
__device__ __forceinline__ float logit(const AttnProblem &p, float dot, float slope, int away, float *bend) {
    float s = dot * p.scale;
    *bend = 1.f;
    if (p.cap > 0.f) {
        const float t = tanhf(s / p.cap);
        s = p.cap * t;
        *bend = 1.f - t * t;
    }
    s *= kLog2e;
    if (p.slopes) s -= slope * (float)away;
    return s;
}

template <int DP>
__global__ void __launch_bounds__(kThreads) attention_f32_kernel(const AttnProblem p, float *out, float *lse) {
    extern __shared__ float4 smem4[];
    float *Q = reinterpret_cast<float *>(smem4), *K = Q + kT * (DP + 4), *V = K + kT * (DP + 4), *P = V + kT * (DP + 4);
    const int b = blockIdx.z, g = blockIdx.y, m0 = (gridDim.x - 1 - blockIdx.x) * kT, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    load_rows<DP>(Q, p, p.q, b, g, m0);
    RowInfo row[4];
    float most[4], sum[4];
    float4 acc[4][DP / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        row[i] = row_info(p, b, g, m0 + ty * 4 + i);
        most[i] = -INFINITY;
        sum[i] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int end = key_end(p, b, m0), pre = p.prefix ? p.prefix[b] : 0;
    for (int j0 = 0; j0 < end; j0 += kT) {
        __syncthreads();
        load_keys<DP>(K, p, p.k, b, g, j0);
        load_keys<DP>(V, p, p.v, b, g, j0);
        __syncthreads();
        float s[4][4];
        products<DP>(s, Q, K, ty, tx);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = most[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = j0 + tx + 16 * j;
                const int dk = p.doc_k && key < p.Tk ? p.doc_k[b * p.doc_k_sb + key] : -1;
                const bool ok = row[i].in && key < p.Tk &&
                                attn_sees(p.causal, p.doc_k != nullptr, row[i].place, key, pre, row[i].doc, dk);
                float bend;
                s[i][j] = ok ? logit(p, s[i][j], row[i].slope, abs(row[i].place - key), &bend) : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float base = top == -INFINITY ? 0.f : top, keep = exp2f(most[i] - base);
            most[i] = top;
            float add = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = exp2f(s[i][j] - base);
                add += e;
                P[(ty * 4 + i) * (kT + 4) + tx + 16 * j] = e;
            }
            sum[i] = sum[i] * keep + add;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) { acc[i][c].x *= keep; acc[i][c].y *= keep; acc[i][c].z *= keep; acc[i][c].w *= keep; }
        }
        __syncthreads();
        mix<DP>(acc, P, V, ty, tx);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty * 4 + i;
#pragma unroll
        for (int d = 8; d; d >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
        if (m >= p.M) continue;
        const float inv = sum[i] > 0.f ? 1.f / sum[i] : sum[i] == 0.f ? 0.f : NAN;
        const int q = m / p.R, h = g * p.R + m - q * p.R;
        float *o = out + (((size_t)b * p.Tq + q) * p.H + h) * p.D;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float v[4] = {acc[i][c].x, acc[i][c].y, acc[i][c].z, acc[i][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = tx * 4 + 64 * c + e;
                if (d < p.D) o[d] = v[e] * inv;
            }
        }
        if (tx == 0) lse[((size_t)b * p.G + g) * p.M + m] = sum[i] == 0.f ? INFINITY : most[i] + log2f(sum[i]);
    }
}

// P and dS of one tile into shared memory; `go` rows and statistics of the rows, the tile's keys from j0 on
template <int DP>
__device__ __forceinline__ void tile_gradients(const AttnProblem &p, const float *Q, const float *K, const float *V, const float *GO,
                                               float *P, float *DS, const float *lse, const float *delta, int b, int g, int m0,
                                               int j0, int pre, int ty, int tx) {
    float s[4][4], gp[4][4];
    products<DP>(s, Q, K, ty, tx);
    products<DP>(gp, GO, V, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty * 4 + i;
        const RowInfo row = row_info(p, b, g, m);
        const float l = row.in ? lse[((size_t)b * p.G + g) * p.M + m] : INFINITY, dl = row.in ? delta[((size_t)b * p.G + g) * p.M + m] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int key = j0 + tx + 16 * j;
            const int dk = p.doc_k && key < p.Tk ? p.doc_k[b * p.doc_k_sb + key] : -1;
            const bool ok = row.in && key < p.Tk && attn_sees(p.causal, p.doc_k != nullptr, row.place, key, pre, row.doc, dk);
            float bend;
            const float x = logit(p, s[i][j], row.slope, abs(row.place - key), &bend);
            const float w = ok ? exp2f(x - l) : 0.f;
            if (P) P[(ty * 4 + i) * (kT + 4) + tx + 16 * j] = w;
            DS[(ty * 4 + i) * (kT + 4) + tx + 16 * j] = ok ? w * (gp[i][j] - dl) * bend * p.scale : 0.f;
        }
    }
}

template <int DP>
__global__ void __launch_bounds__(kThreads) attention_f32_grad_q_kernel(const AttnProblem p, const AttnTensor go, const float *out,
                                                                        const float *lse, float *delta, float *gq) {
    extern __shared__ float4 smem4[];
    float *Q = reinterpret_cast<float *>(smem4), *K = Q + kT * (DP + 4), *V = K + kT * (DP + 4), *GO = V + kT * (DP + 4),
          *DS = GO + kT * (DP + 4);
    const int b = blockIdx.z, g = blockIdx.y, m0 = (gridDim.x - 1 - blockIdx.x) * kT, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    load_rows<DP>(Q, p, p.q, b, g, m0);
    load_rows<DP>(GO, p, go, b, g, m0);
    __syncthreads();
    // delta = sum_d grad_o * o, four threads to a row
    {
        const int r = threadIdx.x >> 2, m = m0 + r;
        float s = 0.f;
        if (m < p.M) {
            const int i = m / p.R, h = g * p.R + m - i * p.R;
            const float *o = out + (((size_t)b * p.Tq + i) * p.H + h) * p.D;
            for (int d = threadIdx.x & 3; d < p.D; d += 4) s += o[d] * GO[r * (DP + 4) + d];
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if (m < p.M && (threadIdx.x & 3) == 0) delta[((size_t)b * p.G + g) * p.M + m] = s;
    }
    float4 acc[4][DP / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int end = key_end(p, b, m0), pre = p.prefix ? p.prefix[b] : 0;
    for (int j0 = 0; j0 < end; j0 += kT) {
        __syncthreads();
        load_keys<DP>(K, p, p.k, b, g, j0);
        load_keys<DP>(V, p, p.v, b, g, j0);
        __syncthreads();
        tile_gradients<DP>(p, Q, K, V, GO, nullptr, DS, lse, delta, b, g, m0, j0, pre, ty, tx);
        __syncthreads();
        mix<DP>(acc, DS, K, ty, tx);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty * 4 + i;
        if (m >= p.M) continue;
        const int q = m / p.R, h = g * p.R + m - q * p.R;
        float *o = gq + (((size_t)b * p.Tq + q) * p.H + h) * p.D;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float v[4] = {acc[i][c].x, acc[i][c].y, acc[i][c].z, acc[i][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = tx * 4 + 64 * c + e;
                if (d < p.D) o[d] = v[e];
            }
        }
    }
}

template <int DP>
__global__ void __launch_bounds__(kThreads) attention_f32_grad_kv_kernel(const AttnProblem p, const AttnTensor go, const float *lse,
                                                                         const float *delta, float *gk, float *gv) {
    extern __shared__ float4 smem4[];
    float *Q = reinterpret_cast<float *>(smem4), *K = Q + kT * (DP + 4), *V = K + kT * (DP + 4), *GO = V + kT * (DP + 4),
          *DS = GO + kT * (DP + 4), *P = DS + kT * (kT + 4);
    const int b = blockIdx.z, g = blockIdx.y, j0 = blockIdx.x * kT, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    load_keys<DP>(K, p, p.k, b, g, j0);
    load_keys<DP>(V, p, p.v, b, g, j0);
    float4 ak[4][DP / 64], av[4][DP / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) ak[i][c] = av[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int pre = p.prefix ? p.prefix[b] : 0;
    // rows that can see the tile's first key
    int first = 0;
    if (p.causal && j0 >= pre) first = max(0, j0 - p.shift) * p.R / kT * kT;
    for (int m0 = first; m0 < p.M; m0 += kT) {
        __syncthreads();
        load_rows<DP>(Q, p, p.q, b, g, m0);
        load_rows<DP>(GO, p, go, b, g, m0);
        __syncthreads();
        tile_gradients<DP>(p, Q, K, V, GO, P, DS, lse, delta, b, g, m0, j0, pre, ty, tx);
        __syncthreads();
        mix_transposed<DP>(av, P, GO, ty, tx);
        mix_transposed<DP>(ak, DS, Q, ty, tx);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = j0 + ty * 4 + i;
        if (j >= p.Tk) continue;
        const size_t at = (((size_t)b * p.Tk + j) * p.G + g) * p.D;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
            const float x[4] = {ak[i][c].x, ak[i][c].y, ak[i][c].z, ak[i][c].w}, y[4] = {av[i][c].x, av[i][c].y, av[i][c].z, av[i][c].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = tx * 4 + 64 * c + e;
                if (d < p.D) { gk[at + d] = x[e]; gv[at + d] = y[e]; }
            }
        }
    }
}

template <int DP>
int forward(const AttnProblem &p, float *out, float *lse, cudaStream_t stream) {
    const size_t smem = sizeof(float) * (3 * kT * (DP + 4) + kT * (kT + 4));
    if (!cuda_ok(cudaFuncSetAttribute(attention_f32_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem))) return LUTGEMM_E_CUDA;
    attention_f32_kernel<DP><<<dim3((p.M + kT - 1) / kT, p.G, p.B), kThreads, smem, stream>>>(p, out, lse);
    return launch_status();
}
template <int DP>
int backward(const AttnProblem &p, const AttnTensor &go, const float *out, const float *lse, float *delta, float *gq, float *gk, float *gv,
             cudaStream_t stream) {
    const size_t smem_q = sizeof(float) * (4 * kT * (DP + 4) + kT * (kT + 4)), smem_kv = sizeof(float) * (4 * kT * (DP + 4) + 2 * kT * (kT + 4));
    if (!cuda_ok(cudaFuncSetAttribute(attention_f32_grad_q_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_q)) ||
        !cuda_ok(cudaFuncSetAttribute(attention_f32_grad_kv_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_kv)))
        return LUTGEMM_E_CUDA;
    if (p.M > 0) {
        attention_f32_grad_q_kernel<DP><<<dim3((p.M + kT - 1) / kT, p.G, p.B), kThreads, smem_q, stream>>>(
            p, go, out, lse, delta, gq);
        const int rc = launch_status();
        if (rc != LUTGEMM_OK) return rc;
    }
    if (p.Tk > 0) {
        attention_f32_grad_kv_kernel<DP><<<dim3((p.Tk + kT - 1) / kT, p.G, p.B), kThreads, smem_kv, stream>>>(
            p, go, lse, delta, gk, gv);
        return launch_status();
    }
    return LUTGEMM_OK;
}

}  // namespace

int attention_f32_forward(const AttnProblem &p, float *out, float *lse, cudaStream_t stream) {
    return forward<128>(p, out, lse, stream);
}

int attention_f32_backward(const AttnProblem &p, const AttnTensor &go, const float *out, const float *lse, float *delta, float *gq, float *gk,
                           float *gv, cudaStream_t stream) {
    return backward<128>(p, go, out, lse, delta, gq, gk, gv, stream);
}

}  // namespace lutgemm
