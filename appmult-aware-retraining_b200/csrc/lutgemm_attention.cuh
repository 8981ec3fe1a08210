// What the attention kernels share: the problem, its masks, loads and stores of three types.
//
// Query i of row b stands at place i + Tk - Tq among the Tk keys.  Of the score s = scale * q.k the kernels form
//     b_ij = [cap * tanh(s / cap) or s] - slope_h * |place_i - j|
// and the softmax over the keys that i may see: those of its own document (ids below zero are padding, which sees and is
// seen by nothing) and, where causal, not behind place_i unless among the first prefix_b.  A query that sees nothing gives
// zeros.  Rows of padding are never multiplied: they are loaded as zeros, whatever they hold.
//
// The heads that share a key head are rows of one matrix: row m of key head g is query i = m / R of head g*R + m % R,
// R = H / G.  A tile of rows then reads its keys once for all R heads, a single query has R rows, and the gradients of a shared
// head are sums over the rows of one product.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

namespace lutgemm {

constexpr float kLog2e = 1.4426950408889634f;

// a [B, T, heads, D] operand: strides in elements, the last one 1
struct AttnTensor {
    const void *p;
    long sb, st, sh;
};

struct AttnProblem {
    AttnTensor q, k, v;
    int B, Tq, Tk, H, G, R, D;
    int M;              // rows per key head: Tq * R
    int shift;          // Tk - Tq
    float scale, cap;   // cap 0: scores as they are
    const float *slopes;  // [H] or null
    int causal;
    const int *prefix;  // [B] or null
    const int *doc_q, *doc_k;  // ids, rows doc_q_sb and doc_k_sb apart; both null or neither
    long doc_q_sb, doc_k_sb;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// whether key j of row b (document dk) is seen from `place` (document dq, prefix of the row `pre`)
__device__ __forceinline__ bool attn_sees(bool causal, bool docs, int place, int j, int pre, int dq, int dk) {
    bool ok = true;
    if (causal) ok = j <= place || j < pre;
    if (docs) ok = ok && dq == dk && dq >= 0;
    return ok;
}

}  // namespace lutgemm
