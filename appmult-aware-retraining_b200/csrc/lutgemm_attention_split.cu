// fp32 operands of attention as three bf16 planes: x = x0 + x1 + x2, each the rest of the ones before rounded to bf16, 8 bits each, so
// that the sum is x up to 2^-25 of it (and to bf16's smallest subnormal, which is fp32's times 2^16).  The tensor cores then form
// products of fp32 accuracy from six products of planes.  DRAM bounds this pass: 4 bytes in and 6 out per value, one launch for all
// operands of a call; the backward pass's also forms delta, the product of grad_o and out of every row, where grad_o goes by.
#include "lutgemm.h"
#include "lutgemm_attention_tc.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

struct SplitArgs {
    SplitOperand op[4];
    long first[5];  // rows of the operands before
    int count, vectors;
    const float *out;
    float *delta;
};

// 16 lanes to a row, four values to a lane
__global__ void __launch_bounds__(256) attention_split_kernel(const AttnProblem p, const SplitArgs a) {
    const long row = blockIdx.x * 16L + (threadIdx.x >> 4);
    const int lane = threadIdx.x & 15, d = lane * 4;
    if (row >= a.first[a.count]) return;  // (whole halves of a warp)
    int k = 0;
    while (row >= a.first[k + 1]) ++k;
    const SplitOperand &o = a.op[k];
    const long at = row - a.first[k], bt = at / o.heads;
    const int h = (int)(at - bt * o.heads), b = (int)(bt / o.T), t = (int)(bt - (long)b * o.T);
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    const bool real = !o.doc || o.doc[b * o.doc_sb + t] >= 0;
    if (real && d < p.D) {
        const float *src = static_cast<const float *>(o.from.p) + b * o.from.sb + t * o.from.st + h * o.from.sh + d;
        if (a.vectors >> k & 1) {
            const float4 v = *reinterpret_cast<const float4 *>(src);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = src[e];
        }
    }
    uint32_t w[3][16];
    plane_words<float, true>(w, 0, x[0], x[1]);
    plane_words<float, true>(w, 1, x[2], x[3]);
#pragma unroll
    for (int e = 0; e < 3; ++e) *reinterpret_cast<uint2 *>(o.to + at * kPlaneWidth + 64 * e + d) = make_uint2(w[e][0], w[e][1]);
    if (k == 3) {
        float s = 0.f;
        if (real && d < p.D) {
            const float4 v = *reinterpret_cast<const float4 *>(a.out + at * p.D + d);
            s = (x[0] * v.x + x[1] * v.y) + (x[2] * v.z + x[3] * v.w);
        }
        const unsigned mask = 0xffffu << (threadIdx.x & 16);
#pragma unroll
        for (int e = 8; e; e >>= 1) s += __shfl_xor_sync(mask, s, e);
        if (lane == 0) a.delta[((long)b * p.G + h / p.R) * p.M + (long)t * p.R + h % p.R] = s;
    }
}

}  // namespace

int attention_split(const AttnProblem &p, const SplitOperand *operands, int count, const float *out, float *delta, cudaStream_t stream) {
    SplitArgs a{};
    a.count = count;
    a.out = out;
    a.delta = delta;
    for (int k = 0; k < count; ++k) {
        const SplitOperand &o = operands[k];
        a.op[k] = o;
        a.first[k + 1] = a.first[k] + (long)p.B * o.T * o.heads;
        const bool fits = !(reinterpret_cast<uintptr_t>(o.from.p) & 15) && (p.B == 1 || o.from.sb % 4 == 0) && (o.T == 1 || o.from.st % 4 == 0) &&
                          (o.heads == 1 || o.from.sh % 4 == 0);
        a.vectors |= (int)fits << k;
    }
    const long blocks = (a.first[count] + 15) / 16;
    if (blocks > 0x7fffffffL) return LUTGEMM_E_TOOLARGE;
    attention_split_kernel<<<(unsigned)blocks, 256, 0, stream>>>(p, a);
    return launch_status();
}

}  // namespace lutgemm
