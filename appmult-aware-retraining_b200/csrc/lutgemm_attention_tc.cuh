// What the tensor-core attention kernels share: operand tiles, the masks of tiles, the walk over the tiles that matter.
#pragma once

#include "lutgemm.h"
#include "lutgemm_attention.cuh"
#include "lutgemm_tcgen.cuh"

namespace lutgemm {

constexpr int kKeyTile = 64;   // keys of a tile, and the rows of the smallest row tile
constexpr int kRowTile = 128;  // rows of a forward or query-gradient tile: the lanes of tensor memory

template <typename T>
struct IsBf16 {
    static constexpr bool value = false;
};
template <>
struct IsBf16<__nv_bfloat16> {
    static constexpr bool value = true;
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (IsBf16<T>::value)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if (IsBf16<T>::value) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// documents of a tile of 64: the smallest and largest id that is not padding (0x7fffffff, -1: none), and whether any is
struct DocRange {
    int least, most, padding, unused;
};
constexpr int kNoLeast = 0x7fffffff;

// last key that query i of row b may see for all masks but the documents
__device__ __forceinline__ int key_limit(const AttnProblem &p, int place, int pre) {
    const int lim = p.causal ? max(place, pre - 1) : p.Tk - 1;
    return min(lim, p.Tk - 1);
}

// `ROWS` rows of 64 * BLOCKS values (16-byte pieces c of a row at c ^ (row & 7)) by 128 threads; row r comes from row(r), null = zeros
template <int ROWS, int BLOCKS, typename Row>
__device__ __forceinline__ void copy_tile(uint32_t dst, int D, int thread, const void *any, Row row) {
    const int c = thread & 7;
#pragma unroll
    for (int n = 0; n < ROWS / 16; ++n) {
        const int r = (thread >> 3) + 16 * n;
        const char *src = static_cast<const char *>(row(r));
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
            const int at = k * 64 + c * 8;
            const bool real = src != nullptr && at < D;
            copy16(dst + k * ROWS * 128 + r * 128 + ((c ^ (r & 7)) << 4), real ? src + 2 * at : any, real);
        }
    }
}
// the tile of keys from j0 on
template <int BLOCKS>
__device__ __forceinline__ void copy_keys(uint32_t dst, const AttnProblem &p, const AttnTensor &t, int b, int g, int j0, int thread) {
    const char *base = static_cast<const char *>(t.p) + 2 * (b * t.sb + g * t.sh);
    copy_tile<kKeyTile, BLOCKS>(dst, p.D, thread, t.p, [&](int r) -> const void * {
        const int j = j0 + r;
        if (j >= p.Tk || (p.doc_k && p.doc_k[b * p.doc_k_sb + j] < 0)) return nullptr;
        return base + 2 * (j * t.st);
    });
}
// the ROWS packed rows from m0 on
template <int ROWS, int BLOCKS>
__device__ __forceinline__ void copy_rows(uint32_t dst, const AttnProblem &p, const AttnTensor &t, int b, int g, int m0, int thread) {
    const char *base = static_cast<const char *>(t.p) + 2 * (b * t.sb + (long)g * p.R * t.sh);
    copy_tile<ROWS, BLOCKS>(dst, p.D, thread, t.p, [&](int r) -> const void * {
        const int m = m0 + r;
        if (m >= p.M) return nullptr;
        const int i = p.R == 1 ? m : m / p.R;
        if (p.doc_q && p.doc_q[b * p.doc_q_sb + i] < 0) return nullptr;
        return base + 2 * (i * t.st + (m - i * p.R) * t.sh);
    });
}

// what a thread knows of its row
struct TileRow {
    int limit, doc;  // last key (-1: none), document
    int place;
    float slope;     // in units of log 2
};
__device__ __forceinline__ TileRow tile_row(const AttnProblem &p, int b, int g, int m, int pre) {
    TileRow r{-1, -1, 0, 0.f};
    if (m < p.M) {
        const int i = p.R == 1 ? m : m / p.R;
        r.place = i + p.shift;
        r.limit = key_limit(p, r.place, pre);
        if (p.doc_q) {
            r.doc = p.doc_q[b * p.doc_q_sb + i];
            if (r.doc < 0) r.limit = -1;
        }
        if (p.slopes) r.slope = p.slopes[g * p.R + m - i * p.R] * kLog2e;
    }
    return r;
}

// a score product in units of log 2, for capped, biased or negatively scaled scores
struct Bend {
    float scale2;      // scale * log2 e
    float in, k1, k2;  // cap: k1 - k2 / (1 + 2^(in * s)) = log2 e * cap * tanh(scale * s / cap)
};
__device__ __forceinline__ Bend make_bend(const AttnProblem &p) {
    Bend b;
    b.scale2 = p.scale * kLog2e;
    b.k1 = p.cap * kLog2e;
    b.k2 = 2.f * b.k1;
    b.in = p.cap > 0.f ? 2.f * b.scale2 / p.cap : 0.f;
    return b;
}

int *device_error_word();

// lutgemm_attention_tc.cu: ranges of the documents of tiles of 64 keys and 64 packed rows ([B][tiles] each); nullptr where nothing
// is gained by them
size_t doc_range_bytes(const AttnProblem &p);
int doc_ranges(const AttnProblem &p, DocRange *keys, DocRange *rows, cudaStream_t stream);

}  // namespace lutgemm
