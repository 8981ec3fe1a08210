// What the tensor-core attention kernels share: operand tiles, the masks of tiles, the walk over the tiles that matter.
#pragma once

#include "lutgemm.h"
#include "lutgemm_attention.cuh"
#include "lutgemm_f32x2.cuh"
#include "lutgemm_tcgen.cuh"
#include "lutgemm_tma.cuh"

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

// How the tensor cores take operands of a type.  16-bit ones as they are; a tile's blocks are then blocks of 64 values of the head.  fp32
// ones as three bf16 planes whose sum they are (8 bits each; attention_split writes them), heads of up to 64 values: the blocks
// are the planes, and a product is the six products of planes that reach 2^-24 of it, the small ones first.
template <typename T, int DP>
struct Operand {
    using Type = T;
    static constexpr bool kPlanes = false, kBf16 = IsBf16<T>::value;
    static constexpr int kBlocks = DP / 64, kProducts = DP / 64;
    __host__ __device__ static constexpr int a(int i) { return i; }
    __host__ __device__ static constexpr int b(int i) { return i; }
};
template <int DP>
struct Operand<float, DP> {
    using Type = __nv_bfloat16;
    static constexpr bool kPlanes = true, kBf16 = true;
    static constexpr int kBlocks = 3, kProducts = 6;
    __host__ __device__ static constexpr int a(int i) { return i == 0 ? 2 : i == 2 || i == 3 ? 1 : 0; }
    __host__ __device__ static constexpr int b(int i) { return i == 1 ? 2 : i == 2 || i == 4 ? 1 : 0; }
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
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    uint32_t r;
    if (IsBf16<T>::value)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
    if (IsBf16<T>::value) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// Two values as words of the planes of their type (one of 16-bit types), for half a word row each.  OPERAND: any finite fp32 values; those
// that would round to an infinity of bf16 take its largest value, and the other planes what is left.
template <typename T, bool OPERAND = false, int N>
__device__ __forceinline__ void plane_words(uint32_t (&w)[N][16], int at, float a, float b) {
    using O = typename Operand<T, 64>::Type;
    if constexpr (OPERAND) {
        const float most = __uint_as_float(0x7f7f0000u);
        w[0][at] = pack_pair<O>(fminf(fmaxf(a, -most), most), fminf(fmaxf(b, -most), most));  // (a NaN is in the other planes)
    } else {
        w[0][at] = pack_pair<O>(a, b);
    }
    if constexpr (N == 3) {
        float2 h = unpack_pair<O>(w[0][at]);
        a -= h.x;
        b -= h.y;
        w[1][at] = pack_pair<O>(a, b);
        h = unpack_pair<O>(w[1][at]);
        w[2][at] = pack_pair<O>(a - h.x, b - h.y);
    }
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

// keys of the tile from j0 on that are not padding (beyond the last key: set), for one warp
__device__ __forceinline__ unsigned long long key_mask(const AttnProblem &p, int b, int j0) {
    if (!p.doc_k) return ~0ull;
    const int lane = threadIdx.x & 31;
    const int *ids = p.doc_k + b * p.doc_k_sb + j0;
    const bool lo = j0 + lane >= p.Tk || ids[lane] >= 0, hi = j0 + 32 + lane >= p.Tk || ids[lane + 32] >= 0;
    return __ballot_sync(0xffffffffu, lo) | (unsigned long long)__ballot_sync(0xffffffffu, hi) << 32;
}
// zeros into the rows of a tile (64 rows of 64 * BLOCKS values) that `mask` leaves out; one warp
template <int BLOCKS>
__device__ __forceinline__ void clear_rows(uint8_t *tile, unsigned long long mask) {
    for (unsigned long long left = ~mask; left; left &= left - 1) {
        const int r = __ffsll(left) - 1;
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) reinterpret_cast<float *>(tile + k * 64 * 128 + r * 128)[threadIdx.x & 31] = 0.f;
    }
}
// tile of 64 keys from j0 on, by one thread; `map` by key_map
template <int BLOCKS>
__device__ __forceinline__ void load_keys(uint32_t dst, const CUtensorMap *map, int b, int g, int j0, uint32_t bar) {
    tma_expect_bytes(bar, BLOCKS * 64 * 128);
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) tma_load_5d(dst + k * 64 * 128, map, 64 * k, 0, j0, g, b, bar);
}
// the 128 packed rows of `width` values from m0 on of a query-side operand, by 128 threads; zeros beyond the end and for padding
template <int BLOCKS>
__device__ __forceinline__ void copy_row_tile(uint32_t dst, const AttnProblem &p, const AttnTensor &t, int width, int b, int g, int m0,
                                              int thread) {
    const char *base = static_cast<const char *>(t.p) + 2 * (b * t.sb + (long)g * p.R * t.sh);
    const int c = thread & 7;
#pragma unroll 4
    for (int n = 0; n < kRowTile / 16; ++n) {
        const int r = (thread >> 3) + 16 * n, m = m0 + r, i = p.R == 1 ? m : m / p.R;
        const bool in = m < p.M && (!p.doc_q || p.doc_q[b * p.doc_q_sb + i] >= 0);
        const char *src = base + 2 * (i * t.st + (m - i * p.R) * t.sh) + 16 * c;
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
            const bool real = in && k * 64 + c * 8 < width;
            copy16(dst + k * kRowTile * 128 + r * 128 + ((c ^ (r & 7)) << 4), real ? src + 128 * k : t.p, real);
        }
    }
}

// Tiles that a block has to visit, in ascending order: [at, end), or, with ranges of documents, those of them whose documents overlap
// the block's own.  For one warp, every lane alike.
struct TileWalk {
    const DocRange *ranges = nullptr;  // of this row of the batch, or null
    DocRange own{};                    // documents of the block's rows or keys
    int at = 0, end = 0;
    int whole_first = 0, whole_last = 0;  // tiles of which the masks by place leave everything
    int base = 0;
    uint32_t visit = 0, whole = 0;  // with ranges: tiles of [base - 32, base) that are left, and those of them without a mask

    // the next tile times two, plus one where no element of it is masked; -1: none
    __device__ __forceinline__ int next(bool docs) {
        if (!ranges) {
            if (at >= end) return -1;
            const int t = at++;
            return 2 * t + (!docs && t >= whole_first && t <= whole_last);
        }
        while (!visit) {
            if (base < at) base = at;  // (the first time)
            if (base >= end) return -1;
            const int t = base + (threadIdx.x & 31);
            bool see = false, all = false;
            if (t < end) {
                const DocRange r = ranges[t];
                see = r.least <= own.most && r.most >= own.least;
                all = see && own.least == own.most && r.least == r.most && !r.padding && !own.padding && t >= whole_first &&
                      t <= whole_last;
            }
            visit = __ballot_sync(0xffffffffu, see);
            whole = __ballot_sync(0xffffffffu, all);
            base += 32;
        }
        const int bit = __ffs(visit) - 1;
        visit &= visit - 1;
        return 2 * (base - 32 + bit) + (whole >> bit & 1);
    }
};
// documents of [first, end) of an axis cut into tiles of `size`
__device__ __forceinline__ DocRange own_range(const DocRange *ranges, int first, int end, int size) {
    DocRange r{kNoLeast, -1, 0, 0};
    for (int t = first / size; t <= (end - 1) / size; ++t) {
        r.least = min(r.least, ranges[t].least);
        r.most = max(r.most, ranges[t].most);
        r.padding |= ranges[t].padding;
    }
    return r;
}
__host__ __device__ constexpr int packed_tile(int R) { return 64 / R * R; }  // rows of a bulk copy of packed rows: whole tokens

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
    float over, small; // scale / cap, and the largest |s| for the series

    // a capped score, and the derivative of the cap.  16-bit operands: by 1 / (1 + 2^x), off by 2^-23 * cap, far below the operands' own
    // roundings; fp32 ones by tanhf.
    template <bool EXACT>
    __device__ __forceinline__ float capped(float s, float *slope) const {
        if (EXACT) {
            const float t = tanhf(s * in);
            *slope = 1.f - t * t;
            return k1 * t;
        }
        const float q = fast_rcp(1.f + fast_exp2(s * in));
        *slope = 4.f * q * (1.f - q);
        return k1 - k2 * q;
    }
    // Two scores far from the cap: tanh y = y (1 - y^2/3 + 2 y^4/15 - ...), its series up to y^11, off by 0.0036 y^13: below 2^-20 of it up
    // to 1/2 and below 2^-26 up to 0.35.  Scores are mostly there, and the two further exponentials and reciprocals per
    // score that `capped` takes would bound the kernels (4 x 4096 x 6 x 64 bf16 forward: 412 us with them, 192 us without a cap).
    __device__ __forceinline__ f32x2 capped_small(f32x2 s, f32x2 *slope) const {
        const f32x2 y = mul2(s, pack2(over, over)), z = mul2(y, y);
        f32x2 p = pack2(-1382.f / 155925.f, -1382.f / 155925.f);
        p = fma2(p, z, pack2(62.f / 2835.f, 62.f / 2835.f));
        p = fma2(p, z, pack2(-17.f / 315.f, -17.f / 315.f));
        p = fma2(p, z, pack2(2.f / 15.f, 2.f / 15.f));
        p = fma2(p, z, pack2(-1.f / 3.f, -1.f / 3.f));
        p = fma2(p, z, pack2(1.f, 1.f));
        const f32x2 t = mul2(p, y);
        *slope = fma2(mul2(t, pack2(-1.f, -1.f)), t, pack2(1.f, 1.f));
        return mul2(t, pack2(k1, k1));
    }
    // whether every score of a warp's is that far from the cap
    template <int N>
    __device__ __forceinline__ bool all_small(const float (&s)[N]) const {
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < N; j += 2) big = fmaxf(big, fmaxf(fabsf(s[j]), fabsf(s[j + 1])));
        return __all_sync(0xffffffffu, big <= small);  // (NaN: not among the largest; the series keeps it)
    }
};
template <bool EXACT>
__device__ __forceinline__ Bend make_bend(const AttnProblem &p) {
    Bend b;
    b.scale2 = p.scale * kLog2e;
    b.k1 = p.cap * kLog2e;
    b.k2 = 2.f * b.k1;
    b.in = p.cap > 0.f ? (EXACT ? p.scale : 2.f * b.scale2) / p.cap : 0.f;
    b.over = p.cap > 0.f ? p.scale / p.cap : 0.f;
    b.small = (EXACT ? 0.35f : 0.5f) / fmaxf(fabsf(b.over), 1e-30f);
    return b;
}

int *device_error_word();

// lutgemm_attention_split.cu: fp32 operands [B, T, heads, D <= 64] as planes [B, T, heads, 3, 64] of bf16, rows of padding as zeros
constexpr int kPlaneWidth = 3 * 64;
struct SplitOperand {
    AttnTensor from;
    __nv_bfloat16 *to;
    const int *doc;  // or null
    long doc_sb;
    int T, heads;
};
inline AttnTensor plane_tensor(const void *p, int T, int heads) {
    return {p, (long)T * heads * kPlaneWidth, (long)heads * kPlaneWidth, kPlaneWidth};
}
inline size_t plane_bytes(int B, int T, int heads) { return 2 * (size_t)B * T * heads * kPlaneWidth; }
// the last operand of four is grad_o, whose products with `out` go to delta
int attention_split(const AttnProblem &p, const SplitOperand *operands, int count, const float *out, float *delta, cudaStream_t stream);

// Tensor map of an operand whose heads come in groups of R: packed rows of a key head in boxes of 64 / R * R (a box of keys: R = 1)
inline bool attention_map(CUtensorMap *map, bool bf16, const AttnTensor &t, int B, int T, int G, int R, int D) {
    const auto bytes = [](long stride, long count) { return (unsigned long long)(count > 1 ? 2 * stride : 16); };
    const unsigned long long dims[5] = {(unsigned long long)D, (unsigned long long)R, (unsigned long long)T, (unsigned long long)G,
                                        (unsigned long long)B};
    const unsigned long long strides[4] = {bytes(t.sh, R), bytes(t.st, T), bytes(R * t.sh, G), bytes(t.sb, B)};
    const unsigned box[5] = {64, (unsigned)R, (unsigned)(64 / R), 1, 1};
    return make_tensor_map_16bit_5d(map, bf16, t.p, dims, strides, box);
}

// lutgemm_attention_tc.cu: ranges of the documents of tiles of 64 keys and of packed_tile(R) rows ([B][tiles] each); no bytes where
// nothing is gained by them
size_t doc_range_bytes(const AttnProblem &p);
int doc_ranges(const AttnProblem &p, void *scratch, const DocRange **keys, const DocRange **rows, cudaStream_t stream);

}  // namespace lutgemm
