// Attention forward on the tensor cores, 16-bit operands.
#include "lutgemm_attention_tc.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

constexpr int kThreads = 128;
constexpr int kAhead = 128;  // tiles whose masks are looked at together

// Tiles of 64 keys that a tile of rows has to visit, in ascending order: all up to the last visible key, or, with ranges of
// documents, those whose documents overlap the rows'.  Every thread of the block calls next() at the same places.
struct TileWalk {
    const DocRange *ranges;  // of this row of the batch, or null
    int qleast, qmost, qpadding, least_limit, end;  // end: one past the last tile
    int at, base;
    uint32_t *masks;  // shared memory: 4 words of tiles to visit, 4 of tiles without a mask

    __device__ __forceinline__ bool whole_by_limit(int t) const { return t * kKeyTile + kKeyTile - 1 <= least_limit; }
    // the next tile times two, plus one where no element of it is masked; -1: none
    __device__ __forceinline__ int next(bool docs) {
        if (!ranges) {
            const int t = at++;
            return t < end ? 2 * t + (!docs && whole_by_limit(t)) : -1;
        }
        for (;;) {
            const int in = at - base;
            for (int w = in >> 5; w < kAhead / 32 && base >= 0; ++w) {
                uint32_t m = masks[w];
                if (w == in >> 5) m &= 0xffffffffu << (in & 31);
                if (m) {
                    const int bit = __ffs(m) - 1, t = base + 32 * w + bit;
                    at = t + 1;
                    return 2 * t + (masks[4 + w] >> bit & 1);
                }
            }
            base = base < 0 ? at / kAhead * kAhead : base + kAhead;
            if (base >= end) {
                base -= kAhead;  // (stays at the end)
                at = base + kAhead;
                return -1;
            }
            at = max(at, base);
            __syncthreads();
            const int t = base + threadIdx.x;
            bool visit = false, whole = false;
            if (t < end) {
                const DocRange r = ranges[t];
                visit = r.least <= qmost && r.most >= qleast;
                whole = visit && qleast == qmost && r.least == r.most && !r.padding && !qpadding && whole_by_limit(t);
            }
            const uint32_t v = __ballot_sync(0xffffffffu, visit), f = __ballot_sync(0xffffffffu, whole);
            if ((threadIdx.x & 31) == 0) {
                masks[threadIdx.x / 32] = v;
                masks[4 + threadIdx.x / 32] = f;
            }
            __syncthreads();
        }
    }
};

// A block has 128 packed rows, one to a thread and lane of tensor memory, and goes over the keys in tiles of 64:
//     S = Q K^T (tcgen05, into tensor memory) -> the thread's 64 scores to registers, mask, maximum, P = exp2 -> P back to tensor
//     memory in 16 bits, over S -> O += P V (tcgen05, P from tensor memory).
// Only one synchronisation of the block stands in a round: behind it one thread issues P V of this tile and S of the tile STAGES
// ahead, which the tensor cores run in order.  Heads of up to 64 values keep one S and leave room for four blocks on an SM, whose
// rounds overlap; larger ones have room for two blocks and keep two S, so that a round never waits for the product it begins
// with.  The running maximum is only raised, and O rescaled, where a row's maximum grows by more than 8 in log 2: probabilities
// then reach 2^8, sums are fp32.  fp16 probabilities are kept 2^7 larger, out of its subnormal range.
// P is rounded to the operands' type, as the tensor cores take it; its row sums are of the unrounded values.
template <typename T, int DP>
struct Layout {
    static constexpr int kBlocks = DP / 64, kStages = DP == 64 ? 1 : 2, kKStages = kStages + 1, kPerSm = DP == 64 ? 4 : 2;
    static constexpr uint32_t kQ = 0, kK = kRowTile * DP * 2, kTile = kKeyTile * DP * 2, kV = kK + kKStages * kTile,
                              kBars = kV + 2 * kTile, kBytes = kBars + 128;
    static constexpr uint32_t kColumns = DP == 64 ? 128 : 256, kO = kStages * 64;  // tensor memory: S, then O
};

template <typename T, int DP, bool BENT>
__global__ void __launch_bounds__(kThreads, Layout<T, DP>::kPerSm)
    attention_tc_kernel(const AttnProblem p, const DocRange *key_ranges, const DocRange *row_ranges, T *out, T *rest, float *lse,
                        float *part, float *part_lse, int splits, int *error_word) {
    using L = Layout<T, DP>;
    constexpr float kShift = IsBf16<T>::value ? 0.f : 7.f;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem), bars = base + L::kBars;
    volatile int *abort_word = reinterpret_cast<int *>(smem + L::kBars + 32);
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::kBars + 36);
    const int tid = threadIdx.x, warp = tid >> 5;
    // blocks in order of falling work: the last rows see the most keys
    int bid = blockIdx.x;
    const int split = bid % splits;
    bid /= splits;
    const int g = bid % p.G;
    bid /= p.G;
    const int b = bid % p.B, tiles = (p.M + kRowTile - 1) / kRowTile, m0 = (tiles - 1 - bid / p.B) * kRowTile;
    if (tid == 0) {
        *abort_word = 0;
        for (int i = 0; i < 3; ++i) mbar_init(bars + 8 * i, 1);  // S of either buffer, O
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(smem_u32(slot), L::kColumns);
    copy_rows<kRowTile, L::kBlocks>(base + L::kQ, p, p.q, b, g, m0, tid);

    const int pre = p.prefix ? p.prefix[b] : 0, last = min(m0 + kRowTile, p.M) - 1;
    TileWalk walk;
    walk.ranges = key_ranges ? key_ranges + (long)b * ((p.Tk + kKeyTile - 1) / kKeyTile) : nullptr;
    walk.masks = reinterpret_cast<uint32_t *>(smem + L::kBars + 64);
    walk.least_limit = key_limit(p, m0 / p.R + p.shift, pre);
    const int all = max(0, key_limit(p, last / p.R + p.shift, pre) + 1 + kKeyTile - 1) / kKeyTile;  // tiles up to the last visible key
    walk.at = 0;
    walk.end = all;
    walk.base = -1;
    if (splits > 1) {
        const int per = (all + splits - 1) / splits;
        walk.at = min(split * per, all);
        walk.end = min(walk.at + per, all);
    }
    if (walk.ranges) {
        const int tiles64 = (p.M + kKeyTile - 1) / kKeyTile;
        const DocRange *r = row_ranges + (long)b * tiles64 + m0 / kKeyTile;
        const DocRange a = r[0], c = m0 / kKeyTile + 1 < tiles64 ? r[1] : DocRange{kNoLeast, -1, 0, 0};
        walk.qleast = min(a.least, c.least);
        walk.qmost = max(a.most, c.most);
        walk.qpadding = a.padding | c.padding;
    }
    const bool docs = p.doc_k != nullptr;
    const int m = m0 + tid;
    const TileRow row = tile_row(p, b, g, m, pre);
    const bool idle = __all_sync(0xffffffffu, row.limit < 0);  // the warp's rows see nothing
    const Bend bend = make_bend(p);

    int queue[L::kKStages];  // this tile and those whose keys are under way
#pragma unroll
    for (int i = 0; i < L::kKStages; ++i) queue[i] = (i == 0 || queue[i > 0 ? i - 1 : 0] >= 0) ? walk.next(docs) : -1;
#pragma unroll
    for (int i = 0; i < L::kStages; ++i)
        if (queue[i] >= 0) copy_keys<L::kBlocks>(base + L::kK + i * L::kTile, p, p.k, b, g, (queue[i] >> 1) * kKeyTile, tid);
    copies_end_group();
    if (queue[0] >= 0) copy_keys<L::kBlocks>(base + L::kV, p, p.v, b, g, (queue[0] >> 1) * kKeyTile, tid);
    if (queue[L::kStages] >= 0)
        copy_keys<L::kBlocks>(base + L::kK + L::kStages * L::kTile, p, p.k, b, g, (queue[L::kStages] >> 1) * kKeyTile, tid);
    copies_end_group();
    copies_wait<1>();
    writes_to_tensor_cores();
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    const uint32_t tmem = *slot, mine = tmem + ((uint32_t)(warp * 32) << 16);
    constexpr uint32_t desc_s = mma_descriptor(IsBf16<T>::value, kKeyTile, false), desc_o = mma_descriptor(IsBf16<T>::value, DP, true);
    auto issue_scores = [&](int n) {  // S of the n-th visited tile
        const uint32_t k = base + L::kK + (n % L::kKStages) * L::kTile, d = tmem + (n % L::kStages) * 64;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
            mma_ss(d, smem_descriptor(base + L::kQ + (i >> 2) * kRowTile * 128 + (i & 3) * 32, 0),
                   smem_descriptor(k + (i >> 2) * kKeyTile * 128 + (i & 3) * 32, 0), desc_s, i > 0);
        mma_commit(bars + 8 * (n % L::kStages));
    };
    if (tid == 0)
#pragma unroll
        for (int i = 0; i < L::kStages; ++i)
            if (queue[i] >= 0) issue_scores(i);

    float most = -INFINITY, sum = 0.f;  // the maximum that P is relative to, in log 2
    int n = 0;
    for (; queue[0] >= 0; ++n) {
        const int tile = queue[0] >> 1, j0 = tile * kKeyTile;
        const bool masked = !(queue[0] & 1);
        const int ahead = queue[L::kKStages - 1] >= 0 ? walk.next(docs) : -1;
        mbar_wait(bars + 8 * (n % L::kStages), (n / L::kStages) & 1, 201, abort_word, error_word);
        tmem_after_sync();
        const uint32_t s_at = mine + (n % L::kStages) * 64;
        // the scores' product is done, so the keys' buffer is free
        if (ahead >= 0) copy_keys<L::kBlocks>(base + L::kK + (n % L::kKStages) * L::kTile, p, p.k, b, g, (ahead >> 1) * kKeyTile, tid);
        float s[2][32];
        float factor = 1.f;
        bool raise = false;
        if (!idle) {
            tmem_load32(s_at, s[0]);
            tmem_load32(s_at + 32, s[1]);
            tmem_loads_done();
            if (BENT) {
                if (p.cap > 0.f) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 32; ++j) s[h][j] = bend.k1 - bend.k2 * fast_rcp(1.f + fast_exp2(s[h][j] * bend.in));
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 32; ++j) s[h][j] *= bend.scale2;
                }
                if (p.slopes) {
                    const float away = (float)(row.place - j0);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 32; ++j) s[h][j] -= row.slope * fabsf(away - (float)(32 * h + j));
                }
            }
            if (masked) {
                const int reach = row.limit - j0;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[h][j] = 32 * h + j <= reach ? s[h][j] : -INFINITY;
                if (docs) {
                    const int *ids = p.doc_k + b * p.doc_k_sb + j0;
                    const int have = p.Tk - j0;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (32 * h + j < have && ids[32 * h + j] != row.doc) s[h][j] = -INFINITY;
                }
            }
            float top[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], s[h][j]);
            float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (!BENT) now *= bend.scale2;
            raise = now > most + 8.f;  // (from -inf on the first visible key)
            if (raise) {
                factor = fast_exp2(most - now);  // 0 from -inf
                most = now;
                sum *= factor;
            }
        }
        if (n > 0) {
            mbar_wait(bars + 16, (n - 1) & 1, 202, abort_word, error_word);
            tmem_after_sync();
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    float o[32];
                    tmem_load32(mine + L::kO + 32 * c, o);
                    tmem_loads_done();
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] *= factor;
                    tmem_store32(mine + L::kO + 32 * c, o);
                }
            }
        }
        // V of the tile before is done with
        if (queue[1] >= 0) copy_keys<L::kBlocks>(base + L::kV + ((n + 1) & 1) * L::kTile, p, p.v, b, g, (queue[1] >> 1) * kKeyTile, tid);
        copies_end_group();
        if (!idle) {
            uint32_t w[2][16];
            const float less = most == -INFINITY ? 0.f : most - kShift;
            float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float a = fast_exp2(BENT ? s[h][j] - less : fmaf(s[h][j], bend.scale2, -less));
                    const float c = fast_exp2(BENT ? s[h][j + 1] - less : fmaf(s[h][j + 1], bend.scale2, -less));
                    add[j & 2] += a;
                    add[(j & 2) + 1] += c;
                    w[h][j / 2] = pack2<T>(a, c);
                }
            sum += (add[0] + add[1]) + (add[2] + add[3]);
            tmem_store16(s_at, w[0]);
            tmem_store16(s_at + 16, w[1]);
        }  // (rows that see nothing: whatever their P holds stays in their own rows of O, which are not used)
        tmem_stores_done();
        copies_wait<1>();
        writes_to_tensor_cores();
        tmem_before_sync();
        __syncthreads();
        if (tid == 0) {
            tmem_after_sync();
            const uint32_t v = base + L::kV + (n & 1) * L::kTile, a = tmem + (n % L::kStages) * 64;
#pragma unroll
            for (int i = 0; i < kKeyTile / 16; ++i)
                mma_ts(tmem + L::kO, a + 8 * i, smem_descriptor(v + i * 16 * 128, kKeyTile * 128), desc_o, n > 0 || i > 0);
            mma_commit(bars + 16);
            if (queue[L::kStages] >= 0) issue_scores(n + L::kStages);
        }
#pragma unroll
        for (int i = 0; i + 1 < L::kKStages; ++i) queue[i] = queue[i + 1];
        queue[L::kKStages - 1] = ahead;
    }
    copies_wait<0>();
    if (n > 0) {
        mbar_wait(bars + 16, (n - 1) & 1, 203, abort_word, error_word);
        tmem_after_sync();
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
    const float stat = sum == 0.f ? INFINITY : most - kShift + log2f(sum);
    const int i = m < p.M ? m / p.R : 0, h = g * p.R + m - i * p.R;
    const long at = ((long)b * p.G + g) * p.M + m;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
        float o[32];
        if (n > 0) {
            tmem_load32(mine + L::kO + 32 * c, o);
            tmem_loads_done();
        }
        if (m < p.M) {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = sum == 0.f ? 0.f : o[j] * inv;
            if (splits > 1) {
                float4 *dst = reinterpret_cast<float4 *>(part + ((long)split * p.B * p.G * p.M + at) * DP + 32 * c);
#pragma unroll
                for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            } else {
                const long to = (((long)b * p.Tq + i) * p.H + h) * p.D + 32 * c;
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                    if (32 * c + j >= p.D) break;
                    uint4 v;
                    uint32_t *r = &v.x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = pack2<T>(o[j + 2 * e], o[j + 2 * e + 1]);
                    *reinterpret_cast<uint4 *>(out + to + j) = v;
                    if (rest) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 hi = unpack2<T>(r[e]);
                            r[e] = pack2<T>(o[j + 2 * e] - hi.x, o[j + 2 * e + 1] - hi.y);
                        }
                        *reinterpret_cast<uint4 *>(rest + to + j) = v;
                    }
                }
            }
        }
        __syncwarp();
    }
    if (m < p.M) {
        if (splits > 1) part_lse[(long)split * p.B * p.G * p.M + at] = sum == 0.f ? -INFINITY : stat;
        else lse[at] = stat;
    }
    tmem_before_sync();
    __syncthreads();
    if (warp == 0) {
        tmem_after_sync();
        tmem_free(tmem, L::kColumns);
    }
}

// Joins the parts of a row: a warp to a row, weights 2^(statistic - largest).
template <typename T, int DP>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttnProblem p, const float *part, const float *part_lse, int splits, T *out,
                                                             T *rest, float *lse) {
    const long rows = (long)p.B * p.G * p.M, at = blockIdx.x * 4L + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (at >= rows) return;
    float most = -INFINITY, sum = 0.f;
    for (int s = lane; s < splits; s += 32) most = fmaxf(most, part_lse[s * rows + at]);
#pragma unroll
    for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    const float from = most == -INFINITY ? 0.f : most;
    constexpr int kPer = DP / 32;
    float o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float w = exp2f(part_lse[s * rows + at] - from);  // (a NaN of a part is its row's)
        sum += w;
        if (w != 0.f) {
            const float *src = part + (s * rows + at) * DP + lane * kPer;
#pragma unroll
            for (int e = 0; e < kPer; ++e) o[e] += w * src[e];
        }
    }
    const long bg = at / p.M;
    const int m = (int)(at - bg * p.M), b = (int)(bg / p.G), g = (int)(bg - (long)b * p.G), i = m / p.R, h = g * p.R + m - i * p.R;
    const long dst = (((long)b * p.Tq + i) * p.H + h) * p.D + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if (lane * kPer + e >= p.D) break;
        const float v = sum == 0.f ? 0.f : o[e] / sum;
        out[dst + e] = from_f32<T>(v);
        if (rest) rest[dst + e] = from_f32<T>(v - to_f32<T>(from_f32<T>(v)));
    }
    if (lane == 0) lse[at] = sum == 0.f ? INFINITY : most + log2f(sum);
}

// a warp to a tile
__global__ void __launch_bounds__(128) attention_doc_ranges_kernel(const AttnProblem p, DocRange *keys, DocRange *rows, int key_tiles,
                                                                   int row_tiles) {
    const int b = blockIdx.y, w = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (w >= key_tiles + row_tiles) return;
    const bool key = w < key_tiles;
    const int t = key ? w : w - key_tiles, end = key ? p.Tk : p.M;
    const int *ids = key ? p.doc_k + b * p.doc_k_sb : p.doc_q + b * p.doc_q_sb;
    int least = kNoLeast, most = -1, padding = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int x = t * kKeyTile + lane + 32 * k;
        if (x < end) {
            const int id = ids[key || p.R == 1 ? x : x / p.R];
            if (id < 0) padding = 1;
            else { least = min(least, id); most = max(most, id); }
        }
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    padding = __any_sync(0xffffffffu, padding);
    if (lane == 0) (key ? keys + (long)b * key_tiles : rows + (long)b * row_tiles)[t] = DocRange{least, most, padding, 0};
}

template <typename T, int DP, bool BENT>
int launch(const AttnProblem &p, const DocRange *kr, const DocRange *rr, void *out, void *rest, float *lse, float *part, float *part_lse,
           int splits, int *error_word, cudaStream_t stream) {
    using L = Layout<T, DP>;
    if (!cuda_ok(cudaFuncSetAttribute(attention_tc_kernel<T, DP, BENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes)))
        return LUTGEMM_E_CUDA;
    const long blocks = (long)((p.M + kRowTile - 1) / kRowTile) * p.B * p.G * splits;
    if (blocks > 0x7fffffffL) return LUTGEMM_E_TOOLARGE;
    attention_tc_kernel<T, DP, BENT><<<(unsigned)blocks, kThreads, L::kBytes, stream>>>(
        p, kr, rr, static_cast<T *>(out), static_cast<T *>(rest), lse, part, part_lse, splits, error_word);
    int rc = launch_status();
    if (rc == LUTGEMM_OK && splits > 1) {
        const long rows = (long)p.B * p.G * p.M;
        attention_join_kernel<T, DP><<<(unsigned)((rows + 3) / 4), 128, 0, stream>>>(p, part, part_lse, splits, static_cast<T *>(out),
                                                                                  static_cast<T *>(rest), lse);
        rc = launch_status();
    }
    return rc;
}

// Parts of the keys: as many as fill the blocks that the GPU holds at a time, of at least four tiles each.
int key_splits(const AttnProblem &p, int sms) {
    const long blocks = (long)((p.M + kRowTile - 1) / kRowTile) * p.B * p.G, slots = (long)sms * (p.D <= 64 ? 4 : 2);
    const long most = (p.Tk + 4 * kKeyTile - 1) / (4 * kKeyTile), want = slots / blocks;
    return (int)(want < 2 || most < 2 ? 1 : want < most ? want : most);
}

}  // namespace

size_t doc_range_bytes(const AttnProblem &p) {
    if (!p.doc_k || p.Tk <= 4 * kKeyTile) return 0;  // a launch costs more than the few tiles that it might spare
    return sizeof(DocRange) * p.B * ((size_t)(p.Tk + kKeyTile - 1) / kKeyTile + (size_t)(p.M + kKeyTile - 1) / kKeyTile);
}
int doc_ranges(const AttnProblem &p, DocRange *keys, DocRange *rows, cudaStream_t stream) {
    const int kt = (p.Tk + kKeyTile - 1) / kKeyTile, rt = (p.M + kKeyTile - 1) / kKeyTile;
    attention_doc_ranges_kernel<<<dim3((kt + rt + 3) / 4, p.B), 128, 0, stream>>>(p, keys, rows, kt, rt);
    return launch_status();
}

size_t attention_tc_scratch_bytes(const AttnProblem &p, int sms) {
    const int splits = key_splits(p, sms), dp = p.D <= 64 ? 64 : 128;
    return doc_range_bytes(p) + (splits > 1 ? sizeof(float) * (size_t)splits * p.B * p.G * p.M * (dp + 1) : 0);
}

int attention_tc_forward(const AttnProblem &p, int dtype, void *out, void *rest, float *lse, void *scratch, int sms, cudaStream_t stream) {
    int *error_word = device_error_word();
    if (!error_word) return LUTGEMM_E_CUDA;
    const int splits = key_splits(p, sms), dp = p.D <= 64 ? 64 : 128;
    DocRange *kr = nullptr, *rr = nullptr;
    const size_t ranges = doc_range_bytes(p);
    if (ranges) {
        kr = static_cast<DocRange *>(scratch);
        rr = kr + (size_t)p.B * ((p.Tk + kKeyTile - 1) / kKeyTile);
        const int rc = doc_ranges(p, kr, rr, stream);
        if (rc != LUTGEMM_OK) return rc;
    }
    float *part = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + ranges), *part_lse = part + (size_t)splits * p.B * p.G * p.M * dp;
    const bool bent = p.cap > 0.f || p.slopes || !(p.scale > 0.f);
#define RUN(T, DP) (bent ? launch<T, DP, true>(p, kr, rr, out, rest, lse, part, part_lse, splits, error_word, stream) \
                         : launch<T, DP, false>(p, kr, rr, out, rest, lse, part, part_lse, splits, error_word, stream))
    if (dtype == LUTGEMM_BF16) return dp == 64 ? RUN(__nv_bfloat16, 64) : RUN(__nv_bfloat16, 128);
    return dp == 64 ? RUN(__half, 64) : RUN(__half, 128);
#undef RUN
}

}  // namespace lutgemm
