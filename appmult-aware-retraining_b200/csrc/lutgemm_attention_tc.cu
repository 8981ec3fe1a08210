// Attention forward on the tensor cores: 16-bit operands, and fp32 ones as three bf16 planes.
#include "lutgemm_attention_tc.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

constexpr int kThreads = 160;  // four warps with a row to a thread, one that brings tiles and issues products

// A block has 128 packed rows, one to a thread of its first four warps and a lane of tensor memory, and goes over the keys in tiles
// of 64:
//     S = Q K^T (tcgen05, into tensor memory) -> the thread's 64 scores to registers, mask, maximum, P = exp2 -> P back to tensor
//     memory in 16 bits, over S -> O += P V (tcgen05, P from tensor memory).
// The fifth warp brings the tiles and, when all rows' P stands, issues P V of this tile and S of the tile STAGES ahead; the tensor
// cores run them in order.  Heads of up to 64 values keep one S and leave room for three blocks on an SM, whose rounds overlap;
// larger ones have room for two blocks and keep two S, so that a round never waits for the product before it.
// The running maximum is only raised, and O rescaled, where a row's maximum grows by more than 8 in log 2: probabilities
// then reach 2^8, sums are fp32.  fp16 probabilities are kept 2^7 larger, out of its subnormal range.
// P is rounded to the operands' type, as the tensor cores take it; its row sums are of the unrounded values.
// fp32: P is split into planes as the operands were, and each tile's products with V start from zero and are added up in registers: the
// tensor cores cut off what an addition loses, which over a long row would add up.
//
// The turns of products and probabilities bound it; no unit is full.  Heads of 64 values: exponential unit 60 %, tensor pipe 30 %, 4 x 4096 x 6
// x 64 bf16 185 us (556 TFLOP/s).  Heads of 128: 50 % each, 2 x 4096, 16 / 4 heads, bf16 288 us (955 TFLOP/s);
// 1 x 8192, 16 heads, fp16, causal 264 us (1040; 8 TB/s of tiles from L2, a third of its rate), 306 in a loop under the power cap.
// fp32, 64 x 197 x 6 x 64: 73 us.  One query, 16 x 16385 keys, 16 / 4 heads of 64 bf16: 60 us with its join (4.5 TB/s).
template <typename T, int DP>
struct Layout {
    using Op = Operand<T, DP>;
    static constexpr int kBlocks = Op::kBlocks, kStages = DP == 64 && !Op::kPlanes ? 1 : 2;  // of S
    static constexpr int kKStages = 3, kVStages = kStages == 1 ? 3 : 2;                        // of tiles of K and V
    static constexpr int kPerSm = Op::kPlanes ? 1 : DP == 64 ? 3 : 2;
    static constexpr uint32_t kTile = kKeyTile * kBlocks * 128, kQ = 0, kK = 2 * kTile, kV = kK + kKStages * kTile, kBars = kV + kVStages * kTile,
                              kBytes = kBars + 128;
    static constexpr uint32_t kS = Op::kPlanes ? 96 : 64, kO = kStages * kS;  // tensor memory: S or P of each stage, then O
    static constexpr uint32_t kColumns = kO + DP <= 128 ? 128 : 256;
};
constexpr int kEnd = -1;  // in place of a tile: there are no more

template <typename T, int DP, bool BENT>
__global__ void __launch_bounds__(kThreads, Layout<T, DP>::kPerSm)
    attention_tc_kernel(const AttnProblem p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const DocRange *key_ranges, const DocRange *row_ranges, T *out, T *rest, float *lse,
                        float *part, float *part_lse, int splits, int *error_word) {
    using L = Layout<T, DP>;
    using Op = typename L::Op;
    constexpr float kShift = Op::kBf16 ? 0.f : 7.f;
    const int width = Op::kPlanes ? kPlaneWidth : p.D;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem), bar_s = base + L::kBars, bar_o = bar_s + 16, bar_p = bar_s + 24, bar_k = bar_s + 32, bar_v = bar_s + 56;  // (three each)
    volatile int *abort_word = reinterpret_cast<int *>(smem + L::kBars + 80);
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::kBars + 84);
    volatile int *tiles = reinterpret_cast<int *>(smem + L::kBars + 88);  // of the last four rounds begun
    const int tid = threadIdx.x, warp = warp_index();
    // blocks in order of falling work: the last rows see the most keys
    int bid = blockIdx.x;
    const int split = bid % splits;
    bid /= splits;
    const int g = bid % p.G;
    bid /= p.G;
    const int b = bid % p.B, row_tiles = (p.M + kRowTile - 1) / kRowTile, m0 = (row_tiles - 1 - bid / p.B) * kRowTile;
    const int pre = p.prefix ? p.prefix[b] : 0;
    const bool docs = p.doc_k != nullptr;
    if (tid == 0) {
        *abort_word = 0;
        mbar_init(bar_s, 2);  // the products' arrival and the issuing lane's own, which orders `tiles`
        mbar_init(bar_s + 8, 2);
        mbar_init(bar_o, 1);
        mbar_init(bar_p, 128);
        for (int i = 0; i < L::kKStages; ++i) mbar_init(bar_k + 8 * i, 1);
        for (int i = 0; i < L::kVStages; ++i) mbar_init(bar_v + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == 4) {
        if (elect_one()) {
            tma_prefetch_map(&map_k);
            tma_prefetch_map(&map_v);
        }
        __syncwarp();
        TileWalk walk;
        const int last = min(m0 + kRowTile, p.M) - 1;
        const int all = max(0, key_limit(p, last / p.R + p.shift, pre) + kKeyTile) / kKeyTile;  // up to the last visible key
        walk.end = all;
        walk.whole_last = max(0, key_limit(p, m0 / p.R + p.shift, pre) + 1) / kKeyTile - 1;
        if (splits > 1) {
            const int per = (all + splits - 1) / splits;
            walk.at = min(split * per, all);
            walk.end = min(walk.at + per, all);
        }
        if (key_ranges) {
            const int size = packed_tile(p.R);
            walk.ranges = key_ranges + (long)b * ((p.Tk + kKeyTile - 1) / kKeyTile);
            walk.own = own_range(row_ranges + (long)b * ((p.M + size - 1) / size), m0, last + 1, size);
        }
        int queue[L::kKStages + 1] = {};  // this round's tile and those behind it
        auto bring = [&](int i) {
            const bool more = i == 0 || queue[i - 1] >= 0;
            queue[i] = more ? walk.next(docs) : kEnd;
        };
        auto bring_k = [&](int i, int stage) {
            if (queue[i] >= 0 && elect_one())
                load_keys<L::kBlocks>(base + L::kK + stage * L::kTile, &map_k, b, g, (queue[i] >> 1) * kKeyTile, bar_k + 8 * stage);
        };
        auto bring_v = [&](int i, int stage) {
            if (queue[i] >= 0 && elect_one())
                load_keys<L::kBlocks>(base + L::kV + stage * L::kTile, &map_v, b, g, (queue[i] >> 1) * kKeyTile, bar_v + 8 * stage);
        };
#pragma unroll
        for (int i = 0; i < L::kKStages; ++i) bring(i);
#pragma unroll
        for (int i = 0; i < L::kKStages; ++i) {
            bring_k(i, i);
            if (i < L::kVStages - 1) bring_v(i, i);
        }
        __syncwarp();
        tmem_alloc(smem_u32(slot), L::kColumns);
        tmem_before_sync();
        __syncthreads();  // Q has come
        tmem_after_sync();
        const uint32_t tmem = *slot;
        constexpr uint32_t desc_s = mma_descriptor(Op::kBf16, kKeyTile, false), desc_o = mma_descriptor(Op::kBf16, DP, true);
        auto issue_scores = [&](int n, int tile) {  // S of round n, or word that there is none; one lane
            const uint32_t bar = bar_s + 8 * (n % L::kStages);
            tiles[n & 3] = tile;
            if (tile >= 0) {
                const uint32_t d = tmem + (n % L::kStages) * L::kS;
                const uint64_t q = smem_descriptor(base + L::kQ, 0), k = smem_descriptor(base + L::kK + (n % L::kKStages) * L::kTile, 0);
#pragma unroll
                for (int i = 0; i < 4 * Op::kProducts; ++i)
                    mma_ss(d, descriptor_at(q, Op::a(i >> 2) * kRowTile * 128 + (i & 3) * 32),
                           descriptor_at(k, Op::b(i >> 2) * kKeyTile * 128 + (i & 3) * 32), desc_s, i > 0);
                mma_commit(bar);
            } else {
                mbar_arrive(bar);
            }
            mbar_arrive(bar);
        };
        // what padding holds: a probability of zero would not hide it in V, and in K it would have a say in how caps are computed
        auto clear_padding = [&](int tile, uint32_t at) {
            if (!docs || Op::kPlanes) return;
            const unsigned long long mask = key_mask(p, b, (tile >> 1) * kKeyTile);
            if (~mask) {
                clear_rows<L::kBlocks>(smem + at, mask);
                writes_to_tensor_cores();
            }
        };
#pragma unroll
        for (int i = 0; i < L::kStages; ++i) {
            if (queue[i] >= 0) {
                mbar_wait(bar_k + 8 * i, 0, 206, abort_word, error_word);
                clear_padding(queue[i], L::kK + i * L::kTile);
                __syncwarp();
            }
            if ((i == 0 || queue[i - 1] >= 0) && elect_one()) issue_scores(i, queue[i]);
        }
        __syncwarp();
        for (int n = 0; queue[0] >= 0; ++n) {
            bring(L::kKStages);
            mbar_wait(bar_v + 8 * (n % L::kVStages), n / L::kVStages & 1, 207, abort_word, error_word);
            clear_padding(queue[0], L::kV + n % L::kVStages * L::kTile);
            if (queue[L::kStages] >= 0 && queue[L::kStages - 1] >= 0) {
                const int stage = (n + L::kStages) % L::kKStages;
                mbar_wait(bar_k + 8 * stage, (n + L::kStages) / L::kKStages & 1, 208, abort_word, error_word);
                clear_padding(queue[L::kStages], L::kK + stage * L::kTile);
            }
            mbar_wait(bar_p, n & 1, 201, abort_word, error_word);
            tmem_after_sync();
            __syncwarp();
            // every row has waited for the products of round n - 1 and S of round n: those buffers are free.  (Copies first: the queue
            // of the tensor cores lets products go one by one)
            bring_v(L::kVStages - 1, (n + L::kVStages - 1) % L::kVStages);
            bring_k(L::kKStages, n % L::kKStages);
            __syncwarp();
            if (elect_one()) {
                const uint64_t v = smem_descriptor(base + L::kV + n % L::kVStages * L::kTile, Op::kPlanes ? 0 : kKeyTile * 128);
                const uint32_t a = tmem + (n % L::kStages) * L::kS;
                if constexpr (Op::kPlanes) {
#pragma unroll
                    for (int i = 0; i < 4 * Op::kProducts; ++i)
                        mma_ts(tmem + L::kO, a + 32 * Op::a(i >> 2) + 8 * (i & 3),
                               descriptor_at(v, Op::b(i >> 2) * kKeyTile * 128 + (i & 3) * 16 * 128), desc_o, i > 0);
                } else {
#pragma unroll
                    for (int i = 0; i < kKeyTile / 16; ++i)
                        mma_ts(tmem + L::kO, a + 8 * i, descriptor_at(v, i * 16 * 128), desc_o, n > 0 || i > 0);
                }
                mma_commit(bar_o);
                if (queue[L::kStages - 1] >= 0) issue_scores(n + L::kStages, queue[L::kStages]);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < L::kKStages; ++i) queue[i] = queue[i + 1];
        }
    } else {
        copy_row_tile<L::kBlocks>(base + L::kQ, p, p.q, width, b, g, m0, tid);
        copies_end_group();
        copies_wait<0>();
        writes_to_tensor_cores();
        __syncthreads();
        tmem_after_sync();
        const uint32_t mine = *slot + ((uint32_t)(warp * 32) << 16);
        const int m = m0 + tid;
        const TileRow row = tile_row(p, b, g, m, pre);
        const bool idle = __all_sync(0xffffffffu, row.limit < 0);  // the warp's rows see nothing
        const Bend bend = make_bend<Op::kPlanes>(p);
        float most = -INFINITY, sum = 0.f;  // the maximum that P is relative to, in log 2
        f32x2 total_o[Op::kPlanes ? 32 : 1] = {};
        auto add_tile = [&](float factor) {  // fp32: the products of the round before
            const f32x2 f2 = pack2(factor, factor);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float o[32];
                tmem_load32(mine + L::kO + 32 * c, o);
                tmem_loads_done();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    f32x2 &t = total_o[Op::kPlanes ? 16 * c + j : 0];
                    t = mul2(add2(t, pack2(o[2 * j], o[2 * j + 1])), f2);
                }
            }
        };
        int n = 0;
        for (;; ++n) {
            mbar_wait(bar_s + 8 * (n % L::kStages), (n / L::kStages) & 1, 202, abort_word, error_word);
            const int tile = tiles[n & 3];
            if (tile < 0 || *abort_word) break;
            tmem_after_sync();
            const uint32_t s_at = mine + (n % L::kStages) * L::kS;
            if (idle) {
                // whatever the P of these rows holds stays in their rows of O, which are not used
                if (n > 0) mbar_wait(bar_o, (n - 1) & 1, 203, abort_word, error_word);
                mbar_arrive(bar_p);
                continue;
            }
            float s[2][32];
            tmem_load32(s_at, s[0]);
            tmem_load32(s_at + 32, s[1]);
            tmem_loads_done();
            const int j0 = (tile >> 1) * kKeyTile;
            if (BENT) {
                if (p.cap > 0.f) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (bend.all_small(s[h])) {
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                f32x2 unused;
                                const float2 x = unpack2(bend.capped_small(pack2(s[h][j], s[h][j + 1]), &unused));
                                s[h][j] = x.x;
                                s[h][j + 1] = x.y;
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                float unused;
                                s[h][j] = bend.template capped<Op::kPlanes>(s[h][j], &unused);
                            }
                        }
                    }
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
            if (!(tile & 1)) {
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
                for (int j = 0; j < 32; j += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fmaxf(s[h][j + e], s[h][j + 4 + e]));
            float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (!BENT) now *= bend.scale2;
            const bool raise = now > most + 8.f;  // (from -inf on the first visible key)
            float factor = 1.f;
            if (raise) {
                factor = fast_exp2(most - now);  // 0 from -inf
                most = now;
                sum *= factor;
            }
            if (n > 0) {
                mbar_wait(bar_o, (n - 1) & 1, 204, abort_word, error_word);
                if constexpr (Op::kPlanes) {
                    tmem_after_sync();
                    add_tile(factor);
                } else if (__any_sync(0xffffffffu, raise)) {
                    tmem_after_sync();
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c) {
                        float o[16];
                        tmem_load16(mine + L::kO + 16 * c, o);
                        tmem_loads_done();
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] *= factor;
                        tmem_store16(mine + L::kO + 16 * c, o);
                    }
                }
            }
            const float less = most == -INFINITY ? 0.f : most - kShift;
            const f32x2 less2 = pack2(-less, -less), scale2 = pack2(bend.scale2, bend.scale2);
            f32x2 add[2] = {0ull, 0ull};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[Op::kPlanes ? 3 : 1][16];
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const f32x2 x = pack2(s[h][j], s[h][j + 1]);
                    const float2 y = unpack2(BENT ? add2(x, less2) : fma2(x, scale2, less2));
                    const float a = fast_exp2(y.x), c = fast_exp2(y.y);
                    add[j / 2 & 1] = add2(add[j / 2 & 1], pack2(a, c));
                    plane_words<T>(w, j / 2, a, c);
                }
#pragma unroll
                for (int e = 0; e < (Op::kPlanes ? 3 : 1); ++e) tmem_store16(s_at + 32 * e + 16 * h, w[e]);
            }
            const float2 total = unpack2(add2(add[0], add[1]));
            sum += total.x + total.y;
            tmem_stores_done();
            tmem_before_sync();
            mbar_arrive(bar_p);
        }
        if (n > 0) {
            mbar_wait(bar_o, (n - 1) & 1, 205, abort_word, error_word);
            tmem_after_sync();
            if constexpr (Op::kPlanes)
                if (!idle) add_tile(1.f);
        }
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
        const float stat = sum == 0.f ? INFINITY : most - kShift + log2f(sum);
        const long at = ((long)b * p.G + g) * p.M + m;
        // Whole rows are stored, through shared memory that Q and K have left (a row to a thread would touch 32 lines with every
        // store): a row's 16-byte pieces c at c ^ (row & 7), the rest of the rounding behind the rows.
        constexpr int kPieces = DP * (int)sizeof(T) / 16, kPer = 16 / (int)sizeof(T);
        uint4 *stage = reinterpret_cast<uint4 *>(smem);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            float o[32];
            if constexpr (Op::kPlanes) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float2 t = unpack2(total_o[16 * c + j]);
                    o[2 * j] = t.x;
                    o[2 * j + 1] = t.y;
                }
            } else if (n > 0) {
                tmem_load32(mine + L::kO + 32 * c, o);
                tmem_loads_done();
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = sum == 0.f ? 0.f : o[j] * inv;
            if (splits > 1) {
                if (m < p.M) {
                    float4 *dst = reinterpret_cast<float4 *>(part + ((long)split * p.B * p.G * p.M + at) * DP + 32 * c);
#pragma unroll
                    for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 32; j += kPer) {
                    uint4 v;
                    uint32_t *r = &v.x;
                    uint4 *to = stage + tid * kPieces + (((32 * c + j) / kPer) ^ (tid & 7));
                    if constexpr (Op::kPlanes) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[e] = __float_as_uint(o[j + e]);
                        *to = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[e] = pack_pair<T>(o[j + 2 * e], o[j + 2 * e + 1]);
                        *to = v;
                        if (rest) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 hi = unpack_pair<T>(r[e]);
                                r[e] = pack_pair<T>(o[j + 2 * e] - hi.x, o[j + 2 * e + 1] - hi.y);
                            }
                            to[kRowTile * kPieces] = v;
                        }
                    }
                }
            }
            __syncwarp();
        }
        if (splits == 1) {
            __syncwarp();
            // (a warp's rows are its own)
            for (int idx = tid & 31; idx < 32 * kPieces; idx += 32) {
                const int r = 32 * warp + idx / kPieces, c = idx % kPieces, row_at = m0 + r;
                if (row_at >= p.M || c * kPer >= p.D) continue;
                const int t = p.R == 1 ? row_at : row_at / p.R;
                const long to = (((long)b * p.Tq + t) * p.H + g * p.R + row_at - t * p.R) * p.D;
                const uint4 *from = stage + r * kPieces + (c ^ (r & 7));
                reinterpret_cast<uint4 *>(out + to)[c] = *from;
                if (!Op::kPlanes && rest) reinterpret_cast<uint4 *>(rest + to)[c] = from[kRowTile * kPieces];
            }
        }
        if (m < p.M) {
            if (splits > 1) part_lse[(long)split * p.B * p.G * p.M + at] = sum == 0.f ? -INFINITY : stat;
            else lse[at] = stat;
        }
        tmem_before_sync();
    }
    settle(abort_word);
    __syncthreads();
    if (warp == 4) {
        tmem_after_sync();
        tmem_free(*slot, L::kColumns);
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
    const int t = key ? w : w - key_tiles, size = key ? kKeyTile : packed_tile(p.R), end = min((t + 1) * size, key ? p.Tk : p.M);
    const int *ids = key ? p.doc_k + b * p.doc_k_sb : p.doc_q + b * p.doc_q_sb;
    int least = kNoLeast, most = -1, padding = 0;
    for (int x = t * size + lane; x < end; x += 32) {
        const int id = ids[key ? x : x / p.R];
        if (id < 0) padding = 1;
        else { least = min(least, id); most = max(most, id); }
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    padding = __any_sync(0xffffffffu, padding);
    if (lane == 0) (key ? keys + (long)b * key_tiles : rows + (long)b * row_tiles)[t] = DocRange{least, most, padding, 0};
}

template <typename T, int DP, bool BENT>
int launch(const AttnProblem &p, const CUtensorMap &map_k, const CUtensorMap &map_v, const DocRange *kr, const DocRange *rr, void *out, void *rest, float *lse, float *part, float *part_lse,
           int splits, int *error_word, cudaStream_t stream) {
    using L = Layout<T, DP>;
    if (!cuda_ok(cudaFuncSetAttribute(attention_tc_kernel<T, DP, BENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes)))
        return LUTGEMM_E_CUDA;
    const long blocks = (long)((p.M + kRowTile - 1) / kRowTile) * p.B * p.G * splits;
    if (blocks > 0x7fffffffL) return LUTGEMM_E_TOOLARGE;
    attention_tc_kernel<T, DP, BENT><<<(unsigned)blocks, kThreads, L::kBytes, stream>>>(
        p, map_k, map_v, kr, rr, static_cast<T *>(out), static_cast<T *>(rest), lse, part, part_lse, splits, error_word);
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
int key_splits(const AttnProblem &p, int dtype, int sms) {
    const long blocks = (long)((p.M + kRowTile - 1) / kRowTile) * p.B * p.G, slots = (long)sms * (dtype == LUTGEMM_F32 ? 1 : p.D <= 64 ? 3 : 2);
    const long most = (p.Tk + 4 * kKeyTile - 1) / (4 * kKeyTile), want = slots / blocks;
    return (int)(want < 2 || most < 2 ? 1 : want < most ? want : most);
}

}  // namespace

size_t doc_range_bytes(const AttnProblem &p) {
    if (!p.doc_k || p.Tk <= 4 * kKeyTile) return 0;  // a launch costs more than the few tiles that it might spare
    const int size = packed_tile(p.R);
    return sizeof(DocRange) * p.B * ((size_t)(p.Tk + kKeyTile - 1) / kKeyTile + (size_t)(p.M + size - 1) / size);
}
int doc_ranges(const AttnProblem &p, void *scratch, const DocRange **keys, const DocRange **rows, cudaStream_t stream) {
    *keys = *rows = nullptr;
    if (!doc_range_bytes(p)) return LUTGEMM_OK;
    const int size = packed_tile(p.R), kt = (p.Tk + kKeyTile - 1) / kKeyTile, rt = (p.M + size - 1) / size;
    DocRange *k = static_cast<DocRange *>(scratch), *r = k + (size_t)p.B * kt;
    *keys = k;
    *rows = r;
    attention_doc_ranges_kernel<<<dim3((kt + rt + 3) / 4, p.B), 128, 0, stream>>>(p, k, r, kt, rt);
    return launch_status();
}

// fp32: the planes of q, k and v; then ranges of documents and the parts of split rows
size_t attention_tc_scratch_bytes(const AttnProblem &p, int dtype, int sms) {
    const int splits = key_splits(p, dtype, sms), dp = p.D <= 64 ? 64 : 128;
    return (dtype == LUTGEMM_F32 ? plane_bytes(p.B, p.Tq, p.H) + 2 * plane_bytes(p.B, p.Tk, p.G) : 0) + doc_range_bytes(p) +
           (splits > 1 ? sizeof(float) * (size_t)splits * p.B * p.G * p.M * (dp + 1) : 0);
}

int attention_tc_forward(const AttnProblem &problem, int dtype, void *out, void *rest, float *lse, void *scratch, int sms, cudaStream_t stream) {
    AttnProblem p = problem;
    int *error_word = device_error_word();
    if (!error_word) return LUTGEMM_E_CUDA;
    uint8_t *at = static_cast<uint8_t *>(scratch);
    int rc;
    if (dtype == LUTGEMM_F32) {
        const size_t nq = plane_bytes(p.B, p.Tq, p.H), nk = plane_bytes(p.B, p.Tk, p.G);
        const SplitOperand ops[3] = {{p.q, reinterpret_cast<__nv_bfloat16 *>(at), p.doc_q, p.doc_q_sb, p.Tq, p.H},
                                     {p.k, reinterpret_cast<__nv_bfloat16 *>(at + nq), p.doc_k, p.doc_k_sb, p.Tk, p.G},
                                     {p.v, reinterpret_cast<__nv_bfloat16 *>(at + nq + nk), p.doc_k, p.doc_k_sb, p.Tk, p.G}};
        rc = attention_split(p, ops, 3, nullptr, nullptr, stream);
        if (rc != LUTGEMM_OK) return rc;
        p.q = plane_tensor(ops[0].to, p.Tq, p.H);
        p.k = plane_tensor(ops[1].to, p.Tk, p.G);
        p.v = plane_tensor(ops[2].to, p.Tk, p.G);
        at += nq + 2 * nk;
    }
    CUtensorMap map_k, map_v;
    const bool bf16 = dtype != LUTGEMM_F16;
    const int width = dtype == LUTGEMM_F32 ? kPlaneWidth : p.D;
    if (!attention_map(&map_k, bf16, p.k, p.B, p.Tk, p.G, 1, width) || !attention_map(&map_v, bf16, p.v, p.B, p.Tk, p.G, 1, width))
        return LUTGEMM_E_CUDA;  // (no tensor maps on this driver)
    const int splits = key_splits(p, dtype, sms), dp = p.D <= 64 ? 64 : 128;
    const DocRange *kr, *rr;
    rc = doc_ranges(p, at, &kr, &rr, stream);
    if (rc != LUTGEMM_OK) return rc;
    float *part = reinterpret_cast<float *>(at + doc_range_bytes(p)), *part_lse = part + (size_t)splits * p.B * p.G * p.M * dp;
    const bool bent = p.cap > 0.f || p.slopes || !(p.scale > 0.f);
#define RUN(T, DP) (bent ? launch<T, DP, true>(p, map_k, map_v, kr, rr, out, rest, lse, part, part_lse, splits, error_word, stream) \
                         : launch<T, DP, false>(p, map_k, map_v, kr, rr, out, rest, lse, part, part_lse, splits, error_word, stream))
    if (dtype == LUTGEMM_F32) return RUN(float, 64);
    if (dtype == LUTGEMM_BF16) return dp == 64 ? RUN(__nv_bfloat16, 64) : RUN(__nv_bfloat16, 128);
    return dp == 64 ? RUN(__half, 64) : RUN(__half, 128);
#undef RUN
}

}  // namespace lutgemm
