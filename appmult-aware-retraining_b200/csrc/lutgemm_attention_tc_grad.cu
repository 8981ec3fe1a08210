// Attention backward on the tensor cores, 16-bit operands.
//
// With P the probabilities, recomputed from the scores and the forward pass's statistics, gP = grad_o v and delta = grad_o . out:
//     dS = P (gP - delta) cap',   grad_v = P^T grad_o,   grad_k = scale dS^T q,   grad_q = scale dS k
// Two kernels of one form give grad_q and grad_k with grad_v: each block keeps 128 rows of one side and goes over the other in tiles of 64,
// so that every sum has one owner and one order and no result depends on timing.  That costs seven products per pair of tiles
// where sums by atomics would need five, which here is the smaller part of the time: the exponentials and conversions bound both.
// delta uses out before its rounding (out + out_rest): where few keys have all of the probability, the rounding of out would be
// the largest error of grad_q and grad_k.
#include "lutgemm_attention_tc.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

// ---- delta ------------------------------------------------------------------------------------------------------------
constexpr int kDeltaRows = 64;  // rows of a block of the first kernel

// delta of every packed row; for fp16 also the largest |grad_o| of every 64 rows.  8 lanes to a row, 16 bytes to a lane and step.
template <typename T>
__global__ void __launch_bounds__(256) attention_delta_kernel(const AttnProblem p, const AttnTensor go, const T *out, const T *rest,
                                                              float *delta, float *most) {
    __shared__ float top[8];
    const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 7;
    float big = 0.f;
#pragma unroll
    for (int k = 0; k < kDeltaRows / 32; ++k) {
        const int m = blockIdx.x * kDeltaRows + 32 * k + (threadIdx.x >> 3);
        float s = 0.f;
        if (m < p.M) {
            const int i = m / p.R, h = g * p.R + m - i * p.R;
            if (!p.doc_q || p.doc_q[b * p.doc_q_sb + i] >= 0) {
                const T *x = static_cast<const T *>(go.p) + b * go.sb + i * go.st + h * go.sh;
                const long at = (((long)b * p.Tq + i) * p.H + h) * p.D;
                for (int d = lane * 8; d < p.D; d += 64) {
                    const uint4 a = *reinterpret_cast<const uint4 *>(x + d), o = *reinterpret_cast<const uint4 *>(out + at + d),
                                r = *reinterpret_cast<const uint4 *>(rest + at + d);
                    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, ov[4] = {o.x, o.y, o.z, o.w}, rv[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 u = unpack_pair<T>(av[e]), v = unpack_pair<T>(ov[e]), w = unpack_pair<T>(rv[e]);
                        s += u.x * (v.x + w.x) + u.y * (v.y + w.y);
                        big = fmaxf(big, fmaxf(fabsf(u.x), fabsf(u.y)));
                    }
                }
            }
        }
#pragma unroll
        for (int d = 4; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (m < p.M && lane == 0) delta[((long)b * p.G + g) * p.M + m] = s;
    }
    if (!most) return;
#pragma unroll
    for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = big;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) big = fmaxf(big, top[w]);
        most[((long)b * p.G + g) * gridDim.x + blockIdx.x] = big;
    }
}

// ---- gradients ----------------------------------------------------------------------------------------------------------
// KEYS: the block keeps 128 keys (K and V) and goes over tiles of packed rows (Q and grad_o); else it keeps 128 packed rows (Q and
// grad_o) and goes over tiles of 64 keys.  With X, Y what it keeps and x, y the tile (x of Q or K, y of grad_o or V), a round is
//     S = X x^T, gP = Y y^T (tcgen05) -> a row to a thread: P, dS in registers -> P and dS in 16 bits to tensor memory, over S and gP ->
//     KEYS: grad_v += P y;   grad_k or grad_q += dS x     (tcgen05, first operand from tensor memory; x and y, in shared memory as
//     they were copied, serve as row and as column operands)
// A further warp brings the tiles and issues the products.  Heads of up to 64 values leave room for two blocks on an SM; with
// larger ones the accumulators fill the tensor memory of an SM, and the block has two groups of four warps that take rounds in
// turn, each with its own S and gP.
// fp16: P is kept 2^10 larger, and grad_o is taken in units of its largest value in this key head (a power of two), so that dS stays
// out of fp16's subnormal range whatever the scale of the loss.
template <typename T, int DP, bool KEYS>
struct GradLayout {
    static constexpr int kBlocks = DP / 64, kGroups = DP / 64, kStages = kGroups + 2, kPerSm = DP == 64 ? 2 : 1;
    static constexpr int kThreads = 128 * kGroups + 32;
    static constexpr uint32_t kTile = 64 * DP * 2, kX = 0, kY = 2 * kTile, kRing = 4 * kTile;  // a stage of the ring: x, y
    static constexpr uint32_t kCols = kRing + kStages * 2 * kTile;  // KEYS: for each stage -lse, -delta, documents, slopes and places of 64 rows
    static constexpr uint32_t kBars = kCols + (KEYS ? kStages * 64 * 20 : 0), kBytes = kBars + 192;
    static constexpr int kSums = KEYS ? 2 : 1;
    static constexpr uint32_t kAcc = kGroups * 128, kColumns = kAcc + kSums * DP <= 256 ? 256 : 512;
};

template <typename T, int DP, bool BENT, bool KEYS>
__global__ void __launch_bounds__(GradLayout<T, DP, KEYS>::kThreads, GradLayout<T, DP, KEYS>::kPerSm)
    attention_tc_grad_kernel(const AttnProblem p, const AttnTensor go, const __grid_constant__ CUtensorMap map_x,
                             const __grid_constant__ CUtensorMap map_y, const DocRange *key_ranges, const DocRange *row_ranges,
                             const float *lse, const float *delta, const float *most, int most_parts, T *g1, T *g2, int *error_word) {
    using L = GradLayout<T, DP, KEYS>;
    constexpr int G = L::kGroups;
    constexpr bool kBf16 = IsBf16<T>::value;
    constexpr float kShift = kBf16 ? 0.f : 10.f;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem), bars = base + L::kBars;
    const uint32_t bar_s = bars, bar_p = bars + 16, bar_acc = bars + 32, bar_full = bars + 40;  // (full: up to four stages)
    volatile int *abort_word = reinterpret_cast<int *>(smem + L::kBars + 72);
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::kBars + 76);
    volatile int *tiles = reinterpret_cast<int *>(smem + L::kBars + 80);  // of the last eight rounds begun
    float *tops = reinterpret_cast<float *>(smem + L::kBars + 128);       // of the warps
    const int tid = threadIdx.x, warp = tid >> 5;
    int bid = blockIdx.x;
    const int g = bid % p.G;
    bid /= p.G;
    const int b = bid % p.B, own_tiles = ((KEYS ? p.Tk : p.M) + 127) / 128;
    // blocks in order of falling work where masks are causal: the first keys and the last rows
    const int o0 = (KEYS ? bid / p.B : own_tiles - 1 - bid / p.B) * 128;
    const int pre = p.prefix ? p.prefix[b] : 0, size = packed_tile(p.R);
    const bool docs = p.doc_k != nullptr;
    const long stat0 = ((long)b * p.G + g) * p.M;
    if (tid == 0) {
        *abort_word = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_s + 8 * i, 2);  // the products' arrival and the issuing lane's own, which orders what it wrote
            mbar_init(bar_p + 8 * i, 128);
        }
        mbar_init(bar_acc, 1);
        for (int i = 0; i < L::kStages; ++i) mbar_init(bar_full + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // fp16: the unit of grad_o, 2^unit >= its largest value
    float unit = 1.f;
    if (!kBf16) {
        float top = 0.f;
        for (int i = tid; i < most_parts; i += L::kThreads) top = fmaxf(top, most[((long)b * p.G + g) * most_parts + i]);
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if ((tid & 31) == 0) tops[warp] = top;
    }
    if (warp == 4 * G) tmem_alloc(smem_u32(slot), L::kColumns);
    if (KEYS && size < 64) {  // rows of a tile that bulk copies never write
        for (int i = tid; i < (int)(L::kStages * 2 * L::kTile / 16); i += L::kThreads)
            *reinterpret_cast<uint4 *>(smem + L::kRing + 16 * i) = make_uint4(0, 0, 0, 0);
        writes_to_tensor_cores();
    }
    if (warp < 4) {
        if (KEYS) {
            // (like rows of one head)
            AttnProblem keys = p;
            keys.M = p.Tk;
            keys.R = 1;
            keys.doc_q = p.doc_k;
            keys.doc_q_sb = p.doc_k_sb;
            copy_row_tile<L::kBlocks>(base + L::kX, keys, p.k, b, g, o0, tid);
            copy_row_tile<L::kBlocks>(base + L::kY, keys, p.v, b, g, o0, tid);
        } else {
            copy_row_tile<L::kBlocks>(base + L::kX, p, p.q, b, g, o0, tid);
            copy_row_tile<L::kBlocks>(base + L::kY, p, go, b, g, o0, tid);
        }
        copies_end_group();
        copies_wait<0>();
        writes_to_tensor_cores();
    }
    __syncthreads();
    tmem_after_sync();
    const uint32_t tmem = *slot;
    if (!kBf16) {
        float top = 0.f;
#pragma unroll
        for (int w = 0; w < 4 * G + 1; ++w) top = fmaxf(top, tops[w]);
        // (an infinite or NaN gradient, or none at all: as it is)
        const int e = (int)(__float_as_uint(top) >> 23);
        if (e > 0 && e < 254) unit = __uint_as_float((uint32_t)(e + 1) << 23);
    }

    if (warp == 4 * G) {
        const int lane = tid & 31;
        TileWalk walk;
        if (KEYS) {
            const int last = min(o0 + 128, p.Tk) - 1;
            // rows that see the block's first key, and from where on they see its last
            const auto from = [&](int j) { return !p.causal || j < pre ? 0 : max(0, j - p.shift); };
            walk.at = (int)min((long)from(o0) * p.R, (long)p.M) / size;
            walk.end = from(o0) >= p.Tq ? 0 : (p.M + size - 1) / size;
            walk.whole_first = (int)((min((long)from(last) * p.R, (long)p.M) + size - 1) / size);
            walk.whole_last = walk.end;
            if (key_ranges) {
                walk.ranges = row_ranges + (long)b * ((p.M + size - 1) / size);
                walk.own = own_range(key_ranges + (long)b * ((p.Tk + kKeyTile - 1) / kKeyTile), o0, last + 1, kKeyTile);
            }
        } else {
            const int last = min(o0 + 128, p.M) - 1;
            walk.end = max(0, key_limit(p, last / p.R + p.shift, pre) + kKeyTile) / kKeyTile;
            walk.whole_last = max(0, key_limit(p, o0 / p.R + p.shift, pre) + 1) / kKeyTile - 1;
            if (key_ranges) {
                walk.ranges = key_ranges + (long)b * ((p.Tk + kKeyTile - 1) / kKeyTile);
                walk.own = own_range(row_ranges + (long)b * ((p.M + size - 1) / size), o0, last + 1, size);
            }
        }
        int queue[L::kStages + 1] = {};  // this round's tile and those behind it
        auto next = [&](int i) {
            const bool more = i == 0 || queue[i - 1] >= 0;
            queue[i] = more ? walk.next(docs) : -1;
        };
        auto bring = [&](int i, int n) {  // queue[i], which is round n's
            if (queue[i] < 0) return;
            const int t = queue[i] >> 1, stage = n % L::kStages;
            const uint32_t at = base + L::kRing + stage * 2 * L::kTile, bar = bar_full + 8 * stage;
            if (KEYS) {
                float *cols = reinterpret_cast<float *>(smem + L::kCols + stage * 64 * 20);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int c = lane + 32 * k, m = t * size + c;
                    const bool in = c < size && m < p.M;
                    cols[c] = in ? kShift - lse[stat0 + m] : -INFINITY;
                    cols[64 + c] = in ? -delta[stat0 + m] : 0.f;
                    const int i = in ? m / p.R : 0;
                    if (docs) reinterpret_cast<int *>(cols)[128 + c] = in ? p.doc_q[b * p.doc_q_sb + i] : -1;
                    if (BENT && p.slopes) {
                        cols[192 + c] = in ? p.slopes[g * p.R + m - i * p.R] * kLog2e : 0.f;
                        cols[256 + c] = (float)(i + p.shift);
                    }
                }
            }
            if (lane == 0) {
                tma_expect_bytes(bar, 2 * L::kBlocks * (KEYS ? size : 64) * 128);
#pragma unroll
                for (int k = 0; k < L::kBlocks; ++k) {
                    const int i0 = KEYS ? t * (size / p.R) : t * 64;
                    tma_load_5d(at + k * 64 * 128, &map_x, 64 * k, 0, i0, g, b, bar);
                    tma_load_5d(at + L::kTile + k * 64 * 128, &map_y, 64 * k, 0, i0, g, b, bar);
                }
            }
        };
        // the tile of round n has come; what padding holds must not meet a probability of zero
        auto arrived = [&](int i, int n) {
            if (queue[i] < 0) return;
            mbar_wait(bar_full + 8 * (n % L::kStages), n / L::kStages & 1, 211, abort_word, error_word);
            if (!docs) return;
            uint8_t *at = smem + L::kRing + n % L::kStages * 2 * L::kTile;
            if (KEYS) {
                const int *ids = reinterpret_cast<const int *>(smem + L::kCols + n % L::kStages * 64 * 20) + 128;
                const unsigned long long mask = __ballot_sync(0xffffffffu, ids[lane] >= 0) |
                                                (unsigned long long)__ballot_sync(0xffffffffu, ids[lane + 32] >= 0) << 32;
                if (~mask) {
                    clear_rows<L::kBlocks>(at, mask);
                    clear_rows<L::kBlocks>(at + L::kTile, mask);
                    writes_to_tensor_cores();
                }
            } else {
                const unsigned long long mask = key_mask(p, b, (queue[i] >> 1) * kKeyTile);
                if (~mask) {
                    clear_rows<L::kBlocks>(at, mask);
                    writes_to_tensor_cores();
                }
            }
        };
        constexpr uint32_t desc_s = mma_descriptor(kBf16, 64, false), desc_acc = mma_descriptor(kBf16, DP, true);
        auto issue_scores = [&](int n, int tile) {  // S and gP of round n, or word that there is none; one lane
            const uint32_t bar = bar_s + 8 * (n % G);
            tiles[n & 7] = tile;
            if (tile >= 0) {
                const uint32_t x = base + L::kRing + n % L::kStages * 2 * L::kTile, d = tmem + n % G * 128;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i)
                    mma_ss(d, smem_descriptor(base + L::kX + (i >> 2) * 128 * 128 + (i & 3) * 32, 0),
                           smem_descriptor(x + (i >> 2) * 64 * 128 + (i & 3) * 32, 0), desc_s, i > 0);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i)
                    mma_ss(d + 64, smem_descriptor(base + L::kY + (i >> 2) * 128 * 128 + (i & 3) * 32, 0),
                           smem_descriptor(x + L::kTile + (i >> 2) * 64 * 128 + (i & 3) * 32, 0), desc_s, i > 0);
                mma_commit(bar);
            } else {
                mbar_arrive(bar);
            }
            mbar_arrive(bar);
        };
#pragma unroll
        for (int i = 0; i < L::kStages; ++i) next(i);
#pragma unroll
        for (int i = 0; i < L::kStages - 1; ++i) bring(i, i);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < G; ++i) {
            arrived(i, i);
            __syncwarp();
            // (every group hears of the end in its own round)
            if (lane == 0) issue_scores(i, queue[i]);
        }
        __syncwarp();
        int n = 0;
        for (; queue[0] >= 0; ++n) {
            next(L::kStages);
            arrived(G, n + G);
            mbar_wait(bar_p + 8 * (n % G), n / G & 1, 212, abort_word, error_word);
            // the products of the round before are done, and with them its stage (before this round's commit: the barrier's parity
            // tells two phases apart, not three)
            if (n > 0) mbar_wait(bar_acc, (n - 1) & 1, 213, abort_word, error_word);
            tmem_after_sync();
            __syncwarp();
            if (lane == 0) {
                const uint32_t x = base + L::kRing + n % L::kStages * 2 * L::kTile, d = tmem + n % G * 128;
                if (KEYS)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_ts(tmem + L::kAcc, d + 8 * i, smem_descriptor(x + L::kTile + i * 16 * 128, 64 * 128), desc_acc, n > 0 || i > 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mma_ts(tmem + L::kAcc + (KEYS ? DP : 0), d + 64 + 8 * i, smem_descriptor(x + i * 16 * 128, 64 * 128), desc_acc,
                           n > 0 || i > 0);
                mma_commit(bar_acc);
                issue_scores(n + G, queue[G]);
            }
            __syncwarp();
            bring(L::kStages - 1, n + L::kStages - 1);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < L::kStages; ++i) queue[i] = queue[i + 1];
        }
        if (n > 0) mbar_wait(bar_acc, (n - 1) & 1, 214, abort_word, error_word);
        if (lane == 0) tiles[8] = n;  // rounds done
    } else {
        const int group = warp >> 2, r = tid & 127;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const Bend bend = make_bend(p);
        const float per_unit = kBf16 ? 1.f : 1.f / (unit * 1024.f);
        TileRow row{-1, -1, 0, 0.f};
        float less = 0.f, less_delta = 0.f;  // of the row
        int key = 0, from = 0x7fffffff;      // KEYS: the first packed row that sees the key
        if (KEYS) {
            key = o0 + r;
            if (key < p.Tk) {
                from = !p.causal || key < pre ? 0 : (int)min((long)max(0, key - p.shift) * p.R, 0x7fffffffL);
                if (docs) {
                    row.doc = p.doc_k[b * p.doc_k_sb + key];
                    if (row.doc < 0) from = 0x7fffffff;
                }
            }
        } else {
            row = tile_row(p, b, g, o0 + r, pre);
            less = o0 + r < p.M ? kShift - lse[stat0 + o0 + r] : -INFINITY;
            less_delta = o0 + r < p.M ? -delta[stat0 + o0 + r] : 0.f;
        }
        const bool idle = __all_sync(0xffffffffu, KEYS ? from == 0x7fffffff : row.limit < 0);
        for (int n = group;; n += G) {
            mbar_wait(bar_s + 8 * group, n / G & 1, 215, abort_word, error_word);
            const int tile = tiles[n & 7];
            if (tile < 0 || *abort_word) break;
            tmem_after_sync();
            const uint32_t at = mine + group * 128;
            if (idle) {
                mbar_arrive(bar_p + 8 * group);
                continue;
            }
            const float *cols = reinterpret_cast<const float *>(smem + L::kCols + n % L::kStages * 64 * 20);
            const int t0 = (tile >> 1) * (KEYS ? size : 64);
            const bool masked = !(tile & 1);
            const f32x2 scale2 = pack2(bend.scale2, bend.scale2), unit2 = pack2(per_unit, per_unit);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float s[32], gp[32];
                tmem_load32(at + 32 * h, s);
                tmem_load32(at + 64 + 32 * h, gp);
                tmem_loads_done();
                // which of the 32 are seen
                uint32_t seen = 0xffffffffu;
                if (masked) {
                    if (KEYS) {
                        const long skip = (long)from - t0 - 32 * h;
                        seen = skip <= 0 ? 0xffffffffu : skip >= 32 ? 0u : 0xffffffffu << skip;
                    } else {
                        const int reach = row.limit - t0 - 32 * h;
                        seen = reach >= 31 ? 0xffffffffu : reach < 0 ? 0u : 0xffffffffu >> (31 - reach);
                    }
                    if (docs) {
                        uint32_t same = 0;
                        if (KEYS) {
                            const int4 *ids = reinterpret_cast<const int4 *>(cols + 128 + 32 * h);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int4 d = ids[j];
                                same |= (uint32_t)(d.x == row.doc) << (4 * j) | (uint32_t)(d.y == row.doc) << (4 * j + 1) |
                                        (uint32_t)(d.z == row.doc) << (4 * j + 2) | (uint32_t)(d.w == row.doc) << (4 * j + 3);
                            }
                        } else {
                            const int *ids = p.doc_k + b * p.doc_k_sb + t0 + 32 * h;
                            const int have = p.Tk - t0 - 32 * h;
#pragma unroll
                            for (int j = 0; j < 32; ++j) if (j < have && ids[j] == row.doc) same |= 1u << j;
                        }
                        seen &= same;
                    }
                }
                uint32_t wp[KEYS ? 16 : 1], ws[16];
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    f32x2 l2, d2;
                    if (KEYS) {
                        l2 = *reinterpret_cast<const f32x2 *>(cols + 32 * h + j);
                        d2 = *reinterpret_cast<const f32x2 *>(cols + 64 + 32 * h + j);
                    } else {
                        l2 = pack2(less, less);
                        d2 = pack2(less_delta, less_delta);
                    }
                    float2 x;
                    float2 b2 = make_float2(1.f, 1.f);
                    if (BENT) {
                        float y[2] = {s[j], s[j + 1]};
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (p.cap > 0.f) {
                                const float q = fast_rcp(1.f + fast_exp2(y[e] * bend.in));
                                y[e] = bend.k1 - bend.k2 * q;
                                (e ? b2.y : b2.x) = 4.f * q * (1.f - q);
                            } else {
                                y[e] *= bend.scale2;
                            }
                            if (p.slopes) {
                                if (KEYS) {
                                    const int c = 32 * h + j + e;
                                    y[e] -= cols[192 + c] * fabsf(cols[256 + c] - (float)key);
                                } else {
                                    y[e] -= row.slope * fabsf((float)(row.place - t0) - (float)(32 * h + j + e));
                                }
                            }
                        }
                        x = unpack2(add2(pack2(y[0], y[1]), l2));
                    } else {
                        x = unpack2(fma2(pack2(s[j], s[j + 1]), scale2, l2));
                    }
                    float a = fast_exp2(x.x), c = fast_exp2(x.y);
                    f32x2 u = add2(pack2(gp[j], gp[j + 1]), d2);
                    if (!kBf16) u = mul2(u, unit2);
                    if (BENT) u = mul2(u, pack2(b2.x, b2.y));
                    float2 ds = unpack2(mul2(pack2(a, c), u));
                    if (masked) {  // (by choice, not by a factor: what is masked may be anything)
                        const bool sa = seen >> j & 1, sc = seen >> (j + 1) & 1;
                        a = sa ? a : 0.f;
                        c = sc ? c : 0.f;
                        ds.x = sa ? ds.x : 0.f;
                        ds.y = sc ? ds.y : 0.f;
                    }
                    if (KEYS) wp[KEYS ? j / 2 : 0] = pack_pair<T>(a, c);
                    ws[j / 2] = pack_pair<T>(ds.x, ds.y);
                }
                if constexpr (KEYS) tmem_store16(at + 16 * h, wp);
                tmem_store16(at + 64 + 16 * h, ws);
            }
            tmem_stores_done();
            tmem_before_sync();
            mbar_arrive(bar_p + 8 * group);
        }
    }
    settle(abort_word);
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    if (warp < 4 * G) {
        const int rounds = tiles[8], group = warp >> 2, r = tid & 127, o = o0 + r;
        const bool in = o < (KEYS ? p.Tk : p.M);
        bool real = in && rounds > 0;
        if (in && docs) real = real && (KEYS ? p.doc_k[b * p.doc_k_sb + o] : p.doc_q[b * p.doc_q_sb + o / p.R]) >= 0;
        if (!KEYS && in && lse[stat0 + o] == INFINITY) real = false;  // a row that sees nothing
        const int i = KEYS ? o : o / p.R, h = KEYS ? g : g * p.R + o - i * p.R;
        const long to = (((long)b * (KEYS ? p.Tk : p.Tq) + i) * (KEYS ? p.G : p.H) + h) * p.D;
        const float f1 = kBf16 ? 1.f : 1.f / 1024.f, f2 = kBf16 ? p.scale : p.scale * unit;
#pragma unroll
        for (int c = 0; c < L::kSums * DP / 32; ++c) {
            if (c % G != group) continue;
            float v[32];
            tmem_load32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + L::kAcc + 32 * c, v);
            tmem_loads_done();
            const bool second = KEYS && c < DP / 32;  // grad_v
            const int d0 = (second || !KEYS ? c : c - DP / 32) * 32;
            T *dst = second ? g2 : g1;
            const float f = second ? f1 : f2;
            if (in)
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                    if (d0 + j >= p.D) break;
                    uint4 w;
                    uint32_t *q = &w.x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[e] = real ? pack_pair<T>(v[j + 2 * e] * f, v[j + 2 * e + 1] * f) : 0u;
                    *reinterpret_cast<uint4 *>(dst + to + d0 + j) = w;
                }
            __syncwarp();
        }
        tmem_before_sync();
    }
    __syncthreads();
    if (warp == 4 * G) {
        tmem_after_sync();
        tmem_free(tmem, L::kColumns);
    }
}

template <typename T, int DP, bool BENT, bool KEYS>
int launch(const AttnProblem &p, const AttnTensor &go, const CUtensorMap &map_x, const CUtensorMap &map_y, const DocRange *kr, const DocRange *rr,
           const float *lse, const float *delta, const float *most, int most_parts, void *g1, void *g2, int *error_word, cudaStream_t stream) {
    using L = GradLayout<T, DP, KEYS>;
    if (!cuda_ok(cudaFuncSetAttribute(attention_tc_grad_kernel<T, DP, BENT, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes)))
        return LUTGEMM_E_CUDA;
    const long blocks = (long)(((KEYS ? p.Tk : p.M) + 127) / 128) * p.B * p.G;
    if (blocks > 0x7fffffffL) return LUTGEMM_E_TOOLARGE;
    attention_tc_grad_kernel<T, DP, BENT, KEYS><<<(unsigned)blocks, L::kThreads, L::kBytes, stream>>>(
        p, go, map_x, map_y, kr, rr, lse, delta, most, most_parts, static_cast<T *>(g1), static_cast<T *>(g2), error_word);
    return launch_status();
}

template <typename T, int DP>
int backward(const AttnProblem &p, const AttnTensor &go, const void *out, const void *rest, const float *lse, float *delta, float *most,
             const DocRange *kr, const DocRange *rr, void *gq, void *gk, void *gv, int *error_word, cudaStream_t stream) {
    constexpr bool bf16 = IsBf16<T>::value;
    CUtensorMap map_q, map_go, map_k, map_v;
    if (!attention_map(&map_q, bf16, p.q, p.B, p.Tq, p.G, p.R, p.D) || !attention_map(&map_go, bf16, go, p.B, p.Tq, p.G, p.R, p.D) ||
        !attention_map(&map_k, bf16, p.k, p.B, p.Tk, p.G, 1, p.D) || !attention_map(&map_v, bf16, p.v, p.B, p.Tk, p.G, 1, p.D))
        return LUTGEMM_E_BADARG;
    const int parts = (p.M + kDeltaRows - 1) / kDeltaRows;
    attention_delta_kernel<T><<<dim3(parts, p.G, p.B), 256, 0, stream>>>(p, go, static_cast<const T *>(out), static_cast<const T *>(rest), delta,
                                                                        bf16 ? nullptr : most);
    int rc = launch_status();
    if (rc != LUTGEMM_OK) return rc;
    const bool bent = p.cap > 0.f || p.slopes;
    rc = bent ? launch<T, DP, true, true>(p, go, map_q, map_go, kr, rr, lse, delta, most, parts, gk, gv, error_word, stream)
              : launch<T, DP, false, true>(p, go, map_q, map_go, kr, rr, lse, delta, most, parts, gk, gv, error_word, stream);
    if (rc != LUTGEMM_OK) return rc;
    return bent ? launch<T, DP, true, false>(p, go, map_k, map_v, kr, rr, lse, delta, most, parts, gq, nullptr, error_word, stream)
                : launch<T, DP, false, false>(p, go, map_k, map_v, kr, rr, lse, delta, most, parts, gq, nullptr, error_word, stream);
}

}  // namespace

// delta, the largest gradients, ranges of documents
size_t attention_tc_backward_scratch_bytes(const AttnProblem &p) {
    const size_t parts = (p.M + kDeltaRows - 1) / kDeltaRows;
    return doc_range_bytes(p) + sizeof(float) * p.B * p.G * (p.M + parts);
}

int attention_tc_backward(const AttnProblem &p, int dtype, const AttnTensor &go, const void *out, const void *rest, const float *lse, void *gq,
                          void *gk, void *gv, void *scratch, cudaStream_t stream) {
    int *error_word = device_error_word();
    if (!error_word) return LUTGEMM_E_CUDA;
    const DocRange *kr, *rr;
    const int rc = doc_ranges(p, scratch, &kr, &rr, stream);
    if (rc != LUTGEMM_OK) return rc;
    float *delta = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + doc_range_bytes(p)), *most = delta + (size_t)p.B * p.G * p.M;
    if (dtype == LUTGEMM_BF16)
        return p.D <= 64 ? backward<__nv_bfloat16, 64>(p, go, out, rest, lse, delta, most, kr, rr, gq, gk, gv, error_word, stream)
                         : backward<__nv_bfloat16, 128>(p, go, out, rest, lse, delta, most, kr, rr, gq, gk, gv, error_word, stream);
    return p.D <= 64 ? backward<__half, 64>(p, go, out, rest, lse, delta, most, kr, rr, gq, gk, gv, error_word, stream)
                     : backward<__half, 128>(p, go, out, rest, lse, delta, most, kr, rr, gq, gk, gv, error_word, stream);
}

}  // namespace lutgemm
