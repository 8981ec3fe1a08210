// Attention backward on the tensor cores: 16-bit operands, and fp32 ones as three bf16 planes.
//
// With P the probabilities, recomputed from the scores and the forward pass's statistics, gP = grad_o v and delta = grad_o . out:
//     dS = P (gP - delta) cap',   grad_v = P^T grad_o,   grad_k = scale dS^T q,   grad_q = scale dS k
// Two kernels of one form give grad_q and grad_k with grad_v: each block keeps 128 rows of one side and goes over the other in tiles of 64,
// so that every sum has one owner and one order and no result depends on timing.  That costs seven products per pair of tiles
// where sums by atomics would need five.
// delta uses out before its rounding (out + out_rest): where a few keys with near values share the probability, gP - delta is no larger than
// that rounding's product with grad_o.
#include "lutgemm_attention_tc.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

// ---- delta ------------------------------------------------------------------------------------------------------------
constexpr int kDeltaRows = 64;  // rows of a block of the first kernel

// fp16: what the score gradients of a batch row and key head are at most.  P (gP - delta) is no more than |grad_o| |v| + |delta|, the lengths as
// vectors, whichever query and key it belongs to.
struct GradBounds {
    float *length;     // of grad_o of every packed row
    float *row_most;   // of every kDeltaRows rows: the largest length, the largest |delta|
    float *key_most;   // of every kDeltaRows keys: the largest length of v
    int row_parts, key_parts;
};
// the power of two that a bound is from 2^14 to 2^15 of, so that no score gradient comes near fp16's largest value and those down to
// 2^-28 of the bound are normal; an infinite or NaN bound, or none at all: one
__device__ __forceinline__ float unit_of(float bound) {
    const int e = (int)(__float_as_uint(bound) >> 23);
    return e > 14 && e < 255 ? __uint_as_float((uint32_t)(e - 14) << 23) : 1.f;
}

// delta of every packed row; for fp16 also the bounds, the keys' by further blocks.  8 lanes to a row, 16 bytes to a lane and step.
template <typename T>
__global__ void __launch_bounds__(256) attention_delta_kernel(const AttnProblem p, const AttnTensor go, const T *out, const T *rest,
                                                              float *delta, const GradBounds bounds) {
    constexpr bool kBounds = !IsBf16<T>::value;
    __shared__ float tops[2][8];
    const int b = blockIdx.z, g = blockIdx.y, lane = threadIdx.x & 7;
    const bool keys = kBounds && (int)blockIdx.x >= bounds.row_parts;
    const int part = blockIdx.x - (keys ? bounds.row_parts : 0);
    float longest = 0.f, most = 0.f;
#pragma unroll
    for (int k = 0; k < kDeltaRows / 32; ++k) {
        const int m = part * kDeltaRows + 32 * k + (threadIdx.x >> 3);
        float s = 0.f, sq = 0.f;
        if (keys) {
            if (m < p.Tk && (!p.doc_k || p.doc_k[b * p.doc_k_sb + m] >= 0)) {
                const T *x = static_cast<const T *>(p.v.p) + b * p.v.sb + m * p.v.st + g * p.v.sh;
                for (int d = lane * 8; d < p.D; d += 64) {
                    const uint4 a = *reinterpret_cast<const uint4 *>(x + d);
                    const uint32_t av[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 u = unpack_pair<T>(av[e]);
                        sq += u.x * u.x + u.y * u.y;
                    }
                }
            }
        } else if (m < p.M) {
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
                        if (kBounds) sq += u.x * u.x + u.y * u.y;
                    }
                }
            }
        }
#pragma unroll
        for (int d = 4; d; d >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, d);
            if (kBounds) sq += __shfl_xor_sync(0xffffffffu, sq, d);
        }
        if (!keys && m < p.M && lane == 0) {
            delta[((long)b * p.G + g) * p.M + m] = s;
            if (kBounds) bounds.length[((long)b * p.G + g) * p.M + m] = sqrtf(sq);
        }
        longest = fmaxf(longest, sq);
        most = fmaxf(most, fabsf(s));
    }
    if (!kBounds) return;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        longest = fmaxf(longest, __shfl_xor_sync(0xffffffffu, longest, d));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    }
    if ((threadIdx.x & 31) == 0) {
        tops[0][threadIdx.x >> 5] = longest;
        tops[1][threadIdx.x >> 5] = most;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) {
            longest = fmaxf(longest, tops[0][w]);
            most = fmaxf(most, tops[1][w]);
        }
        const long at = (long)b * p.G + g;
        if (keys) {
            bounds.key_most[at * bounds.key_parts + part] = sqrtf(longest);
        } else {
            bounds.row_most[2 * (at * bounds.row_parts + part)] = sqrtf(longest);
            bounds.row_most[2 * (at * bounds.row_parts + part) + 1] = most;
        }
    }
}

// ---- gradients ----------------------------------------------------------------------------------------------------------
// KEYS: the block keeps 128 keys (K and V) and goes over tiles of packed rows (Q and grad_o); else it keeps 128 packed rows (Q and
// grad_o) and goes over tiles of 64 keys.  With X, Y what it keeps and x, y the tile (x of Q or K, y of grad_o or V), a round is
//     S = X x^T, gP = Y y^T (tcgen05) -> a row to a thread: P, dS in registers -> P and dS in 16 bits to tensor memory, over S and gP ->
//     KEYS: grad_v += P y;   grad_k or grad_q += dS x     (tcgen05, first operand from tensor memory; x and y, in shared memory as
//     they were copied, serve as row and as column operands)
// Eight warps share a round, four with the first 32 columns and four with the others; one further warp issues the products and one
// brings the tiles (when one warp did both, copies were asked for only behind the products of a round, which the queue of the
// tensor cores lets go one by one: a round of 128-value heads took 3200 clocks for 1300 of products).  What overlaps rounds:
//   heads of more than 64 values    their sums fill the tensor memory of an SM; two groups of eight warps take rounds in turn, each with
//                                   its own S and gP, and keep P over S and dS over gP
//   up to 64 values                 one group, P and dS over S and gP, and two blocks on an SM
//   the same with bent scores       (a cap, a bias) whose exponentials take longer: two groups with P and dS of their own, so that the
//                                   scores of a group's next round are formed as soon as this round's are in registers, by a warp
//                                   for each group; another warp issues the sums, in order.  4 x 4096 x 6 x 64 bf16: with a cap
//                                   950 us for both kernels (as above 1100), without one 600 us (as above 530)
// Results go through shared memory, which the ring has left, so that whole rows are written (a row to a thread took 6000 clocks of
// a block of 16000 where there are 197 keys).
// fp16: P is kept 2^10 larger, out of its subnormal range down to 2^-24.  dS is in units (powers of two) of what it is at most: with rows kept, for
// every row by itself; with keys kept, for all rows that the block goes over, whose sums it shares.  So dS keeps its bits whatever the
// scale of the loss and of the values down to 2^-28 of the most: P of 2^-12 in a row whose gradients are 2^-12 of the largest, say.
// fp32: P and dS are split into planes as the operands were; there is one group, and each round's sums start from zero and are added up
// in registers (in the accumulators, what additions cut off came to 2e-5 of the gradients of 4096 rows).
// No unit is full (tensor pipe 58 % with keys kept and 49 % with rows kept, exponential unit 30 and 34 %, issue 38 and 33 %): what a round
// waits for, scores, workers and sums handing over to each other, bounds both kernels.  2 x 4096, 16 / 4 heads of 128, bf16: 546 us with keys kept (256 blocks, not two
// whole rounds of the GPU), 435 with rows kept; 719 TFLOP/s of the formula's five products.
template <typename T, int DP, bool BENT, bool KEYS>
struct GradLayout {
    using Op = Operand<T, DP>;
    static constexpr bool kSmall = DP == 64 && !Op::kPlanes && !BENT;  // two blocks on an SM
    static constexpr bool kEarly = DP == 64 && !kSmall;  // P and dS have room of their own; a warp for each group's scores and one for the sums
    static constexpr int kBlocks = Op::kBlocks, kGroups = Op::kPlanes || kSmall ? 1 : 2, kPerSm = kSmall ? 2 : 1;
    static constexpr int kStages = Op::kPlanes ? 2 : kSmall ? 3 : kEarly ? 6 : 4;
    static constexpr int kWorkers = 256 * kGroups, kThreads = kWorkers + (kEarly ? 64 + 32 * kGroups : 64), kSums = KEYS ? 2 : 1;
    static constexpr uint32_t kTile = 64 * kBlocks * 128, kX = 0, kY = 2 * kTile, kRing = 4 * kTile;  // a stage of the ring: x, y
    static constexpr uint32_t kCols = kRing + kStages * 2 * kTile;  // KEYS: for each stage -lse, -delta, documents, slopes and places of 64 rows
    static constexpr uint32_t kBars = kCols + (KEYS ? kStages * 64 * 20 : 0), kBytes = kBars + 384;
    // tensor memory of a group: S, gP and, behind them or over them, P and dS (64 values of 16 bits: 32 columns); then the sums
    static constexpr uint32_t kP = kEarly ? 128 : 0, kDS = Op::kPlanes ? 224 : kEarly ? 160 : 64, kGroup = Op::kPlanes ? 320 : kEarly ? 192 : 128;
    static constexpr uint32_t kAcc = kGroups * kGroup, kColumns = kSmall ? 256 : 512;
    static_assert(kAcc + kSums * DP <= kColumns, "tensor memory");
    // where a half of the columns of P or dS lies, and the operand of the i-th sixteen of them
    __device__ static constexpr uint32_t half(int h) { return kEarly ? 16 * h : 32 * h; }
    __device__ static constexpr uint32_t sixteen(int i) { return half(i >> 1) + 8 * (i & 1); }
};

template <typename T, int DP, bool BENT, bool KEYS>
__global__ void __launch_bounds__(GradLayout<T, DP, BENT, KEYS>::kThreads, GradLayout<T, DP, BENT, KEYS>::kPerSm)
    attention_tc_grad_kernel(const AttnProblem p, const AttnTensor go, const __grid_constant__ CUtensorMap map_x,
                             const __grid_constant__ CUtensorMap map_y, const DocRange *key_ranges, const DocRange *row_ranges,
                             const float *lse, const float *delta, const GradBounds bounds, T *g1, T *g2, int *error_word) {
    using L = GradLayout<T, DP, BENT, KEYS>;
    constexpr int G = L::kGroups;
    using Op = typename L::Op;
    constexpr bool kBf16 = Op::kBf16;
    constexpr float kShift = kBf16 ? 0.f : 10.f;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem), bars = base + L::kBars;
    // S and gP of a group are formed, are in registers (early), P and dS stand, their products are done (early); the ring
    const uint32_t bar_s = bars, bar_l = bars + 16, bar_p = bars + 32, bar_acc = bars + 48, bar_full = bars + 64, bar_empty = bars + 112,
                   bar_end = bars + 160;
    volatile int *abort_word = reinterpret_cast<int *>(smem + L::kBars + 168);
    uint32_t *slot = reinterpret_cast<uint32_t *>(smem + L::kBars + 172);
    volatile int *tiles = reinterpret_cast<int *>(smem + L::kBars + 176);    // of the last eight rounds begun; then how many there were
    volatile int *brought = reinterpret_cast<int *>(smem + L::kBars + 212);  // of the stages
    volatile int *rounds_seen = reinterpret_cast<int *>(smem + L::kBars + 236);  // how many there are, once that is known
    float *tops = reinterpret_cast<float *>(smem + L::kBars + 240);          // of the workers' warps, twice 16
    const int tid = threadIdx.x, warp = warp_index();
    int bid = blockIdx.x;
    const int g = bid % p.G;
    bid /= p.G;
    const int b = bid % p.B, own_tiles = ((KEYS ? p.Tk : p.M) + 127) / 128;
    // blocks in order of falling work where masks are causal: the first keys and the last rows
    const int o0 = (KEYS ? bid / p.B : own_tiles - 1 - bid / p.B) * 128;
    const int pre = p.prefix ? p.prefix[b] : 0, size = packed_tile(p.R);
    const bool docs = p.doc_k != nullptr;
    const int width = Op::kPlanes ? kPlaneWidth : p.D;
    const long stat0 = ((long)b * p.G + g) * p.M;
    if (tid == 0) {
        *abort_word = 0;
        *rounds_seen = 0x7fffffff;
        for (int i = 0; i < G; ++i) {
            mbar_init(bar_s + 8 * i, 2);  // the products' arrival and the issuing lane's own, which orders what it wrote
            mbar_init(bar_l + 8 * i, 256);
            mbar_init(bar_p + 8 * i, 256);
            mbar_init(bar_acc + 8 * i, 1);
        }
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_empty + 8 * i, 1);
        }
        mbar_init(bar_end, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (KEYS && size < 64) {  // rows of a tile that bulk copies never write
        for (int i = tid; i < (int)(L::kStages * 2 * L::kTile / 16); i += L::kThreads)
            *reinterpret_cast<uint4 *>(smem + L::kRing + 16 * i) = make_uint4(0, 0, 0, 0);
        writes_to_tensor_cores();
    }
    __syncthreads();
    // (the warp that brings tiles begins at once; the others meet again when X and Y have come)
    float unit = 1.f;  // fp16: of dS, of this thread's row (with KEYS of the block)
    uint32_t tmem = 0;
    if (warp != L::kWorkers / 32 + 1) {
        if (warp == L::kWorkers / 32) tmem_alloc(smem_u32(slot), L::kColumns);
        if (!kBf16 && warp < L::kWorkers / 32) {
            // with KEYS the largest length of grad_o and |delta| of the rows that may see the block, else the largest length of v
            float top = 0.f, top_delta = 0.f;
            const long at = (long)b * p.G + g;
            if (KEYS) {
                const int first = p.causal && o0 >= pre ? (int)min((long)max(0, o0 - p.shift) * p.R, (long)p.M) / kDeltaRows : 0;
                for (int i = first + tid; i < bounds.row_parts; i += L::kWorkers) {
                    top = fmaxf(top, bounds.row_most[2 * (at * bounds.row_parts + i)]);
                    top_delta = fmaxf(top_delta, bounds.row_most[2 * (at * bounds.row_parts + i) + 1]);
                }
            } else {
                for (int i = tid; i < bounds.key_parts; i += L::kWorkers) top = fmaxf(top, bounds.key_most[at * bounds.key_parts + i]);
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                top_delta = fmaxf(top_delta, __shfl_xor_sync(0xffffffffu, top_delta, d));
            }
            if ((tid & 31) == 0) {
                tops[warp] = top;
                tops[16 + warp] = top_delta;
            }
        }
        if (warp < 8) {  // X by four warps, Y by four
            const bool y = warp >= 4;
            const uint32_t to = base + (y ? L::kY : L::kX);
            if (KEYS) {
                // (like rows of one head)
                AttnProblem keys = p;
                keys.M = p.Tk;
                keys.R = 1;
                keys.doc_q = p.doc_k;
                keys.doc_q_sb = p.doc_k_sb;
                copy_row_tile<L::kBlocks>(to, keys, y ? p.v : p.k, width, b, g, o0, tid & 127);
            } else {
                copy_row_tile<L::kBlocks>(to, p, y ? go : p.q, width, b, g, o0, tid & 127);
            }
            copies_end_group();
            copies_wait<0>();
            writes_to_tensor_cores();
        }
        tmem_before_sync();
        asm volatile("bar.sync 1, %0;" ::"n"(L::kThreads - 32) : "memory");
        tmem_after_sync();
        tmem = *slot;
        if (!kBf16) {
            float top = 0.f, top_delta = 0.f;
#pragma unroll
            for (int w = 0; w < L::kWorkers / 32; ++w) {
                top = fmaxf(top, tops[w]);
                top_delta = fmaxf(top_delta, tops[16 + w]);
            }
            if (KEYS) {
                const float *own = bounds.key_most + ((long)b * p.G + g) * bounds.key_parts;
                const int part = o0 / kDeltaRows;
                unit = unit_of(top * fmaxf(own[part], own[min(part + 1, bounds.key_parts - 1)]) + top_delta);
            } else {
                const int m = o0 + (tid & 127);
                if (m < p.M) unit = unit_of(bounds.length[stat0 + m] * top + fabsf(delta[stat0 + m]));
            }
        }
    }

    // of the workers: the round group, the half of a round's columns, the row
    const int group = warp >> 3, h = warp >> 2 & 1, r = tid & 127;
    f32x2 sums[Op::kPlanes ? 16 * L::kSums : 1] = {};  // fp32: the worker's half of its row's sums
    if (warp == L::kWorkers / 32 + 1) {  // brings the tiles
        const int lane = tid & 31;
        if (elect_one()) {
            tma_prefetch_map(&map_x);
            tma_prefetch_map(&map_y);
        }
        __syncwarp();
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
        int ends = 0;
        for (int n = 0;; ++n) {
            const int tile = ends ? -1 : walk.next(docs), t = tile >> 1, stage = n % L::kStages;
            // KEYS: what a round needs of its rows, two to a lane
            float row_stat[2], row_delta[2], row_slope[2], row_place[2];
            int row_doc[2];
            if (KEYS && tile >= 0)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int c = lane + 32 * k, m = t * size + c;
                    const bool in = c < size && m < p.M;
                    row_stat[k] = in ? lse[stat0 + m] : INFINITY;
                    row_delta[k] = in ? delta[stat0 + m] : 0.f;
                    if (docs || (BENT && p.slopes)) {
                        const int i = in ? m / p.R : 0;
                        if (docs) row_doc[k] = in ? p.doc_q[b * p.doc_q_sb + i] : -1;
                        if (BENT && p.slopes) {
                            row_slope[k] = in ? p.slopes[g * p.R + m - i * p.R] * kLog2e : 0.f;
                            row_place[k] = (float)(i + p.shift - o0);
                        }
                    }
                }
            if (n >= L::kStages) mbar_wait(bar_empty + 8 * stage, (n / L::kStages - 1) & 1, 211, abort_word, error_word);
            if (KEYS && tile >= 0) {
                float *cols = reinterpret_cast<float *>(smem + L::kCols + stage * 64 * 20);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int c = lane + 32 * k;
                    cols[c] = kShift - row_stat[k];
                    cols[64 + c] = -row_delta[k];
                    if (docs) reinterpret_cast<int *>(cols)[128 + c] = row_doc[k];
                    if (BENT && p.slopes) {
                        cols[192 + c] = row_slope[k];
                        cols[256 + c] = row_place[k];
                    }
                }
            }
            __syncwarp();
            if (elect_one()) {
                const uint32_t at = base + L::kRing + stage * 2 * L::kTile, bar = bar_full + 8 * stage;
                brought[stage] = tile - ends;  // (-1: the end; -2: behind it)
                if (tile >= 0) {
                    tma_expect_bytes(bar, 2 * L::kBlocks * (KEYS ? size : 64) * 128);
#pragma unroll
                    for (int k = 0; k < L::kBlocks; ++k) {
                        const int i0 = KEYS ? t * (size / p.R) : t * 64;
                        tma_load_5d(at + k * 64 * 128, &map_x, 64 * k, 0, i0, g, b, bar);
                        tma_load_5d(at + L::kTile + k * 64 * 128, &map_y, 64 * k, 0, i0, g, b, bar);
                    }
                } else {
                    mbar_arrive(bar);
                }
            }
            __syncwarp();
            ends += tile < 0;
            if (ends == G || *abort_word) break;  // (each group hears of the end)
        }
    } else if (warp >= L::kWorkers / 32) {  // issue the products
        const int lane = tid & 31;
        constexpr uint32_t desc_s = mma_descriptor(kBf16, 64, false), desc_acc = mma_descriptor(kBf16, DP, true);
        // the tile of round n when it has come; -1: there is none
        auto arrived = [&](int n, bool more) {
            int tile = -1;
            if (more) {
                const int stage = n % L::kStages;
                mbar_wait(bar_full + 8 * stage, n / L::kStages & 1, 212, abort_word, error_word);
                tile = *abort_word ? -1 : brought[stage];
                if (docs && !Op::kPlanes && tile >= 0) {
                    // what padding holds must not meet a probability of zero (planes of padding are zeros)
                    uint8_t *at = smem + L::kRing + stage * 2 * L::kTile;
                    if (KEYS) {
                        const int *ids = reinterpret_cast<const int *>(smem + L::kCols + stage * 64 * 20) + 128;
                        const unsigned long long mask = __ballot_sync(0xffffffffu, ids[lane] >= 0) |
                                                        (unsigned long long)__ballot_sync(0xffffffffu, ids[lane + 32] >= 0) << 32;
                        if (~mask) {
                            clear_rows<L::kBlocks>(at, mask);
                            clear_rows<L::kBlocks>(at + L::kTile, mask);
                            writes_to_tensor_cores();
                        }
                    } else {
                        const unsigned long long mask = key_mask(p, b, (tile >> 1) * kKeyTile);
                        if (~mask) {
                            clear_rows<L::kBlocks>(at, mask);
                            writes_to_tensor_cores();
                        }
                    }
                }
            }
            return tile;
        };
        // S and gP of round n, or word that there is none; one lane
        auto issue_scores = [&](int n, int tile) {
            const uint32_t bar = bar_s + 8 * (n % G);
            tiles[n & 7] = tile;
            if (tile >= 0) {
                const uint32_t d = tmem + n % G * L::kGroup;
                const uint64_t own = smem_descriptor(base + L::kX, 0), x = smem_descriptor(base + L::kRing + n % L::kStages * 2 * L::kTile, 0);
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int i = 0; i < 4 * Op::kProducts; ++i)
                        mma_ss(d + 64 * e, descriptor_at(own, (e ? L::kY : L::kX) + Op::a(i >> 2) * 128 * 128 + (i & 3) * 32),
                               descriptor_at(x, e * L::kTile + Op::b(i >> 2) * 64 * 128 + (i & 3) * 32), desc_s, i > 0);
                mma_commit(bar);
            } else {
                mbar_arrive(bar);
            }
            mbar_arrive(bar);
        };
        auto issue_sums = [&](int n) {
            const uint32_t d = tmem + n % G * L::kGroup;
            const uint64_t x = smem_descriptor(base + L::kRing + n % L::kStages * 2 * L::kTile, Op::kPlanes ? 0 : 64 * 128);
#pragma unroll
            for (int e = 0; e < L::kSums; ++e) {  // grad_v with KEYS, then grad_k or grad_q
                const bool first = KEYS && e == 0;
                const uint32_t from = d + (first ? L::kP : L::kDS);
                const uint64_t with = descriptor_at(x, first ? L::kTile : 0);
                if constexpr (Op::kPlanes) {
#pragma unroll
                    for (int i = 0; i < 4 * Op::kProducts; ++i)
                        mma_ts(tmem + L::kAcc + e * DP, from + 32 * Op::a(i >> 2) + L::sixteen(i & 3),
                               descriptor_at(with, Op::b(i >> 2) * 64 * 128 + (i & 3) * 16 * 128), desc_acc, i > 0);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_ts(tmem + L::kAcc + e * DP, from + L::sixteen(i), descriptor_at(with, i * 16 * 128), desc_acc, n > 0 || i > 0);
                }
            }
            mma_commit(bar_empty + 8 * (n % L::kStages));
            if (L::kEarly) mma_commit(bar_acc + 8 * (n % G));
        };
        int n = 0;
        if (!L::kEarly) {
            int ahead[G];  // tiles of the rounds that have begun
#pragma unroll
            for (int i = 0; i < G; ++i) {
                ahead[i] = arrived(i, i == 0 || ahead[i > 0 ? i - 1 : 0] >= 0);
                tmem_after_sync();
                __syncwarp();
                if (elect_one()) issue_scores(i, ahead[i]);
                __syncwarp();
            }
            for (; ahead[0] >= 0; ++n) {
                const int tile = arrived(n + G, ahead[G - 1] >= 0);
                mbar_wait(bar_p + 8 * (n % G), n / G & 1, 213, abort_word, error_word);
                tmem_after_sync();
                __syncwarp();
                if (elect_one()) {
                    issue_sums(n);
                    issue_scores(n + G, tile);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i + 1 < G; ++i) ahead[i] = ahead[i + 1];
                ahead[G - 1] = tile;
            }
        } else if (warp != L::kWorkers / 32 + 2) {  // the scores of a group
            for (int k = warp == L::kWorkers / 32 ? 0 : 1;; k += G) {
                const int tile = arrived(k, true);
                if (k >= G) mbar_wait(bar_l + 8 * (k % G), (k / G - 1) & 1, 217, abort_word, error_word);
                if (tile == -1 && k >= G) {
                    // Word of the end goes to the sums in place of the workers' arrivals, when those of the group's last round are all
                    // there and the sums have taken note of them: a barrier's parity tells two phases apart, not three.  (The
                    // first wait makes the second one sure of its phase.)
                    mbar_wait(bar_p + 8 * (k % G), (k / G - 1) & 1, 221, abort_word, error_word);
                    mbar_wait(bar_acc + 8 * (k % G), (k / G - 1) & 1, 222, abort_word, error_word);
                }
                tmem_after_sync();
                __syncwarp();
                if (elect_one()) {
                    issue_scores(k, tile);
                    if (tile == -1) {
                        *rounds_seen = k;
                        mbar_arrive_many(bar_p + 8 * (k % G), 256);
                    }
                }
                __syncwarp();
                if (tile < 0 || *abort_word) break;
            }
        } else {  // the sums
            for (;; ++n) {
                mbar_wait(bar_p + 8 * (n % G), n / G & 1, 213, abort_word, error_word);
                if (n >= *rounds_seen || *abort_word) break;
                tmem_after_sync();
                __syncwarp();
                if (elect_one()) issue_sums(n);
                __syncwarp();
            }
        }
        if (n > 0) {  // every product is done
            if (elect_one()) mma_commit(bar_end);
            __syncwarp();
            mbar_wait(bar_end, 0, 214, abort_word, error_word);
        }
        if (lane == 0 && warp == L::kWorkers / 32 + (L::kEarly ? 2 : 0)) tiles[8] = n;  // rounds done
    } else {
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const Bend bend = make_bend<Op::kPlanes>(p);
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
        // fp32: the sums of a round, which are done
        auto add_sums = [&](int n) {
            mbar_wait(bar_acc, n & 1, 218, abort_word, error_word);
            tmem_after_sync();
#pragma unroll
            for (int c = 0; c < L::kSums; ++c) {
                float v[32];
                tmem_load32(mine + L::kAcc + 32 * (L::kSums * h + c), v);
                tmem_loads_done();
#pragma unroll
                for (int j = 0; j < 16; ++j) sums[Op::kPlanes ? 16 * c + j : 0] = add2(sums[Op::kPlanes ? 16 * c + j : 0], pack2(v[2 * j], v[2 * j + 1]));
            }
        };
        int n = group;
        for (;; n += G) {
            mbar_wait(bar_s + 8 * group, n / G & 1, 215, abort_word, error_word);
            const int tile = tiles[n & 7];
            if (tile < 0 || *abort_word) break;
            tmem_after_sync();
            const uint32_t at = mine + group * L::kGroup;
            if (idle) {
                if (L::kEarly) {
                    mbar_arrive(bar_l + 8 * group);
                    // (not ahead of the others: an arrival before their last round's would be taken for that)
                    if (n >= G) mbar_wait(bar_acc + 8 * group, (n / G - 1) & 1, 220, abort_word, error_word);
                }
                mbar_arrive(bar_p + 8 * group);
                continue;
            }
            const float *cols = reinterpret_cast<const float *>(smem + L::kCols + n % L::kStages * 64 * 20);
            const int t0 = (tile >> 1) * (KEYS ? size : 64);
            const bool masked = !(tile & 1);
            const f32x2 scale2 = pack2(bend.scale2, bend.scale2), unit2 = pack2(per_unit, per_unit);
            float s[32], gp[32];
            tmem_load32(at + 32 * h, s);
            tmem_load32(at + 64 + 32 * h, gp);
            tmem_loads_done();
            if (L::kEarly) {
                tmem_before_sync();
                mbar_arrive(bar_l + 8 * group);
            }
            if (Op::kPlanes && n > 0) add_sums(n - 1);
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
            const bool small = BENT && p.cap > 0.f && bend.all_small(s);
            uint32_t wp[Op::kPlanes ? 3 : 1][16], ws[Op::kPlanes ? 3 : 1][16];
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
                f32x2 b2 = pack2(1.f, 1.f);
                if (BENT) {
                    f32x2 y;
                    if (p.cap > 0.f) {
                        if (small) {
                            y = bend.capped_small(pack2(s[j], s[j + 1]), &b2);
                        } else {
                            float da, dc;
                            const float ya = bend.template capped<Op::kPlanes>(s[j], &da), yc = bend.template capped<Op::kPlanes>(s[j + 1], &dc);
                            y = pack2(ya, yc);
                            b2 = pack2(da, dc);
                        }
                    } else {
                        y = mul2(pack2(s[j], s[j + 1]), scale2);
                    }
                    if (p.slopes) {
                        float2 away, less;  // distances, and what they take from the scores
                        if (KEYS) {
                            const int c = 32 * h + j;
                            // (from the block's first key on: places are not whole numbers of fp32 for ever)
                            away = make_float2(fabsf(cols[256 + c] - (float)r), fabsf(cols[257 + c] - (float)r));
                            less = make_float2(-cols[192 + c], -cols[193 + c]);
                        } else {
                            const float first = (float)(row.place - t0) - (float)(32 * h + j);
                            away = make_float2(fabsf(first), fabsf(first - 1.f));
                            less = make_float2(-row.slope, -row.slope);
                        }
                        y = fma2(pack2(less.x, less.y), pack2(away.x, away.y), y);
                    }
                    x = unpack2(add2(y, l2));
                } else {
                    x = unpack2(fma2(pack2(s[j], s[j + 1]), scale2, l2));
                }
                float a = fast_exp2(x.x), c = fast_exp2(x.y);
                f32x2 u = add2(pack2(gp[j], gp[j + 1]), d2);
                if (!kBf16) u = mul2(u, unit2);
                if (BENT) u = mul2(u, b2);
                float2 ds = unpack2(mul2(pack2(a, c), u));
                if (masked) {  // (by choice, not by a factor: what is masked may be anything)
                    const bool sa = seen >> j & 1, sc = seen >> (j + 1) & 1;
                    a = sa ? a : 0.f;
                    c = sc ? c : 0.f;
                    ds.x = sa ? ds.x : 0.f;
                    ds.y = sc ? ds.y : 0.f;
                }
                if (KEYS) plane_words<T>(wp, j / 2, a, c);
                plane_words<T>(ws, j / 2, ds.x, ds.y);
            }
            // the products of this group's last round are done (fp32: have been waited for)
            if (L::kEarly && !Op::kPlanes && n >= G) mbar_wait(bar_acc + 8 * group, (n / G - 1) & 1, 219, abort_word, error_word);
#pragma unroll
            for (int e = 0; e < (Op::kPlanes ? 3 : 1); ++e) {
                if constexpr (KEYS) tmem_store16(at + L::kP + 32 * e + L::half(h), wp[e]);
                tmem_store16(at + L::kDS + 32 * e + L::half(h), ws[e]);
            }
            tmem_stores_done();
            tmem_before_sync();
            mbar_arrive(bar_p + 8 * group);
        }
        if (Op::kPlanes && n > 0) add_sums(n - 1);
    }
    settle(abort_word);
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    if (warp < L::kWorkers / 32) {
        const int rounds = tiles[8], o = o0 + r;
        const bool in = o < (KEYS ? p.Tk : p.M);
        bool real = in && rounds > 0;
        if (in && docs) real = real && (KEYS ? p.doc_k[b * p.doc_k_sb + o] : p.doc_q[b * p.doc_q_sb + o / p.R]) >= 0;
        if (!KEYS && in && lse[stat0 + o] == INFINITY) real = false;  // a row that sees nothing
        const float f1 = kBf16 ? 1.f : 1.f / 1024.f, f2 = kBf16 ? p.scale : p.scale * unit;
        constexpr int kChunks = L::kSums * DP / 32, kOwn = (kChunks + 2 * G - 1) / (2 * G);  // 32 columns each
        constexpr int kPieces = DP * (int)sizeof(T) / 16;  // of 16 bytes, of a row; piece c of row r lies at c ^ (r & 7)
        uint8_t *stage = smem + L::kRing;                  // grad_q or grad_k, then grad_v
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const int c = kOwn * (2 * group + h) + k;
            if (c >= kChunks) break;
            float v[32];
            if constexpr (Op::kPlanes) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float2 t = unpack2(sums[16 * k + j]);
                    v[2 * j] = t.x;
                    v[2 * j + 1] = t.y;
                }
            } else {
                tmem_load32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + L::kAcc + 32 * c, v);
                tmem_loads_done();
            }
            const bool second = KEYS && c < DP / 32;  // grad_v
            const int d0 = (second || !KEYS ? c : c - DP / 32) * 32;
            const float f = second ? f1 : f2;
            uint4 *row_out = reinterpret_cast<uint4 *>(stage) + ((second ? 128 : 0) + r) * kPieces;
            constexpr int kPer = 16 / (int)sizeof(T);  // values of a piece
#pragma unroll
            for (int j = 0; j < 32; j += kPer) {
                uint4 w;
                uint32_t *q = &w.x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (Op::kPlanes) q[e] = real ? __float_as_uint(v[j + e] * f) : 0u;
                    else q[e] = real ? pack_pair<T>(v[j + 2 * e] * f, v[j + 2 * e + 1] * f) : 0u;
                }
                row_out[((d0 + j) / kPer) ^ (r & 7)] = w;
            }
            __syncwarp();
        }
        tmem_before_sync();
        asm volatile("bar.sync 2, %0;" ::"n"(L::kWorkers) : "memory");
        for (int idx = tid; idx < L::kSums * 128 * kPieces; idx += L::kWorkers) {
            const int which = idx / (128 * kPieces), at = idx % (128 * kPieces), row_at = at / kPieces, c = at % kPieces, m = o0 + row_at;
            if (m >= (KEYS ? p.Tk : p.M) || c * (16 / (int)sizeof(T)) >= p.D) continue;
            const int t = KEYS || p.R == 1 ? m : m / p.R, head = KEYS ? g : g * p.R + m - t * p.R;
            T *dst = (which ? g2 : g1) + (((long)b * (KEYS ? p.Tk : p.Tq) + t) * (KEYS ? p.G : p.H) + head) * p.D;
            reinterpret_cast<uint4 *>(dst)[c] = reinterpret_cast<const uint4 *>(stage)[(which * 128 + row_at) * kPieces + (c ^ (row_at & 7))];
        }
    }
    __syncthreads();
    if (warp == L::kWorkers / 32) {
        tmem_after_sync();
        tmem_free(tmem, L::kColumns);
    }
}

template <typename T, int DP, bool BENT, bool KEYS>
int launch(const AttnProblem &p, const AttnTensor &go, const CUtensorMap &map_x, const CUtensorMap &map_y, const DocRange *kr, const DocRange *rr,
           const float *lse, const float *delta, const GradBounds &bounds, void *g1, void *g2, int *error_word, cudaStream_t stream) {
    using L = GradLayout<T, DP, BENT, KEYS>;
    if (!cuda_ok(cudaFuncSetAttribute(attention_tc_grad_kernel<T, DP, BENT, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kBytes)))
        return LUTGEMM_E_CUDA;
    const long blocks = (long)(((KEYS ? p.Tk : p.M) + 127) / 128) * p.B * p.G;
    if (blocks > 0x7fffffffL) return LUTGEMM_E_TOOLARGE;
    attention_tc_grad_kernel<T, DP, BENT, KEYS><<<(unsigned)blocks, L::kThreads, L::kBytes, stream>>>(
        p, go, map_x, map_y, kr, rr, lse, delta, bounds, static_cast<T *>(g1), static_cast<T *>(g2), error_word);
    return launch_status();
}

// the two kernels; delta and, for fp16, the bounds stand in scratch
template <typename T, int DP>
int gradients(const AttnProblem &p, const AttnTensor &go, const float *lse, const float *delta, const GradBounds &bounds, const DocRange *kr,
              const DocRange *rr, void *gq, void *gk, void *gv, int *error_word, cudaStream_t stream) {
    using Op = Operand<T, DP>;
    const int width = Op::kPlanes ? kPlaneWidth : p.D;
    CUtensorMap map_q, map_go, map_k, map_v;
    if (!attention_map(&map_q, Op::kBf16, p.q, p.B, p.Tq, p.G, p.R, width) || !attention_map(&map_go, Op::kBf16, go, p.B, p.Tq, p.G, p.R, width) ||
        !attention_map(&map_k, Op::kBf16, p.k, p.B, p.Tk, p.G, 1, width) || !attention_map(&map_v, Op::kBf16, p.v, p.B, p.Tk, p.G, 1, width))
        return LUTGEMM_E_CUDA;  // (no tensor maps on this driver)
    const bool bent = p.cap > 0.f || p.slopes;
    const int rc = bent ? launch<T, DP, true, true>(p, go, map_q, map_go, kr, rr, lse, delta, bounds, gk, gv, error_word, stream)
                        : launch<T, DP, false, true>(p, go, map_q, map_go, kr, rr, lse, delta, bounds, gk, gv, error_word, stream);
    if (rc != LUTGEMM_OK) return rc;
    return bent ? launch<T, DP, true, false>(p, go, map_k, map_v, kr, rr, lse, delta, bounds, gq, nullptr, error_word, stream)
                : launch<T, DP, false, false>(p, go, map_k, map_v, kr, rr, lse, delta, bounds, gq, nullptr, error_word, stream);
}

template <typename T>
int backward(const AttnProblem &p, const AttnTensor &go, const void *out, const void *rest, const float *lse, float *delta, const DocRange *kr,
             const DocRange *rr, void *gq, void *gk, void *gv, int *error_word, cudaStream_t stream) {
    const int row_parts = (p.M + kDeltaRows - 1) / kDeltaRows, key_parts = (p.Tk + kDeltaRows - 1) / kDeltaRows;
    const long heads = (long)p.B * p.G;
    GradBounds bounds{};
    if (!IsBf16<T>::value)
        bounds = {delta + heads * p.M, delta + 2 * heads * p.M, delta + 2 * heads * (p.M + row_parts), row_parts, key_parts};
    attention_delta_kernel<T><<<dim3(row_parts + bounds.key_parts, p.G, p.B), 256, 0, stream>>>(p, go, static_cast<const T *>(out),
                                                                                               static_cast<const T *>(rest), delta, bounds);
    const int rc = launch_status();
    if (rc != LUTGEMM_OK) return rc;
    return p.D <= 64 ? gradients<T, 64>(p, go, lse, delta, bounds, kr, rr, gq, gk, gv, error_word, stream)
                     : gradients<T, 128>(p, go, lse, delta, bounds, kr, rr, gq, gk, gv, error_word, stream);
}

}  // namespace

// fp32: the planes of q, grad_o, k and v; ranges of documents, delta, fp16's bounds
size_t attention_tc_backward_scratch_bytes(const AttnProblem &p, int dtype) {
    const size_t row_parts = (p.M + kDeltaRows - 1) / kDeltaRows, key_parts = (p.Tk + kDeltaRows - 1) / kDeltaRows;
    return (dtype == LUTGEMM_F32 ? 2 * plane_bytes(p.B, p.Tq, p.H) + 2 * plane_bytes(p.B, p.Tk, p.G) : 0) + doc_range_bytes(p) +
           sizeof(float) * p.B * p.G * (p.M + (dtype == LUTGEMM_F16 ? p.M + 2 * row_parts + key_parts : 0));
}

int attention_tc_backward(const AttnProblem &problem, int dtype, const AttnTensor &grad, const void *out, const void *rest, const float *lse,
                          void *gq, void *gk, void *gv, void *scratch, cudaStream_t stream) {
    AttnProblem p = problem;
    int *error_word = device_error_word();
    if (!error_word) return LUTGEMM_E_CUDA;
    uint8_t *at = static_cast<uint8_t *>(scratch);
    const size_t nq = plane_bytes(p.B, p.Tq, p.H), nk = plane_bytes(p.B, p.Tk, p.G);
    if (dtype == LUTGEMM_F32) at += 2 * nq + 2 * nk;
    const DocRange *kr, *rr;
    int rc = doc_ranges(p, at, &kr, &rr, stream);
    if (rc != LUTGEMM_OK) return rc;
    float *delta = reinterpret_cast<float *>(at + doc_range_bytes(p));
    if (dtype == LUTGEMM_BF16) return backward<__nv_bfloat16>(p, grad, out, rest, lse, delta, kr, rr, gq, gk, gv, error_word, stream);
    if (dtype == LUTGEMM_F16) return backward<__half>(p, grad, out, rest, lse, delta, kr, rr, gq, gk, gv, error_word, stream);
    __nv_bfloat16 *planes = static_cast<__nv_bfloat16 *>(scratch);
    const SplitOperand ops[4] = {{p.q, planes, p.doc_q, p.doc_q_sb, p.Tq, p.H},
                                 {p.k, planes + nq / 2, p.doc_k, p.doc_k_sb, p.Tk, p.G},
                                 {p.v, planes + (nq + nk) / 2, p.doc_k, p.doc_k_sb, p.Tk, p.G},
                                 {grad, planes + nq / 2 + nk, p.doc_q, p.doc_q_sb, p.Tq, p.H}};
    rc = attention_split(p, ops, 4, static_cast<const float *>(out), delta, stream);
    if (rc != LUTGEMM_OK) return rc;
    p.q = plane_tensor(ops[0].to, p.Tq, p.H);
    p.k = plane_tensor(ops[1].to, p.Tk, p.G);
    p.v = plane_tensor(ops[2].to, p.Tk, p.G);
    return gradients<float, 64>(p, plane_tensor(ops[3].to, p.Tq, p.H), lse, delta, GradBounds{}, kr, rr, gq, gk, gv, error_word, stream);
}

}  // namespace lutgemm
