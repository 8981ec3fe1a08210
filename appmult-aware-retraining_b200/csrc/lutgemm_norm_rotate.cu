// Norm of every head of queries and keys with the rotation by position, in one pass over both:
//     n = x / sqrt(mean(x^2) + eps),   y = R(position) (n * w)
// and its backward pass, with u = R(-position) grad_y:
//     grad_w = sum over tokens and heads of u * n,   grad_x = (u*w - n * mean(u*w*n)) / sqrt(mean(x^2) + eps)
// R turns pairs of the first `rot` values by the angles of a table: pair i is (i, i + rot/2) in the half layout and (2i, 2i + 1) in
// the interleaved one; the values behind them stay.  A negative position leaves its token unturned, one beyond the table gives NaN.
// Sums and products are fp32 whatever the type, each value is rounded once.
//
// DRAM bounds these kernels.  A lane holds `slots` of two vectors of V values (16 bytes where alignment and the pairs allow) such
// that both halves of a pair are in the same lane, so a rotation needs no exchange and a norm one shuffle reduction over the few
// lanes of a head (4 for 64 bf16 values).  A group of lanes takes HEADS heads of one token at a time: weights and angles
// are loaded once for them and their loads are in flight together; a grid of few tokens takes one head per group instead, so that
// it spreads over the GPU.  Where groups go round often, the loads of the next two rounds are under way in a ring in shared memory
// (each thread reads what it asked for itself, so the ring needs no barrier) and the next angles in registers.  The blocks are
// split between queries and keys, by their groups' turns; weights then stay with a block, and so do the sums of their gradients: per lane
// in registers, per block in shared memory, over the blocks by a second kernel in ascending order, so results do not depend on
// timing.  4 x 8192 tokens of 32 + 8 bf16 heads of 128: 113 us forward (0.67 GB, 5.9 TB/s), 179 us backward (1.01 GB, 5.6 TB/s).
#include "lutgemm.h"
#include "lutgemm_attention.cuh"
#include "lutgemm_common.cuh"
#include "lutgemm_f32x2.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

constexpr int kBlock = 256;

struct Side {
    const void *x;   // [B, T, heads, D] by strides
    long sb, st, sh;
    const void *g;   // backward: gradient of y, by strides
    long gb, gt, gh;
    const float *w;  // [D] or null
    void *y;         // contiguous; backward: gradient of x
    float *part;     // backward: [blocks of this side][D] or null
    float *gw;
    int heads, blocks;
};
struct NormArgs {
    Side side[2];
    const float *cos, *sin;  // [table, rot / 2]
    const int *pos;          // [B, T] or null
    int table, B, T, D, rot, interleaved, lanes;
    float eps;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ void load_vec(float (&dst)[V], const T *src) {
    const Vec<T, V> x = *reinterpret_cast<const Vec<T, V> *>(src);
#pragma unroll
    for (int i = 0; i < V; ++i) dst[i] = to_f32<T>(x.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *dst, const float (&src)[V]) {
    Vec<T, V> x;
#pragma unroll
    for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(src[i]);
    *reinterpret_cast<Vec<T, V> *>(dst) = x;
}

// A slot's two vectors: places in the head, and the angles that turn them (-1: none).  Neighbouring lanes take neighbouring vectors, so
// that every load and store of a warp covers whole sectors: with both vectors of a slot side by side each touched half of every sector
// and the training pass of 4 x 8192 x 40 heads of 128 bf16 values took 414 us instead of 338.
struct Slot {
    int a, b, angle, angle_b;
};
template <int V>
__device__ __forceinline__ Slot slot_of(const NormArgs &p, int c) {
    Slot s;
    if (p.interleaved && V > 1) {  // pairs lie within a vector
        s.a = c * V;
        s.b = p.D / 2 + c * V;
        s.angle = s.a < p.rot ? s.a / 2 : -1;
        s.angle_b = s.b < p.rot ? s.b / 2 : -1;
    } else if (p.interleaved) {
        s.a = 2 * c;
        s.b = s.a + 1;
        s.angle = s.angle_b = s.a < p.rot ? c : -1;
    } else if (c * V >= p.rot / 2) {
        s.a = p.rot / 2 + c * V;
        s.b = s.a + (p.D - p.rot) / 2;
        s.angle = s.angle_b = -1;
    } else {
        s.a = c * V;
        s.b = s.a + p.rot / 2;
        s.angle = s.angle_b = s.a;
    }
    return s;
}
// A slot's 2V values as packed pairs, in order a, b.  P is a pair of lanes of packed fp32 arithmetic; the partner of value e in a rotation is
// the same place of the other vector (half layout) or its neighbour (interleaved).
template <int V>
struct Packed {
    static constexpr int n = V == 1 ? 1 : V;  // pairs of 2V values
    f32x2 v[n];
};
template <typename T, int V>
__device__ __forceinline__ void widen(Packed<V> &d, const Vec<T, V> &a, const Vec<T, V> &b) {
    if constexpr (V == 1) {
        d.v[0] = pack2(to_f32<T>(a.v[0]), to_f32<T>(b.v[0]));
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            d.v[i] = pack2(to_f32<T>(a.v[2 * i]), to_f32<T>(a.v[2 * i + 1]));
            d.v[V / 2 + i] = pack2(to_f32<T>(b.v[2 * i]), to_f32<T>(b.v[2 * i + 1]));
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_slot(T *p, int a, int b, const Packed<V> &d) {
    float x[V], y[V];
    if constexpr (V == 1) {
        const float2 t = unpack2(d.v[0]);
        x[0] = t.x;
        y[0] = t.y;
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 t = unpack2(d.v[i]), u = unpack2(d.v[V / 2 + i]);
            x[2 * i] = t.x;
            x[2 * i + 1] = t.y;
            y[2 * i] = u.x;
            y[2 * i + 1] = u.y;
        }
    }
    store_vec<T, V>(p + a, x);
    store_vec<T, V>(p + b, y);
}
// what the value in place i of a rotation is paired with
template <int V>
__device__ __forceinline__ f32x2 partner(const Packed<V> &d, int i, bool interleaved) {
    if (V == 1 || interleaved) {  // (with one value to a vector both layouts pair a with b)
        const float2 t = unpack2(d.v[i]);
        return pack2(t.y, t.x);
    }
    return d.v[i < V / 2 ? i + V / 2 : i - V / 2];
}
// cosines and signed sines of a slot's values: turned = x * c + partner * s
template <int V>
__device__ __forceinline__ void angles(Packed<V> &c, Packed<V> &s, const float (&co)[V], const float (&si)[V], bool interleaved) {
    if constexpr (V == 1) {
        c.v[0] = pack2(co[0], co[0]);
        s.v[0] = pack2(-si[0], si[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            if (interleaved) {  // pair i of a, pair V/2 + i of b
                c.v[i] = pack2(co[i], co[i]);
                s.v[i] = pack2(-si[i], si[i]);
                c.v[V / 2 + i] = pack2(co[V / 2 + i], co[V / 2 + i]);
                s.v[V / 2 + i] = pack2(-si[V / 2 + i], si[V / 2 + i]);
            } else {
                c.v[i] = c.v[V / 2 + i] = pack2(co[2 * i], co[2 * i + 1]);
                s.v[i] = pack2(-si[2 * i], -si[2 * i + 1]);
                s.v[V / 2 + i] = pack2(si[2 * i], si[2 * i + 1]);
            }
        }
    }
}
__device__ __forceinline__ float both(f32x2 v) {
    const float2 t = unpack2(v);
    return t.x + t.y;
}

constexpr int kStages = 3;  // rounds of vectors that a ring in shared memory holds

// V values to a vector, SPL slots to a lane, HEADS heads of a token at a time.  INTER: the interleaved layout.  RING: vectors of 16
// bytes are asked for two rounds ahead, angles one
template <typename T, int V, int SPL, int HEADS, bool INTER, bool RING, bool BACKWARD>
__global__ void __launch_bounds__(kBlock, 2) norm_rotate_kernel(const NormArgs p) {
    constexpr int N = Packed<V>::n;
    constexpr int kPieces = BACKWARD ? 4 : 2, kRing = RING ? kStages : 0;
    // the vectors on their way, [stage][head][slot][piece][thread]; backward: then sums [groups][D]
    extern __shared__ __align__(16) unsigned char shared[];
    Vec<T, V> *ring = reinterpret_cast<Vec<T, V> *>(shared) + threadIdx.x;
    float *sums = reinterpret_cast<float *>(shared);
    const bool second = (int)blockIdx.x >= p.side[0].blocks;
    const Side &sd = p.side[second];
    const int block = blockIdx.x - (second ? p.side[0].blocks : 0);
    const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = kBlock / p.lanes;
    const int chunks = (sd.heads + HEADS - 1) / HEADS, slots = p.D / (2 * V), half = p.rot / 2;
    const unsigned units = (unsigned)p.B * p.T * chunks;
    const float inv_d = 1.f / (float)p.D;
    Slot slot[SPL];
    Packed<V> w[SPL], dw[BACKWARD ? SPL : 1];
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
        const int c = lane + s * p.lanes;
        slot[s] = slot_of<V>(p, c);
        if (c >= slots) slot[s].a = -1;
#pragma unroll
        for (int i = 0; i < N; ++i) w[s].v[i] = pack2(1.f, 1.f);
        if (slot[s].a >= 0 && sd.w) {
            float x[V], y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {  // (weights may lie on any boundary)
                x[i] = sd.w[slot[s].a + i];
                y[i] = sd.w[slot[s].b + i];
            }
            if constexpr (V == 1) {
                w[s].v[0] = pack2(x[0], y[0]);
            } else {
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    w[s].v[i] = pack2(x[2 * i], x[2 * i + 1]);
                    w[s].v[V / 2 + i] = pack2(y[2 * i], y[2 * i + 1]);
                }
            }
        }
        if constexpr (BACKWARD)
#pragma unroll
            for (int i = 0; i < N; ++i) dw[s].v[i] = 0ull;
    }
    struct Unit {
        bool in;
        unsigned token, b, t;
        int h0, heads;
    };
    const auto unit = [&](unsigned u) {
        Unit r;
        r.in = u < units;
        r.token = r.in ? u / chunks : 0u;
        r.b = r.token / (unsigned)p.T;
        r.t = r.token - r.b * (unsigned)p.T;
        r.h0 = r.in ? (int)(u - r.token * chunks) * HEADS : 0;
        r.heads = r.in ? min(HEADS, sd.heads - r.h0) : 0;
        return r;
    };
    // load(where, piece, address, is there) for the vectors of a unit: a and b of x, of g
    const auto vectors = [&](const Unit &r, auto load) {
        const T *x = static_cast<const T *>(sd.x) + (long)r.b * sd.sb + (long)r.t * sd.st + r.h0 * sd.sh;
        [[maybe_unused]] const T *g = BACKWARD ? static_cast<const T *>(sd.g) + (long)r.b * sd.gb + (long)r.t * sd.gt + r.h0 * sd.gh : nullptr;
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
#pragma unroll
            for (int s = 0; s < SPL; ++s) {
                const bool there = h < r.heads && slot[s].a >= 0;
                load(h * SPL + s, 0, x + h * sd.sh + slot[s].a, there);
                load(h * SPL + s, 1, x + h * sd.sh + slot[s].b, there);
                if constexpr (BACKWARD) {
                    load(h * SPL + s, 2, g + h * sd.gh + slot[s].a, there);
                    load(h * SPL + s, 3, g + h * sd.gh + slot[s].b, there);
                }
            }
    };
    const auto fetch = [&](unsigned u, int stage) {
        vectors(unit(u), [&](int at, int piece, const T *from, bool there) {
            cp_async16_zfill(ring + (((size_t)stage * HEADS * SPL + at) * kPieces + piece) * kBlock, there ? from : static_cast<const T *>(sd.x), there);
        });
    };
    const auto place = [&](const Unit &r) { return p.pos ? (r.in ? p.pos[r.token] : -1) : (int)r.t; };
    const auto turns = [&](int at, float (&co)[SPL][V], float (&si)[SPL][V]) {
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
            // (interleaved: the first half of the angles turns a, the second b)
            constexpr int P = INTER && V > 1 ? 2 : 1, W = V / P;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const int angle = k ? slot[s].angle_b : slot[s].angle;
                const bool turned = slot[s].a >= 0 && angle >= 0 && at >= 0;
                float x[W], y[W];
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    x[i] = turned ? NAN : 1.f;  // (a position beyond the table)
                    y[i] = 0.f;
                }
                if (turned && at < p.table) {
                    load_vec<float, W>(x, p.cos + (long)at * half + angle);
                    load_vec<float, W>(y, p.sin + (long)at * half + angle);
                }
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    co[s][k * W + i] = x[i];
                    si[s][k * W + i] = y[i];
                }
            }
        }
    };
    float co[SPL][V], si[SPL][V];
    int ahead = 0;  // the place of the next unit
    // (whole warps go round together: the shuffles below are over groups of lanes of one warp)
    const unsigned u1 = (unsigned)block * groups, step = (unsigned)sd.blocks * groups;
    if constexpr (kRing > 0)
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) {
            fetch(u1 + i * step + group, i);
            cp_async_commit();
        }
    if constexpr (kRing > 0) {
        turns(place(unit(u1 + group)), co, si);
        ahead = place(unit(u1 + step + group));
    }
    int stage = 0;
    for (unsigned u0 = u1; u0 < units; u0 += step) {
        const Unit r = unit(u0 + group);
        const unsigned token = r.token;
        const int h0 = r.h0, heads = r.heads;
        T *y = static_cast<T *>(sd.y) + ((long)token * sd.heads + h0) * p.D;
        // as they lie in memory, all heads' loads in flight together
        Vec<T, V> raw[HEADS * SPL][kPieces];
        if constexpr (kRing > 0) {
            // a thread reads what it fetched itself, and fetches where it read a round ago
            cp_async_wait<kRing - 2>();
            const int next = stage == 0 ? kRing - 1 : stage - 1;
            fetch(u0 + (kRing - 1) * step + group, next);
            cp_async_commit();
#pragma unroll
            for (int i = 0; i < HEADS * SPL; ++i)
#pragma unroll
                for (int k = 0; k < kPieces; ++k) raw[i][k] = ring[(((size_t)stage * HEADS * SPL + i) * kPieces + k) * kBlock];
            stage = stage == kRing - 1 ? 0 : stage + 1;
        } else {
            vectors(r, [&](int at, int piece, const T *from, bool there) {
#pragma unroll
                for (int i = 0; i < V; ++i) raw[at][piece].v[i] = from_f32<T>(0.f);
                if (there) raw[at][piece] = *reinterpret_cast<const Vec<T, V> *>(from);
            });
        }
        if constexpr (kRing == 0) turns(place(r), co, si);
        Packed<V> c[SPL], sn[SPL];  // forward: with the weights
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
            if (BACKWARD)
#pragma unroll
                for (int i = 0; i < V; ++i) si[s][i] = -si[s][i];
            angles<V>(c[s], sn[s], co[s], si[s], INTER);
            if constexpr (!BACKWARD) {
                Packed<V> ws;
#pragma unroll
                for (int i = 0; i < N; ++i) ws.v[i] = mul2(sn[s].v[i], partner<V>(w[s], i, INTER));
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    sn[s].v[i] = ws.v[i];
                    c[s].v[i] = mul2(c[s].v[i], w[s].v[i]);
                }
            }
        }
        if constexpr (kRing > 0) {
            turns(ahead, co, si);
            ahead = place(unit(u0 + 2 * step + group));
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            Packed<V> xv[SPL], gv[SPL];
            f32x2 sq2 = 0ull;
#pragma unroll
            for (int s = 0; s < SPL; ++s) {
                widen<T, V>(xv[s], raw[h * SPL + s][0], raw[h * SPL + s][1]);
                if constexpr (BACKWARD) widen<T, V>(gv[s], raw[h * SPL + s][2], raw[h * SPL + s][3]);
#pragma unroll
                for (int i = 0; i < N; ++i) sq2 = fma2(xv[s].v[i], xv[s].v[i], sq2);
            }
            float sq = both(sq2);
            for (int d = p.lanes / 2; d; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
            // (a head that is not there: zeros, also where eps is zero and the reciprocal infinite)
            const float r = !BACKWARD || h < heads ? rsqrtf(sq * inv_d + p.eps) : 0.f;
            const f32x2 r2 = pack2(r, r);
            if constexpr (!BACKWARD) {
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    Packed<V> o;
#pragma unroll
                    for (int i = 0; i < N; ++i) xv[s].v[i] = mul2(xv[s].v[i], r2);
#pragma unroll
                    for (int i = 0; i < N; ++i) o.v[i] = fma2(partner<V>(xv[s], i, INTER), sn[s].v[i], mul2(xv[s].v[i], c[s].v[i]));
                    if (h < heads && slot[s].a >= 0) store_slot<T, V>(y + h * p.D, slot[s].a, slot[s].b, o);
                }
            } else {
                f32x2 dot2 = 0ull;
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    Packed<V> o;
#pragma unroll
                    for (int i = 0; i < N; ++i) o.v[i] = fma2(partner<V>(gv[s], i, INTER), sn[s].v[i], mul2(gv[s].v[i], c[s].v[i]));
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        xv[s].v[i] = mul2(xv[s].v[i], r2);
                        dw[s].v[i] = fma2(o.v[i], xv[s].v[i], dw[s].v[i]);  // (rows that are not there are zeros)
                        gv[s].v[i] = mul2(o.v[i], w[s].v[i]);
                        dot2 = fma2(gv[s].v[i], xv[s].v[i], dot2);
                    }
                }
                float dot = both(dot2);
                for (int d = p.lanes / 2; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
                dot *= -inv_d;
                const f32x2 d2 = pack2(dot, dot);
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
#pragma unroll
                    for (int i = 0; i < N; ++i) gv[s].v[i] = mul2(r2, fma2(xv[s].v[i], d2, gv[s].v[i]));
                    if (h < heads && slot[s].a >= 0) store_slot<T, V>(y + h * p.D, slot[s].a, slot[s].b, gv[s]);
                }
            }
        }
    }
    if constexpr (kRing > 0) {
        cp_async_wait<0>();
        __syncthreads();  // (the sums below lie where the ring did)
    }
    if constexpr (BACKWARD) {
        if (!sd.part) return;
#pragma unroll
        for (int s = 0; s < SPL; ++s)
            if (slot[s].a >= 0) store_slot<float, V>(sums + group * p.D, slot[s].a, slot[s].b, dw[s]);
        __syncthreads();
        for (int d = threadIdx.x; d < p.D; d += kBlock) {
            float t = 0.f;
            for (int k = 0; k < groups; ++k) t += sums[k * p.D + d];
            sd.part[(size_t)block * p.D + d] = t;
        }
    }
}

// gradient of the weights of a side: the blocks' sums in ascending order, 32 values of d to a block, 32 runs of blocks
__global__ void __launch_bounds__(1024) norm_weight_sums_kernel(const NormArgs p) {
    __shared__ float run[32][33];
    const Side &sd = p.side[blockIdx.y];
    if (!sd.part) return;
    const int d = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float t = 0.f;
    if (d < p.D)
        for (int i = k; i < sd.blocks; i += 32) t += sd.part[(size_t)i * p.D + d];
    run[k][threadIdx.x & 31] = t;
    __syncthreads();
    if (k == 0 && d < p.D) {
        t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += run[i][threadIdx.x];
        sd.gw[d] = t;
    }
}

template <typename T, int V, int SPL, bool BACKWARD>
int launch(NormArgs &p, int sms, cudaStream_t stream) {
    constexpr int kMany = SPL > 1 ? 1 : BACKWARD ? 2 : 4;  // (as many as leave two blocks to an SM by their registers)
    const int groups = kBlock / p.lanes;
    const long rows = (long)p.B * p.T * (p.side[0].heads + p.side[1].heads);
    const bool many = rows >= 8L * sms * groups;  // four blocks an SM with two heads to a group
    // two blocks an SM with a ring, where each goes round at least eight times: 4 x 8192 tokens of 32 + 8 bf16 heads of 128 take 305 us
    // for both passes, 338 without it; 64 x 197 tokens of 6 + 6 fp32 heads of 64, which go round twice, 59 with it and 55 without
    const bool ring = sizeof(T) * V == 16 && rows >= 8L * 2 * sms * groups * kMany;
    // blocks by turns of groups, which take as long for one head as for several (by heads, 4 x 8192 tokens of 16 + 1 bf16 heads of 128 took
    // 120 us forward, by turns 58)
    const auto share = [&](int i) { return (long)(p.side[i].heads + (many ? kMany - 1 : 0)) / (many ? kMany : 1); };
    long blocks[2];
    for (int i = 0; i < 2; ++i) {
        const int hc = many ? kMany : 1;
        const long units = (long)p.B * p.T * ((p.side[i].heads + hc - 1) / hc);
        const long most = (ring ? 2L * sms : norm_rotate_blocks(sms)) * share(i) / (share(0) + share(1));
        blocks[i] = (units + groups - 1) / groups;
        if (blocks[i] > most) blocks[i] = most > 0 ? most : 1;
        p.side[i].blocks = (int)blocks[i];
    }
    if (BACKWARD && p.side[1].part) p.side[1].part = p.side[1].part + (size_t)blocks[0] * p.D;
    const int grid = (int)(blocks[0] + blocks[1]);
    const auto run = [&](auto kernel, size_t ring_bytes) {
        const size_t sums = BACKWARD ? sizeof(float) * groups * p.D : 0, smem = ring_bytes > sums ? ring_bytes : sums;
        if (smem > 48 * 1024 && !cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem))) return LUTGEMM_E_CUDA;
        kernel<<<grid, kBlock, smem, stream>>>(p);
        return launch_status();
    };
    int rc = LUTGEMM_OK;
    if constexpr (sizeof(T) * V == 16) {
        constexpr size_t kBytes = (size_t)kStages * kMany * SPL * (BACKWARD ? 4 : 2) * kBlock * 16;
        if (ring)
            rc = p.interleaved ? run(norm_rotate_kernel<T, V, SPL, kMany, true, true, BACKWARD>, kBytes)
                               : run(norm_rotate_kernel<T, V, SPL, kMany, false, true, BACKWARD>, kBytes);
    }
    if (!ring && many)
        rc = p.interleaved ? run(norm_rotate_kernel<T, V, SPL, kMany, true, false, BACKWARD>, 0)
                           : run(norm_rotate_kernel<T, V, SPL, kMany, false, false, BACKWARD>, 0);
    else if (!ring)
        rc = p.interleaved ? run(norm_rotate_kernel<T, V, SPL, 1, true, false, BACKWARD>, 0)
                           : run(norm_rotate_kernel<T, V, SPL, 1, false, false, BACKWARD>, 0);
    if (rc == LUTGEMM_OK && BACKWARD && (p.side[0].part || p.side[1].part)) {
        norm_weight_sums_kernel<<<dim3((p.D + 31) / 32, 2), 1024, 0, stream>>>(p);
        rc = launch_status();
    }
    return rc;
}

template <typename T, bool BACKWARD>
int by_vector(NormArgs &p, int v, int sms, cudaStream_t stream) {
    const int slots = p.D / (2 * v);
    p.lanes = 1;
    while (p.lanes < slots && p.lanes < 32) p.lanes *= 2;
    if (sizeof(T) == 2 && v == 8) return launch<T, (sizeof(T) == 2 ? 8 : 4), 1, BACKWARD>(p, sms, stream);
    if (v == 4) return launch<T, 4, 1, BACKWARD>(p, sms, stream);
    if (v == 2) return launch<T, 2, 2, BACKWARD>(p, sms, stream);
    return launch<T, 1, 4, BACKWARD>(p, sms, stream);
}

// the widest vector that every access of the problem allows
int vector_width(const NormArgs &p, int size, bool backward) {
    for (int v = 16 / size; v > 1; v /= 2) {
        if (p.D % (2 * v)) continue;
        if (p.interleaved ? p.rot % (2 * v) != 0 : p.rot / 2 % v != 0 || (p.D - p.rot) % (2 * v) != 0) continue;
        const uintptr_t bytes = (uintptr_t)v * size;
        bool ok = ((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & (4 * v - 1)) == 0 && p.rot / 2 % v == 0;
        for (int i = 0; i < 2 && ok; ++i) {
            const Side &s = p.side[i];
            ok = ((reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y)) & (bytes - 1)) == 0 && s.sb % v == 0 &&
                 s.st % v == 0 && s.sh % v == 0;
            if (backward)
                ok = ok && (reinterpret_cast<uintptr_t>(s.g) & (bytes - 1)) == 0 && s.gb % v == 0 && s.gt % v == 0 && s.gh % v == 0;
        }
        if (ok) return v;
    }
    return 1;
}

NormArgs make_args(const NormRotate &n) {
    NormArgs p{};
    for (int i = 0; i < 2; ++i) {
        Side &s = p.side[i];
        s.x = n.x[i].p; s.sb = n.x[i].sb; s.st = n.x[i].st; s.sh = n.x[i].sh;
        s.g = n.g[i].p; s.gb = n.g[i].sb; s.gt = n.g[i].st; s.gh = n.g[i].sh;
        s.w = n.w[i];
        s.y = n.y[i];
        s.gw = n.gw[i];
        s.heads = n.heads[i];
    }
    p.cos = n.cos; p.sin = n.sin; p.pos = n.pos; p.table = n.table;
    p.B = n.B; p.T = n.T; p.D = n.D; p.rot = n.rot; p.interleaved = n.interleaved; p.eps = n.eps;
    return p;
}

}  // namespace

long norm_rotate_blocks(int sms) { return 6L * sms; }

int norm_rotate_forward(const NormRotate &n, int dtype, int sms, cudaStream_t stream) {
    NormArgs p = make_args(n);
    const int v = vector_width(p, dtype == LUTGEMM_F32 ? 4 : 2, false);
    if (dtype == LUTGEMM_F32) return by_vector<float, false>(p, v, sms, stream);
    if (dtype == LUTGEMM_BF16) return by_vector<__nv_bfloat16, false>(p, v, sms, stream);
    return by_vector<__half, false>(p, v, sms, stream);
}

int norm_rotate_backward(const NormRotate &n, int dtype, float *scratch, int sms, cudaStream_t stream) {
    NormArgs p = make_args(n);
    // (the second side's blocks follow the first's)
    for (int i = 0; i < 2; ++i) p.side[i].part = n.gw[i] ? scratch : nullptr;
    const int v = vector_width(p, dtype == LUTGEMM_F32 ? 4 : 2, true);
    if (dtype == LUTGEMM_F32) return by_vector<float, true>(p, v, sms, stream);
    if (dtype == LUTGEMM_BF16) return by_vector<__nv_bfloat16, true>(p, v, sms, stream);
    return by_vector<__half, true>(p, v, sms, stream);
}

}  // namespace lutgemm
