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
// it spreads over the GPU.  The blocks are split between queries and keys, in proportion; weights then stay with a block, and
// so do the sums of their gradients: per lane in registers, per block in shared memory, over the blocks by a second kernel in
// ascending order, so results do not depend on timing.
#include "lutgemm.h"
#include "lutgemm_attention.cuh"
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

// a slot's two vectors: places in the head, and the first angle (-1: not turned)
struct Slot {
    int a, b, angle;
};
template <int V>
__device__ __forceinline__ Slot slot_of(const NormArgs &p, int c) {
    Slot s;
    if (p.interleaved || c * V >= p.rot / 2) {
        s.a = p.interleaved ? c * 2 * V : p.rot + (c - p.rot / 2 / V) * 2 * V;
        s.b = s.a + V;
        s.angle = p.interleaved && s.a < p.rot ? c * V : -1;
    } else {
        s.a = c * V;
        s.b = s.a + p.rot / 2;
        s.angle = s.a;
    }
    return s;
}
// pairs of a slot: the half layout pairs a[i] with b[i], the interleaved one neighbours in (a, b)
template <int V>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V], bool interleaved) {
    if (!interleaved || V == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * c[i] - y * s[i];
            b[i] = y * c[i] + x * s[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            float x = a[2 * i], y = a[2 * i + 1];
            a[2 * i] = x * c[i] - y * s[i];
            a[2 * i + 1] = y * c[i] + x * s[i];
            x = b[2 * i];
            y = b[2 * i + 1];
            b[2 * i] = x * c[V / 2 + i] - y * s[V / 2 + i];
            b[2 * i + 1] = y * c[V / 2 + i] + x * s[V / 2 + i];
        }
    }
}

// V values to a vector, SPL slots to a lane, HEADS heads of a token at a time
template <typename T, int V, int SPL, int HEADS, bool BACKWARD>
__global__ void __launch_bounds__(kBlock) norm_rotate_kernel(const NormArgs p) {
    extern __shared__ float sums[];  // backward: [groups][D]
    const bool second = (int)blockIdx.x >= p.side[0].blocks;
    const Side &sd = p.side[second];
    const int block = blockIdx.x - (second ? p.side[0].blocks : 0);
    const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = kBlock / p.lanes;
    const int chunks = (sd.heads + HEADS - 1) / HEADS, slots = p.D / (2 * V), half = p.rot / 2;
    const long units = (long)p.B * p.T * chunks;
    const float inv_d = 1.f / (float)p.D;
    Slot slot[SPL];
    float wa[SPL][V], wb[SPL][V], da[SPL][V], db[SPL][V];
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
        const int c = lane + s * p.lanes;
        slot[s] = slot_of<V>(p, c);
        if (c >= slots) slot[s].a = -1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            wa[s][i] = slot[s].a >= 0 && sd.w ? sd.w[slot[s].a + i] : 1.f;
            wb[s][i] = slot[s].a >= 0 && sd.w ? sd.w[slot[s].b + i] : 1.f;
            da[s][i] = db[s][i] = 0.f;
        }
    }
    // (whole warps go round together: the shuffles below are over groups of lanes of one warp)
    for (long u0 = (long)block * groups; u0 < units; u0 += (long)sd.blocks * groups) {
        const long u = u0 + group;
        const bool in = u < units;
        const long token = in ? u / chunks : 0;
        const int h0 = in ? (int)(u - token * chunks) * HEADS : 0, b = (int)(token / p.T), t = (int)(token - (long)b * p.T);
        const int at = p.pos ? (in ? p.pos[token] : -1) : t;
        const T *x = static_cast<const T *>(sd.x) + b * sd.sb + t * sd.st + h0 * sd.sh;
        const T *g = BACKWARD ? static_cast<const T *>(sd.g) + b * sd.gb + t * sd.gt + h0 * sd.gh : nullptr;
        T *y = static_cast<T *>(sd.y) + (token * sd.heads + h0) * p.D;
        float xa[HEADS][SPL][V], xb[HEADS][SPL][V], ga[BACKWARD ? HEADS : 1][SPL][V], gb[BACKWARD ? HEADS : 1][SPL][V];
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
#pragma unroll
            for (int s = 0; s < SPL; ++s) {
                const bool ok = in && h0 + h < sd.heads && slot[s].a >= 0;
                if (ok) {
                    load_vec<T, V>(xa[h][s], x + h * sd.sh + slot[s].a);
                    load_vec<T, V>(xb[h][s], x + h * sd.sh + slot[s].b);
                    if (BACKWARD) {
                        load_vec<T, V>(ga[h][s], g + h * sd.gh + slot[s].a);
                        load_vec<T, V>(gb[h][s], g + h * sd.gh + slot[s].b);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        xa[h][s][i] = xb[h][s][i] = 0.f;
                        if (BACKWARD) ga[h][s][i] = gb[h][s][i] = 0.f;
                    }
                }
            }
        float c[SPL][V], sn[SPL][V];
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
            const bool turned = slot[s].a >= 0 && slot[s].angle >= 0 && at >= 0;
#pragma unroll
            for (int i = 0; i < V; ++i) { c[s][i] = 1.f; sn[s][i] = 0.f; }
            if (turned && at < p.table) {
                load_vec<float, V>(c[s], p.cos + (long)at * half + slot[s].angle);
                load_vec<float, V>(sn[s], p.sin + (long)at * half + slot[s].angle);
            } else if (turned) {
#pragma unroll
                for (int i = 0; i < V; ++i) c[s][i] = NAN;
            }
            if (BACKWARD)
#pragma unroll
                for (int i = 0; i < V; ++i) sn[s][i] = -sn[s][i];
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            float sq = 0.f;
#pragma unroll
            for (int s = 0; s < SPL; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) sq += xa[h][s][i] * xa[h][s][i] + xb[h][s][i] * xb[h][s][i];
            for (int d = p.lanes / 2; d; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
            const float r = rsqrtf(sq * inv_d + p.eps);
            const bool row = in && h0 + h < sd.heads;
            if (!BACKWARD) {
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
#pragma unroll
                    for (int i = 0; i < V; ++i) { xa[h][s][i] *= r * wa[s][i]; xb[h][s][i] *= r * wb[s][i]; }
                    turn<V>(xa[h][s], xb[h][s], c[s], sn[s], p.interleaved);
                    if (row && slot[s].a >= 0) {
                        store_vec<T, V>(y + h * p.D + slot[s].a, xa[h][s]);
                        store_vec<T, V>(y + h * p.D + slot[s].b, xb[h][s]);
                    }
                }
            } else {
                float dot = 0.f;
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    turn<V>(ga[h][s], gb[h][s], c[s], sn[s], p.interleaved);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        xa[h][s][i] *= r;
                        xb[h][s][i] *= r;
                        da[s][i] += row ? ga[h][s][i] * xa[h][s][i] : 0.f;
                        db[s][i] += row ? gb[h][s][i] * xb[h][s][i] : 0.f;
                        ga[h][s][i] *= wa[s][i];
                        gb[h][s][i] *= wb[s][i];
                        dot += ga[h][s][i] * xa[h][s][i] + gb[h][s][i] * xb[h][s][i];
                    }
                }
                for (int d = p.lanes / 2; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
                dot *= inv_d;
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        ga[h][s][i] = r * (ga[h][s][i] - xa[h][s][i] * dot);
                        gb[h][s][i] = r * (gb[h][s][i] - xb[h][s][i] * dot);
                    }
                    if (row && slot[s].a >= 0) {
                        store_vec<T, V>(y + h * p.D + slot[s].a, ga[h][s]);
                        store_vec<T, V>(y + h * p.D + slot[s].b, gb[h][s]);
                    }
                }
            }
        }
    }
    if (!BACKWARD || !sd.part) return;
#pragma unroll
    for (int s = 0; s < SPL; ++s)
        if (slot[s].a >= 0)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                sums[group * p.D + slot[s].a + i] = da[s][i];
                sums[group * p.D + slot[s].b + i] = db[s][i];
            }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += kBlock) {
        float t = 0.f;
        for (int k = 0; k < groups; ++k) t += sums[k * p.D + d];
        sd.part[(size_t)block * p.D + d] = t;
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
    constexpr int kMany = SPL > 1 || BACKWARD ? 2 : 4;
    const int groups = kBlock / p.lanes;
    const long rows = (long)p.B * p.T * (p.side[0].heads + p.side[1].heads);
    const bool many = rows >= 8L * sms * groups;  // four blocks an SM with two heads to a group
    long blocks[2];
    for (int i = 0; i < 2; ++i) {
        const int hc = many ? kMany : 1;
        const long units = (long)p.B * p.T * ((p.side[i].heads + hc - 1) / hc);
        const long most = norm_rotate_blocks(sms) * (long)p.side[i].heads / (p.side[0].heads + p.side[1].heads);
        blocks[i] = (units + groups - 1) / groups;
        if (blocks[i] > most) blocks[i] = most > 0 ? most : 1;
        if (p.side[i].heads == 0) blocks[i] = 0;
        p.side[i].blocks = (int)blocks[i];
    }
    if (BACKWARD && p.side[1].part) p.side[1].part = p.side[1].part + (size_t)blocks[0] * p.D;
    const size_t smem = BACKWARD ? sizeof(float) * groups * p.D : 0;
    if (many)
        norm_rotate_kernel<T, V, SPL, kMany, BACKWARD><<<(int)(blocks[0] + blocks[1]), kBlock, smem, stream>>>(p);
    else
        norm_rotate_kernel<T, V, SPL, 1, BACKWARD><<<(int)(blocks[0] + blocks[1]), kBlock, smem, stream>>>(p);
    int rc = launch_status();
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
            if (s.heads == 0) continue;
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
