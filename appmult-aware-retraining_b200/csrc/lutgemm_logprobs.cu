// Log probability of a given class in each row of logits, the row's entropy and its most probable classes, in one pass over the
// logits, and the gradient of the first two.
//
// With m the row's largest logit, a sum over the others and d_j = m - x_j >= 0:
//     s = sum_j exp(-d_j),  u = sum_j exp(-d_j) d_j     (one occurrence of m left out of s; it adds nothing to u)
//     log p_j = -d_j - L,  L = log1p(s);   entropy = L + U,  U = u / (1 + s);   log p_j + entropy = U - d_j
// No difference of near values occurs, so a row in which one class has nearly all of the probability keeps its entropy and its
// gradient, which are what is left beside it (with the sum over all classes both are lost from 1 - p = 2^-24 on).  The pass itself
// sums over all classes; where 1 + s comes out below 2, the one thread that has m sums those around it again without it.
//     grad_j = g_logp (1[j is given] - p_j) - g_entropy p_j (log p_j + entropy);   1 - p = -expm1(log p) for the given class
//
// DRAM bounds the gradient (logits in, gradient out), issued instructions the forward pass.  A block has a row, or a part of one where
// there are few rows; every thread keeps (m, 1 + s, u) of its own values, four vectors at a time, so that the maximum is looked at
// once for 32 values of 16 bits, and the block joins them.  It also keeps which four vectors hold its largest value and how large
// the others get: a second look at values (below, and above) is then one more load, not a pass.  The most probable classes come
// from the same pass: the k-th largest of the thread groups' largest logits is a bound that at least k values reach, so only
// threads whose own largest value reaches it look at their values once more, and the candidates are ranked by counting.  Ties go
// to the lower class.  Rows with so many ties that the candidates do not fit are gone through once per answer instead.
//
// 8192 rows of 32001 bf16 classes with 5 answers: 128 us (4.1 TB/s, 74 % of the issue slots; 178 before states were joined maximum first
// and offers were made from bits), gradient 214 us (1.05 GB, 4.7 TB/s).
#include "lutgemm.h"
#include "lutgemm_attention.cuh"
#include "lutgemm_f32x2.cuh"
#include "lutgemm_kernels.h"

namespace lutgemm {

namespace {

constexpr int kMaxTop = 32, kMaxParts = 64, kCandidates = 512;

// running sums of a set of logits; the empty set has m = -inf, s = -1
struct RowState {
    float m, s, u;
};
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// sum of exp(-(d + d_j)) (d + d_j) from all = sum of exp(-d_j) and u = sum of exp(-d_j) d_j, with e = exp(-d).  Nothing where e is 0: d, from
// logits masked with a type's lowest value, may be so large that its product with a sum is infinite.  (A NaN is in the sums themselves.)
__device__ __forceinline__ float farther(float e, float d, float all, float u) { return e == 0.f ? 0.f : e * (u + d * all); }
__device__ __forceinline__ RowState join(const RowState &a, const RowState &b) {
    const RowState &x = a.m >= b.m ? a : b, &y = a.m >= b.m ? b : a;
    if (y.m == -INFINITY) return {x.m, x.s + (y.s == -1.f ? 0.f : y.s), x.u};  // (a NaN in y.s stays)
    const float d = x.m - y.m, e = __expf(-d), n = 1.f + y.s;
    return {x.m, x.s + e * n, x.u + farther(e, d, n, y.u)};
}
// order of values by whole numbers: NaN above +inf, -0 as 0 (no key is all ones: that is where the search for ties begins)
constexpr uint32_t kNanOrder = 0xfffffffeu;
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return kNanOrder;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, long j) {
    return (unsigned long long)order_of(x) << 32 | (0xffffffffu - (uint32_t)j);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    if (o == kNanOrder) return NAN;
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

struct LogpArgs {
    const void *x;
    long pitch;
    long N;
    int C, top, parts, part_len;  // part_len: classes of a part
    const long long *target;
    long long ignore;
    float *logp, *entropy, *stats;  // stats [N][3]: m, L, U
    float *top_logp;
    long long *top_at;
    RowState *part_state;           // [N][parts]
    unsigned long long *part_keys;  // [N][parts][top]
};

template <typename T>
struct Wide {
    static constexpr int n = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float get(int i) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t h = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
        const unsigned short hs = (unsigned short)h;
        return to_f32<T>(*reinterpret_cast<const T *>(&hs));
    }
    __device__ __forceinline__ f32x2 pair(int i) const { return pack2(get(2 * i), get(2 * i + 1)); }
};

// How THREADS threads share the values of [first, end) of a row: up to the first 16-byte boundary and behind the last one a value each (round
// -1), in between four vectors to a thread and round.
template <typename T, int THREADS>
struct Share {
    static constexpr int n = Wide<T>::n;
    const T *x;
    int first, end, head, vecs;

    __device__ __forceinline__ Share(const T *row, int from, int to) : x(row), first(from), end(to) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(x + first);
        head = min(end - first, (int)(((16 - (a & 15)) & 15) / sizeof(T)));
        vecs = (end - first - head) / n;
    }
    __device__ __forceinline__ int tail() const { return first + head + vecs * n; }
    __device__ __forceinline__ int rounds() const { return max(0, (vecs - (int)threadIdx.x + 4 * THREADS - 1) / (4 * THREADS)); }
    // one(place, value) for this thread's values outside the vectors
    template <typename One>
    __device__ __forceinline__ void ends(One one) const {
        if ((int)threadIdx.x < head) one(first + threadIdx.x, to_f32<T>(x[first + threadIdx.x]));
        if (tail() + (int)threadIdx.x < end) one(tail() + threadIdx.x, to_f32<T>(x[tail() + threadIdx.x]));
    }
    // the vectors of a round; how many there are
    __device__ __forceinline__ int load(Wide<T> (&w)[4], int round) const {
        const uint4 *v = reinterpret_cast<const uint4 *>(x + first + head);
        const int i = threadIdx.x + round * 4 * THREADS;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * THREADS < vecs) w[k].raw = v[i + k * THREADS];
        return min(4, (vecs - i + THREADS - 1) / THREADS);
    }
    // one(place, value) for the values of a round
    template <typename One>
    __device__ __forceinline__ void round(int r, One one) const {
        if (r < 0) {
            ends(one);
            return;
        }
        Wide<T> w[4];
        const int have = load(w, r);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < have)
#pragma unroll
                for (int i = 0; i < n; ++i) one(place(r, k) + i, w[k].get(i));
    }
    // of this thread's k-th vector of a round
    __device__ __forceinline__ int place(int r, int k) const { return first + head + (threadIdx.x + (r * 4 + k) * THREADS) * n; }
    template <typename One>
    __device__ __forceinline__ void every(One one) const {
        for (int r = -1; r < rounds(); ++r) round(r, one);
    }
};

// sums over this thread's values: 1 + s instead of s, in two parts; the round with the largest value, and the largest of the other rounds
struct ThreadState {
    float m = -INFINITY, second = -INFINITY;
    float best = 0.f, rest = 0.f, u = 0.f;  // sums of the round with m, of the others
    int at = -1;

    // a round whose largest value is `top` begins: whether it holds m now
    __device__ __forceinline__ bool raise(float top, int round) {
        if (!(top > m)) {
            second = fmaxf(second, top);
            return false;
        }
        const float d = top - m, e = __expf(-d);  // (0 from -inf)
        rest += best;
        u = farther(e, d, rest, u);
        rest *= e;
        best = 0.f;
        second = m;
        m = top;
        at = round;
        return true;
    }
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ float all() const { return rest + best; }
};

template <int THREADS>
__device__ __forceinline__ void block_sync() {
    if (THREADS == 32) __syncwarp(); else __syncthreads();
}

// the states of a block's threads joined, for all of them: the largest value first, then the sums relative to it (a join of two states
// at every step of the exchange would take an exponential and the same sums each time)
template <int THREADS>
__device__ __forceinline__ RowState join_block(const ThreadState &st, float (*shared)[3]) {
    float m = st.m;
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (THREADS > 32) {
        if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32][0] = m;
        __syncthreads();
        m = shared[0][0];
#pragma unroll
        for (int w = 1; w < THREADS / 32; ++w) m = fmaxf(m, shared[w][0]);
    }
    // (nothing but -inf: no sums of its own; a NaN among them stays in s)
    const float e = st.m == m ? 1.f : __expf(st.m - m), all = st.all();
    float s = all * e, u = st.m == -INFINITY ? 0.f : st.m == m ? st.u : farther(e, m - st.m, all, st.u);
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, d);
        u += __shfl_xor_sync(0xffffffffu, u, d);
    }
    if (THREADS > 32) {
        if (threadIdx.x % 32 == 0) {
            shared[threadIdx.x / 32][1] = s;
            shared[threadIdx.x / 32][2] = u;
        }
        __syncthreads();
        s = u = 0.f;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            s += shared[w][1];
            u += shared[w][2];
        }
    }
    return {m, m == -INFINITY && s == 0.f ? -1.f : m == -INFINITY ? s : s - 1.f, u};
}
// the states of parts joined one by one, so that s of the part with the largest value keeps its bits; for all threads of a block
template <int THREADS>
__device__ __forceinline__ RowState join_states(RowState all, RowState *shared) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const RowState other{__shfl_xor_sync(0xffffffffu, all.m, d), __shfl_xor_sync(0xffffffffu, all.s, d), __shfl_xor_sync(0xffffffffu, all.u, d)};
        // (both lanes join in the same order, so that they agree)
        all = threadIdx.x & d ? join(other, all) : join(all, other);
    }
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = all;
    __syncthreads();
    all = shared[0];
    for (int w = 1; w < THREADS / 32; ++w) all = join(all, shared[w]);
    return all;
}
template <int THREADS>
__device__ __forceinline__ float sum_block(float v, float *shared) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (THREADS == 32) return v;
    if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < THREADS / 32; ++w) v += shared[w];
    return v;
}

// the `top` largest of the candidates in order, by counting; every thread of the block
template <int THREADS, typename Put>
__device__ __forceinline__ void rank_out(const unsigned long long *cand, int n, int top, Put put) {
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long k = cand[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += cand[j] > k;
        if (rank < top) put(rank, k);
    }
}

__device__ __forceinline__ void finish_row(const LogpArgs &p, long row, RowState st, float given) {
    if (st.m == INFINITY) st.s = NAN;
    const bool none = st.m == -INFINITY && st.s == -1.f;  // no class has any probability
    const float L = none ? 0.f : log1pf(st.s), U = none ? 0.f : st.u / (1.f + st.s);
    p.stats[row * 3] = st.m;
    p.stats[row * 3 + 1] = L;
    p.stats[row * 3 + 2] = U;
    p.entropy[row] = L + U;
    const long long t = p.target[row];
    float v = 0.f;
    if (t != p.ignore) v = t < 0 || t >= p.C ? NAN : none ? -INFINITY : (given - st.m) - L;
    p.logp[row] = v;
}
__device__ __forceinline__ float logp_of(float x, float m, float L) { return m == -INFINITY ? -INFINITY : (x - m) - L; }

template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(const LogpArgs p) {
    constexpr int kGroup = THREADS >= 64 ? THREADS / 64 : 1, kGroups = THREADS / kGroup, kWarps = THREADS / 32;
    __shared__ float states[kWarps][3];
    __shared__ __align__(16) float group_top[TOP ? kGroups : 4];
    __shared__ unsigned long long cand[TOP ? kCandidates : 1];
    __shared__ int count;
    __shared__ uint32_t bound;  // in the order of whole numbers; 0: none
    const long row = blockIdx.x;
    const int part = blockIdx.y, first = part * p.part_len, end = min(p.C, first + p.part_len);
    const T *x = static_cast<const T *>(p.x) + row * p.pitch;
    const Share<T, THREADS> share(x, first, end);
    ThreadState st;
    {
        float top = -INFINITY, sum = 0.f;
        share.ends([&](int, float v) { top = fmaxf(top, v); });
        const bool best = st.raise(top, -1);
        share.ends([&](int, float v) {
            const float t = v - st.base(), e = __expf(t);
            sum += e;
            st.u += e * fminf(-t, 1e30f);  // (-inf: exp gives 0, and 0 * inf must not reach u; a NaN reaches both sums through e)
        });
        (best ? st.best : st.rest) += sum;
    }
    for (int r = 0, rounds = share.rounds(); r < rounds; ++r) {
        constexpr int n = Wide<T>::n;
        Wide<T> w[4];
        const int have = share.load(w, r);
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < have)
#pragma unroll
                for (int i = 0; i < n; ++i) top = fmaxf(top, w[k].get(i));
        const bool best = st.raise(top, r);
        const float from = -st.base();
        const f32x2 from2 = pack2(from, from), log2e2 = pack2(kLog2e, kLog2e);
        f32x2 sum2 = 0ull, u2 = 0ull;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < have)
#pragma unroll
                for (int i = 0; i < n / 2; ++i) {
                    const f32x2 t = add2(w[k].pair(i), from2);
                    const float2 z = unpack2(mul2(t, log2e2));
                    const f32x2 e = pack2(exp2_approx(z.x), exp2_approx(z.y));
                    sum2 = add2(sum2, e);
                    u2 = fma2(e, t, u2);
                }
        const float2 sum = unpack2(sum2), u = unpack2(u2);
        (best ? st.best : st.rest) += sum.x + sum.y;
        st.u -= u.x + u.y;
    }
    if (st.u != st.u && st.all() == st.all()) {  // -inf among the values: 0 * inf reached u
        st.u = 0.f;
        share.every([&](int, float v) {
            const float t = v - st.base();
            st.u += __expf(t) * fminf(-t, 1e30f);
        });
    }
    const float mine = st.m;
    RowState all = join_block<THREADS>(st, states);
    if (all.m > -INFINITY && all.s < 1.f) {
        // one class has m, and s may be all rounding of 1 + s: the sum around it without it
        float sum = st.all() * __expf(mine - all.m);  // (0 where nothing was seen)
        if (mine == all.m) {
            sum = st.rest;
            share.round(st.at, [&](int, float v) { sum += v == all.m ? 0.f : __expf(v - all.m); });
        }
        block_sync<THREADS>();
        all.s = sum_block<THREADS>(sum, &states[0][0]);
    }
    if (TOP) {
        float gt = mine;
#pragma unroll
        for (int d = 1; d < kGroup; d <<= 1) gt = fmaxf(gt, __shfl_xor_sync(0xffffffffu, gt, d));
        if (threadIdx.x % kGroup == 0) group_top[threadIdx.x / kGroup] = gt;
        if (threadIdx.x == 0) count = 0, bound = 0;
    }
    if (threadIdx.x == 0) {
        if (p.parts == 1) {
            const long long t = p.target[row];
            finish_row(p, row, all, t >= 0 && t < p.C ? to_f32<T>(x[t]) : 0.f);
        } else {
            p.part_state[row * p.parts + part] = all;
        }
    }
    if (!TOP) return;
    const int top = min(p.top, end - first);
    block_sync<THREADS>();
    if ((int)threadIdx.x < kGroups) {
        // the top-th largest of the groups' largest values, where there are as many groups: the largest that as many reach
        const float v = group_top[threadIdx.x];
        int reach = 0;
#pragma unroll
        for (int i = 0; i < kGroups; i += 4) {
            const float4 g = *reinterpret_cast<const float4 *>(group_top + i);
            reach += (g.x >= v) + (g.y >= v) + (g.z >= v) + (g.w >= v);
        }
        if (reach >= top) atomicMax(&bound, order_of(v));
    }
    block_sync<THREADS>();
    const float least = bound ? value_of((unsigned long long)bound << 32) : -INFINITY;
    const bool odd = isnan(all.s);  // NaN among the logits: the bound says nothing of them
    if (mine >= least || odd) {
        auto offer = [&](int j, float v) {
            if (!(v < least)) {
                const int at = atomicAdd(&count, 1);
                if (at < kCandidates) cand[at] = key_of(v, j);
            }
        };
        // (which values of a round reach it as bits: code for an offer in every place would not fit the instruction cache)
        auto look = [&](int r) {
            Wide<T> w[4];
            constexpr int n = Wide<T>::n;
            const int have = share.load(w, r);
            uint32_t hits = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < have)
#pragma unroll
                    for (int i = 0; i < n; ++i) hits |= w[k].get(i) < least ? 0u : 1u << (k * n + i);
            for (; hits; hits &= hits - 1) {
                const int at = __ffs(hits) - 1, j = share.place(r, at / n) + at % n;
                offer(j, to_f32<T>(x[j]));
            }
        };
        const bool all_rounds = odd || st.second >= least;
        if (all_rounds || st.at < 0) share.ends(offer);
        for (int r = all_rounds ? 0 : st.at, end = all_rounds ? share.rounds() : r + 1; r < end; ++r)
            if (r >= 0) look(r);
    }
    block_sync<THREADS>();
    const float m = all.m, L = p.parts == 1 ? p.stats[row * 3 + 1] : 0.f;
    auto put = [&](int rank, unsigned long long key) {
        if (p.parts > 1) {
            p.part_keys[(row * p.parts + part) * p.top + rank] = key;
        } else {
            p.top_logp[row * p.top + rank] = logp_of(value_of(key), m, L);
            p.top_at[row * p.top + rank] = 0xffffffffu - (uint32_t)key;
        }
    };
    if (p.parts > 1)  // a part shorter than `top`: keys below every other
        for (int i = top + threadIdx.x; i < p.top; i += THREADS) p.part_keys[(row * p.parts + part) * p.top + i] = 0;
    if (count <= kCandidates) {
        rank_out<THREADS>(cand, count, top, put);
        return;
    }
    // too many ties: the largest key below the last one, `top` times
    unsigned long long last = ~0ull;
    for (int r = 0; r < top; ++r) {
        unsigned long long best = 0;
        auto look = [&](int j, float v) {
            const unsigned long long k = key_of(v, j);
            if (k < last && k > best) best = k;
        };
        share.every(look);
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, d);
            best = o > best ? o : best;
        }
        block_sync<THREADS>();
        if (threadIdx.x % 32 == 0) cand[threadIdx.x / 32] = best;
        block_sync<THREADS>();
        for (int w = 0; w < kWarps; ++w) best = cand[w] > best ? cand[w] : best;
        if (threadIdx.x == 0) put(r, best);
        last = best;
    }
}

// joins the parts of a row
template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_join_kernel(const LogpArgs p) {
    __shared__ RowState states[8];
    __shared__ unsigned long long keys[kMaxParts * kMaxTop], cand[kCandidates], bound;
    __shared__ int count;
    const long row = blockIdx.x;
    const int total = p.parts * p.top;
    for (int i = threadIdx.x; i < total; i += 256) keys[i] = p.part_keys[row * total + i];
    const long long t = p.target[row];
    const float given = threadIdx.x == 0 && t >= 0 && t < p.C ? to_f32<T>(static_cast<const T *>(p.x)[row * p.pitch + t]) : 0.f;
    if (threadIdx.x == 0) {
        count = 0;
        bound = 0;
    }
    const RowState mine = (int)threadIdx.x < p.parts ? p.part_state[row * p.parts + threadIdx.x] : RowState{-INFINITY, -1.f, 0.f};
    const RowState all = join_states<256>(mine, states);
    if (threadIdx.x == 0) finish_row(p, row, all, given);
    if (!p.top) return;
    __syncthreads();
    // a key that at least `top` keys reach: the top-th largest of the parts' largest, where there are as many parts
    if ((int)threadIdx.x < p.parts) {
        const unsigned long long k = keys[threadIdx.x * p.top];
        int above = 0;
        for (int j = 0; j < p.parts; ++j) above += keys[j * p.top] > k;
        if (above == p.top - 1) bound = k;
    }
    __syncthreads();
    const unsigned long long least = bound > 1 ? bound : 1;
    // (at most `top` parts reach it, with `top` keys each)
    for (int i = threadIdx.x; i < total; i += 256)
        if (keys[i] >= least) {
            const int at = atomicAdd(&count, 1);
            if (at < kCandidates) cand[at] = keys[i];
        }
    __syncthreads();
    const float L = p.stats[row * 3 + 1];
    auto put = [&](int rank, unsigned long long key) {
        p.top_logp[row * p.top + rank] = logp_of(value_of(key), all.m, L);
        p.top_at[row * p.top + rank] = 0xffffffffu - (uint32_t)key;
    };
    if (count <= kCandidates) {
        rank_out<256>(cand, count, p.top, put);
        return;
    }
    for (int i = threadIdx.x; i < total; i += 256) {
        const unsigned long long k = keys[i];
        if (k < least) continue;
        int rank = 0;
        for (int j = 0; j < total; ++j) rank += keys[j] > k;
        if (rank < p.top) put(rank, k);
    }
}

struct GradArgs {
    const void *x;
    long pitch, N;
    int C;
    const long long *target;
    long long ignore;
    const float *stats, *g_logp, *g_entropy;  // either gradient may be null
    void *gx;                                 // contiguous [N, C]
    int span;                                 // classes of a block
};

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_grad_kernel(const GradArgs p) {
    const long row = blockIdx.x;
    const int first = blockIdx.y * p.span, end = min(p.C, first + p.span);
    const T *x = static_cast<const T *>(p.x) + row * p.pitch;
    T *gx = static_cast<T *>(p.gx) + row * p.C;
    constexpr int n = Wide<T>::n;
    const uintptr_t a = reinterpret_cast<uintptr_t>(x + first), b = reinterpret_cast<uintptr_t>(gx + first);
    const bool aligned = !((a ^ b) & 15);  // else rows lie differently on 16-byte boundaries
    const int head = aligned ? min(end - first, (int)(((16 - (a & 15)) & 15) / sizeof(T))) : end - first;
    const int vecs = (end - first - head) / n, tail = first + head + vecs * n;
    const uint4 *v = reinterpret_cast<const uint4 *>(x + first + head);
    uint4 *o = reinterpret_cast<uint4 *>(gx + first + head);
    Wide<T> w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if ((int)threadIdx.x + k * 256 < vecs) w[k].raw = v[threadIdx.x + k * 256];
    // (a row without any probability: p = 0 everywhere)
    const bool none = p.stats[row * 3] == -INFINITY && p.stats[row * 3 + 1] == 0.f;
    const float m = none ? 0.f : p.stats[row * 3], L = none ? INFINITY : p.stats[row * 3 + 1], U = p.stats[row * 3 + 2];
    const long long t = p.target[row];
    const bool bad = t != p.ignore && (t < 0 || t >= p.C);
    const int given = bad || t == p.ignore ? -1 : (int)t;
    const float gl = bad ? NAN : t != p.ignore && p.g_logp ? p.g_logp[row] : 0.f, ge = p.g_entropy ? p.g_entropy[row] : 0.f;
    // -p (gl + ge (U - d)), and for the given class gl more, without the difference of near values
    const f32x2 from2 = pack2(-m, -m), log2e2 = pack2(kLog2e, kLog2e), less2 = pack2(-L * kLog2e, -L * kLog2e),
                ge2 = pack2(-ge, -ge), gu2 = pack2(-(gl + ge * U), -(gl + ge * U));
    const auto grads = [&](f32x2 x) {
        const f32x2 t = add2(x, from2);
        const float2 z = unpack2(fma2(t, log2e2, less2)), d = unpack2(t);
        // (p is 0 from a distance of 88 on, where the distance, infinite or times a large g_entropy, must not reach the product as an
        // infinity; a NaN reaches it through p)
        return unpack2(mul2(pack2(exp2_approx(z.x), exp2_approx(z.y)), fma2(ge2, pack2(fmaxf(d.x, -1e4f), fmaxf(d.y, -1e4f)), gu2)));
    };
    const auto grad = [&](int j, float x) {
        if (j != given) return grads(pack2(x, x)).x;
        const float t = x - m, pr = __expf(t - L);
        return none ? 0.f : -gl * expm1f(t - L) - (pr != 0.f ? ge * pr * (t + U) : 0.f);
    };
    for (int j = threadIdx.x; j < head; j += 256) gx[first + j] = from_f32<T>(grad(first + j, to_f32<T>(x[first + j])));
    if (tail + (int)threadIdx.x < end) gx[tail + threadIdx.x] = from_f32<T>(grad(tail + threadIdx.x, to_f32<T>(x[tail + threadIdx.x])));
    for (int i = threadIdx.x; i < vecs; i += 4 * 256) {
        if (i != (int)threadIdx.x)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k * 256 < vecs) w[k].raw = v[i + k * 256];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k * 256 >= vecs) break;
            union {
                uint4 raw;
                T v[n];
            } r;
#pragma unroll
            for (int e = 0; e < n / 2; ++e) {
                const float2 g = grads(w[k].pair(e));
                r.v[2 * e] = from_f32<T>(g.x);
                r.v[2 * e + 1] = from_f32<T>(g.y);
            }
            o[i + k * 256] = r.raw;
            const int base = first + head + (i + k * 256) * n;
            if ((unsigned)(given - base) < (unsigned)n) gx[given] = from_f32<T>(grad(given, to_f32<T>(x[given])));
        }
    }
}

template <typename T, int THREADS>
void launch_forward(const LogpArgs &p, cudaStream_t stream) {
    if (p.top)
        token_logprobs_kernel<T, THREADS, true><<<dim3((unsigned)p.N, p.parts), THREADS, 0, stream>>>(p);
    else
        token_logprobs_kernel<T, THREADS, false><<<dim3((unsigned)p.N, p.parts), THREADS, 0, stream>>>(p);
}

template <typename T>
int forward(LogpArgs &p, cudaStream_t stream) {
    // a warp for short rows, two warps for longer ones (20000 x 1000 fp32: 41 us with one, 59 with two, 86 with four; 8192 x 4097 bf16:
    // 61 us with two, 65 with four), four for rows that fit many to an SM (8192 x 32001: 182 us, 195 with two), sixteen for the longest
    if (p.part_len <= (p.N >= 2048 ? 1024 : 512))
        launch_forward<T, 32>(p, stream);
    else if (p.part_len <= 6144)
        launch_forward<T, 64>(p, stream);
    else if (p.part_len <= 65536)
        launch_forward<T, 128>(p, stream);
    else
        launch_forward<T, 512>(p, stream);
    int rc = launch_status();
    if (rc == LUTGEMM_OK && p.parts > 1) {
        token_logprobs_join_kernel<T><<<(unsigned)p.N, 256, 0, stream>>>(p);
        rc = launch_status();
    }
    return rc;
}

template <typename T>
int backward(const GradArgs &p, cudaStream_t stream) {
    token_logprobs_grad_kernel<T><<<dim3((unsigned)p.N, (p.C + p.span - 1) / p.span), 256, 0, stream>>>(p);
    return launch_status();
}

}  // namespace

// parts of a row: none where the rows fill the GPU, else parts of at least 2048 classes up to two blocks to an SM
int logprobs_parts(long N, int C, int sms) {
    const long want = (2L * sms) / (N > 0 ? N : 1), most = (C + 2047) / 2048;
    const long parts = want < most ? want : most;
    return parts < 2 ? 1 : (int)(parts > kMaxParts ? kMaxParts : parts);
}
size_t logprobs_scratch_bytes(long N, int C, int top, int sms) {
    const int parts = logprobs_parts(N, C, sms);
    return parts == 1 ? 0 : (size_t)N * parts * (16 + sizeof(unsigned long long) * top);
}

int logprobs_forward(const void *x, int dtype, long pitch, long N, int C, const long long *target, long long ignore, int top, float *logp,
                     float *entropy, float *stats, float *top_logp, long long *top_at, void *scratch, int sms, cudaStream_t stream) {
    LogpArgs p{x, pitch, N, C, top, logprobs_parts(N, C, sms), C, target, ignore, logp, entropy, stats, top_logp, top_at, nullptr, nullptr};
    if (p.parts > 1) {
        p.part_len = ((C + p.parts - 1) / p.parts + 7) / 8 * 8;
        p.parts = (C + p.part_len - 1) / p.part_len;
        p.part_keys = static_cast<unsigned long long *>(scratch);
        p.part_state = reinterpret_cast<RowState *>(p.part_keys + (size_t)N * p.parts * top);
    }
    if (dtype == LUTGEMM_F32) return forward<float>(p, stream);
    if (dtype == LUTGEMM_BF16) return forward<__nv_bfloat16>(p, stream);
    return forward<__half>(p, stream);
}

int logprobs_backward(const void *x, int dtype, long pitch, long N, int C, const long long *target, long long ignore, const float *stats,
                      const float *g_logp, const float *g_entropy, void *gx, cudaStream_t stream) {
    GradArgs p{x, pitch, N, C, target, ignore, stats, g_logp, g_entropy, gx, 0};
    // four vectors to a thread, fewer where the blocks would not fill the GPU
    const int full = 4 * 256 * (dtype == LUTGEMM_F32 ? 4 : 8);
    p.span = N * ((C + full - 1) / full) < 512 ? full / 4 : full;
    while ((long)(C + p.span - 1) / p.span > 65535) p.span *= 2;
    if (dtype == LUTGEMM_F32) return backward<float>(p, stream);
    if (dtype == LUTGEMM_BF16) return backward<__nv_bfloat16>(p, stream);
    return backward<__half>(p, stream);
}

}  // namespace lutgemm
