// token_logprobs.cu — log probabilities of given tokens, entropy and the k
// likeliest tokens of rows of logits (bh_token_logprobs).
//
// With u = scale * x, m = max u: z = sum e^(u - m), a = sum (u - m) e^(u - m);
// log p(i) = u_i - m - ln z, entropy = ln z - a / z. One pass: every thread
// keeps (m, z, a) of the values it has seen. HBM bound for many rows; latency
// bound for a few. Measured in a graph, rows of 151936: 2048 of bf16 with the 20
// likeliest 122 us, 5.1 TB/s; 8 of fp32 with the 8 likeliest 11 us, of which the
// read is 0.8.
//
// What the pass needs of the arithmetic units is about five instructions a
// value where bf16 at full bandwidth leaves room for eleven: pairs of fp32
// operations, and m in use only follows a larger value by more than 2^8 (z and
// a then stay far from overflow), so that the sums are rescaled once or twice.
//
// The same pass costs the top k almost nothing: a thread also remembers where
// its largest value was, and the largest of its other vectors. The k-th largest
// of the CTA's thread maxima is a lower bound of its k-th largest value, so
// after the pass only the vectors behind the maxima that reach it, and the few
// threads whose other vectors reach it too, are looked at again: a few more than
// k candidates to sort. (Looking through all vectors of each such thread read a
// third more from memory.) Order is by 64-bit keys (value, lowest index first),
// all different, so the result does not depend on who came first.
//
// Rows are split over CTAs when there are fewer rows than the machine has room
// for; the last CTA of a row to arrive joins the parts in their order.
#include "paged_kv.cuh"

namespace bh {

constexpr int LP_THREADS = 256;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_CAND = 2048;  // candidates of a CTA before it falls back to one search for each of the k

struct LogprobParams {
    const void* logits;
    const int32_t* tokens;
    float *logprob, *entropy, *top_lp;
    int32_t* top_ids;
    uint32_t* counters;
    uint8_t* partials;
    int64_t row_stride;
    float scale;
    int n_rows, n_vocab, n_given, k, splits;
};

// Partial result of one (row, split): m, z, a, then BH_MAX_TOP keys.
struct LogprobPart {
    float m, z, a, pad;
    uint64_t top[BH_MAX_TOP];
};

// Larger key = larger value, equal values by the lowest index; NaN below
// everything; 0 is below every key.
__device__ __forceinline__ uint64_t top_key(float x, uint32_t index) {
    const uint32_t b = __float_as_uint(x + 0.f);  // -0 counts as 0
    const uint32_t o = x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((uint64_t)o << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o == 0 ? 0x7fffffffu : (o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
    return __shfl_xor_sync(0xffffffffu, (unsigned long long)v, m);
}

// Bitonic sort of one key a lane, descending by lane.
__device__ __forceinline__ uint64_t warp_sort(uint64_t v, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const uint64_t o = shfl_xor64(v, d);
            const bool keep_max = ((lane & d) == 0) == ((lane & size) == 0);
            v = (v > o) == keep_max ? v : o;
        }
    }
    return v;
}
// The 32 largest of two descending lists of 32, descending.
__device__ __forceinline__ uint64_t warp_merge(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = __shfl_sync(0xffffffffu, (unsigned long long)b, 31 - lane);
    uint64_t v = a > r ? a : r;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const uint64_t o = shfl_xor64(v, d);
        v = (v > o) == ((lane & d) == 0) ? v : o;
    }
    return v;
}

// The CTA's 32 largest of one sorted list a warp, in lists[0][0..32).
__device__ __forceinline__ void block_merge(uint64_t mine, uint64_t (*lists)[32], int warp, int lane) {
    lists[warp][lane] = mine;
#pragma unroll
    for (int d = LP_WARPS / 2; d > 0; d >>= 1) {
        __syncthreads();
        if (warp < d) lists[warp][lane] = warp_merge(lists[warp][lane], lists[warp + d][lane], lane);
    }
    __syncthreads();
}

struct Softmax {
    float m, z, a;  // raw maximum; sums in units of log2: a = sum t 2^t, t = (x - m) * c
};
__device__ __forceinline__ float fmax_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// (x - m) * c, at least -200 so that a probability of 0 adds 0 to both sums
__device__ __forceinline__ float log2_term(float x, float m, float c) { return fmax_nan((x - m) * c, -200.f); }
__device__ __forceinline__ float pow2(float t) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
    return r;
}
__device__ __forceinline__ void rebase(Softmax& s, float m, float c) {
    const float t = log2_term(s.m, m, c), f = pow2(t);
    s.a = __fmaf_rn(s.z, t, s.a) * f;
    s.z *= f;
    s.m = m;
}
__device__ __forceinline__ Softmax join(Softmax x, Softmax y, float c) {
    const float m = fmaxf(x.m, y.m);
    rebase(x, m, c);
    rebase(y, m, c);
    return Softmax{m, x.z + y.z, x.a + y.a};
}

// The CTA's sums from every thread's, in a fixed order.
__device__ __forceinline__ void block_join(Softmax& s, Softmax* warps, int warp, int lane, float c) {
    // a warp's and then the CTA's maximum first, so that every thread rescales once
    float m = s.m;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    __syncthreads();
    if (lane == 0) warps[warp].m = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) m = fmaxf(m, warps[w].m);
    rebase(s, m, c);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        s.z += __shfl_xor_sync(0xffffffffu, s.z, d);
        s.a += __shfl_xor_sync(0xffffffffu, s.a, d);
    }
    if (lane == 0) warps[warp].z = s.z, warps[warp].a = s.a;
    __syncthreads();
    s.z = s.a = 0.f;
#pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) s.z += warps[w].z, s.a += warps[w].a;
}

// Two values as floats; for sums where the maximum in use is far above it, -inf
// as a value so low that its probability is 0 all the same (0 times -inf would
// make the entropy's sum NaN), and all of a bf16 row below it alike. Seen::move
// says where that holds.
template <typename T>
__device__ __forceinline__ uint32_t lift(uint32_t u);
template <>
__device__ __forceinline__ uint32_t lift<__nv_bfloat16>(uint32_t u) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0xf680f680u));  // -2^110
    return r;
}
template <>
__device__ __forceinline__ uint32_t lift<__half>(uint32_t u) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0xfbfffbffu));  // -65504
    return r;
}
template <typename T>
__device__ __forceinline__ void two_values(uint32_t u, float& a, float& b) {
    if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
        a = f.x, b = f.y;
    } else {
        a = __uint_as_float(u << 16), b = __uint_as_float(u & 0xffff0000u);
    }
}

// What a thread has seen of its part of a row.
template <typename T>
struct Seen {
    static constexpr int V = 16 / sizeof(T);
    uint64_t z = 0, a = 0;  // pairs of sums
    float m = -3.402823466e38f, limit = -3.402823466e38f;  // the maximum in use, and when to move it
    // -m c rounded. Where `plain` the terms are x c + shift = t + rest(), one
    // operation a value, and sums() takes the rest out again; it is below 2^-5, for
    // |m c| is below 2^20 (beyond it, and where products with c overflow, the terms
    // are (x - m) c).
    float shift = 0.f;
    bool plain = false;
    float best = -__builtin_huge_valf(), second = -__builtin_huge_valf();
    int best_vec = -1;

    __device__ __forceinline__ float rest(float c) const { return plain ? __fmaf_rn(m, c, shift) : 0.f; }
    __device__ __forceinline__ void move(float to, float c) {
        float t = log2_term(m, to, c) - rest(c);
        m = to;
        limit = to + 8.f / c;
        shift = -to * c;
        // lifted values: their products with c finite, and their terms 0: of bf16,
        // below 2^20 less 2^110 c, of f16, below (30000 - 65504) c (c = 2^17: a
        // temperature of 1e-5, 2^-7: of 180)
        constexpr bool half = std::is_same<T, __half>::value;
        plain = fabsf(to) * c < 0x1p20f && fabsf(to) < (half ? 3e4f : 1e30f) &&
                (sizeof(T) == 4 || (c < 0x1p17f && c > (half ? 0x1p-7f : 0x1p-80f)));
        t += rest(c);
        const float f = pow2(t);
        const uint64_t f2 = pair(f, f), t2 = pair(t, t);
        a = fma2(fma2(z, t2, a), f2, 0);
        z = fma2(z, f2, 0);
    }
    __device__ __forceinline__ void term(float t0, float t1) {
        const uint64_t e = pair(pow2(t0), pow2(t1));
        z = add2(z, e);
        a = fma2(e, pair(t0, t1), a);
    }
    // N (1 or 2) vectors of 16 bytes, the first of them `vec`, the second a CTA's threads behind it
    template <int N>
    __device__ __forceinline__ void add(const uint4* raw, int vec, float c) {
        float x[N * V];
        const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
        for (int i = 0; i < N * 4; ++i) {
            if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
            else two_values<T>(w[i], x[2 * i], x[2 * i + 1]);
        }
        // NaN are passed over, so that a vector of nothing else counts as -inf
        float tops[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            tops[j] = -__builtin_huge_valf();
#pragma unroll
            for (int i = 0; i < V; i += 2) tops[j] = max3(tops[j], x[j * V + i], x[j * V + i + 1]);
        }
        const float top = N == 2 ? fmaxf(tops[0], tops[N - 1]) : tops[0], less = N == 2 ? fminf(tops[0], tops[N - 1]) : top;
        second = max3(second, fminf(best, top), N == 2 ? less : second);
        if (top > best || best_vec < 0) best = top, best_vec = N == 2 && tops[N - 1] > tops[0] ? vec + LP_THREADS : vec;
        if (top > limit) move(top, c);
        if (plain) {
            const uint64_t c2 = pair(c, c), shift2 = pair(shift, shift);
#pragma unroll
            for (int i = 0; i < N * V; i += 2) {
                float t0, t1;
                if constexpr (sizeof(T) == 4) {
                    unpair(fma2(pair(x[i], x[i + 1]), c2, shift2), t0, t1);
                    t0 = fmax_nan(t0, -200.f), t1 = fmax_nan(t1, -200.f);
                } else {
                    two_values<T>(lift<T>(w[i / 2]), t0, t1);
                    unpair(fma2(pair(t0, t1), c2, shift2), t0, t1);
                }
                term(t0, t1);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N * V; i += 2) term(log2_term(x[i], m, c), log2_term(x[i + 1], m, c));
        }
    }
    __device__ __forceinline__ Softmax sums(float c) const {
        float z0, z1, a0, a1;
        unpair(z, z0, z1);
        unpair(a, a0, a1);
        // from the terms' t + rest to t: 2^-rest by its series, whose error the small rest hides
        const float r = rest(c), y = r * -0.6931471805599453f;
        const float f = __fmaf_rn(y, __fmaf_rn(y, __fmaf_rn(y, 1.f / 6.f, 0.5f), 1.f), 1.f);
        return Softmax{m, (z0 + z1) * f, __fmaf_rn(z0 + z1, -r, a0 + a1) * f};
    }
};

// A vector whose values outside the row are -inf.
template <typename T>
__device__ __forceinline__ uint4 broken_run(const T* row, int v, int shift, int n) {
    constexpr int V = 16 / sizeof(T);
    Pack<T, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = v * V - shift + i;
        p.v[i] = from_f32<T>(e >= 0 && e < n ? to_f32(row[e]) : __int_as_float(0xff800000));
    }
    return *reinterpret_cast<const uint4*>(&p);
}

// V consecutive values as floats: vector `v` of the row, whose first value has
// index v * V - shift; values outside [0, n) are -inf.
template <typename T, int V>
__device__ __forceinline__ void load_run(float (&x)[V], const T* row, int v, int shift, int n) {
    const int first = v * V - shift;
    if (first >= 0 && first + V <= n) {
        const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(row + first);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_f32(p.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            x[i] = first + i >= 0 && first + i < n ? to_f32(row[first + i]) : __int_as_float(0xff800000);
    }
}

// A 16-byte load that leaves the L1 alone.
__device__ __forceinline__ uint4 load_stream(const uint4* p) {
    uint4 u;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
    return u;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 4) token_logprobs_kernel(const LogprobParams p) {
    constexpr int V = 16 / sizeof(T), UNROLL = 4;
    __shared__ uint64_t cand[LP_CAND];
    __shared__ uint64_t lists[LP_WARPS][32];
    __shared__ Softmax warp_soft[LP_WARPS];
    __shared__ int n_cand;
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row_i = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
    const T* row = static_cast<const T*>(p.logits) + (int64_t)row_i * p.row_stride;
    const int n = p.n_vocab;
    const float c = fminf(p.scale * 1.4426950408889634f, 3.402823466e38f);  // finite: 0 times c is 0
    // 16-byte vectors from the aligned address at or before the row
    const int shift = (int)((reinterpret_cast<uintptr_t>(row) % 16) / sizeof(T));
    const int n_vec = (n + shift + V - 1) / V;
    const int v0 = (int)((int64_t)n_vec * split / p.splits), v1 = (int)((int64_t)n_vec * (split + 1) / p.splits);

    // whole vectors [w0, w1) of the part, four a thread on the way while four
    // are worked on; a broken one at an end of the row first
    Seen<T> seen;
    const int w0 = v0 == 0 && shift ? 1 : v0, w1 = v1 == n_vec && (n + shift) % V ? max(v1 - 1, w0) : v1;
    {
        const int v = threadIdx.x == 0 && w0 > v0 ? v0 : threadIdx.x == 1 && w1 < v1 ? v1 - 1 : -1;
        if (v >= 0) {
            const uint4 x = broken_run(row, v, shift, n);
            seen.template add<1>(&x, v, c);
        }
    }
    {
        const uint4* vecs = reinterpret_cast<const uint4*>(row - shift);
        const int blocks = (w1 - w0) / (LP_THREADS * UNROLL);
        int v = w0 + (int)threadIdx.x;
        uint4 next[UNROLL];
        if (blocks > 0) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) next[u] = load_stream(vecs + v + u * LP_THREADS);
        }
        for (int b = 0; b < blocks; ++b, v += LP_THREADS * UNROLL) {
            uint4 now[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) now[u] = next[u];
            if (b + 1 < blocks) {
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) next[u] = load_stream(vecs + v + (UNROLL + u) * LP_THREADS);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; u += 2) seen.template add<2>(now + u, v + u * LP_THREADS, c);
        }
        // what is left is less than a block
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (v + u * LP_THREADS < w1) next[u] = load_stream(vecs + v + u * LP_THREADS);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (v + u * LP_THREADS < w1) seen.template add<1>(next + u, v + u * LP_THREADS, c);
    }
    const Softmax s_own = seen.sums(c);
    Softmax s = s_own;
    if (lane == 0 && warp == 0) n_cand = 0;
    const int k = p.k;
    if (k > 0) {
        // A key at most that of every thread's largest value (the vector's last
        // index), then the k-th largest of them: a bound that at least k values reach.
        uint64_t key = 0;
        if (seen.best_vec >= 0) {
            // NaN (they make z NaN) counted as -inf, but come behind it
            const bool nan = seen.best == -__builtin_huge_valf() && s_own.z != s_own.z;
            key = top_key(nan ? __int_as_float(0x7fffffff) : seen.best, (uint32_t)min(seen.best_vec * V - shift + V - 1, n - 1));
        }
        block_merge(warp_sort(key, lane), lists, warp, lane);
        const uint64_t floor_key = lists[0][k - 1];
        __syncthreads();
        const float none = __int_as_float(0xff800000);
        // a thread's NaN count as -inf in `best` and `second`, and so they do here
        const bool floor_is_value = floor_key >> 32 != 0;  // not NaN, and there is one
        const float floor_value = floor_is_value ? key_value(floor_key) : none;
        auto look_at = [&](int v) {
            float x[V];
            load_run<T, V>(x, row, v, shift, n);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = v * V - shift + i;
                if (e < 0 || e >= n) continue;
                const uint64_t o = top_key(x[i], (uint32_t)e);
                if (o >= floor_key) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < LP_CAND) cand[at] = o;
                }
            }
        };
        const bool reach = seen.best_vec >= 0 && seen.best >= floor_value, more = reach && seen.second >= floor_value;
        if (reach && !more) look_at(seen.best_vec);
        // The warp looks through the vectors of a thread whose others reach it
        // too: all, or, where they only equal it, those that begin before the
        // bound's index (a row that masks most tokens equals it everywhere).
        uint32_t todo = __ballot_sync(0xffffffffu, more);
        while (todo) {
            const int who = __ffs(todo) - 1;
            todo &= todo - 1;
            const int t = warp * 32 + who;
            int end = w1;
            if (!(__shfl_sync(0xffffffffu, seen.second, who) > floor_value) && floor_is_value)
                end = min(w1, ((int)key_index(floor_key) + shift) / V + 1);
            for (int v = w0 + t + lane * LP_THREADS; v < end; v += 32 * LP_THREADS) look_at(v);
            // a thread's largest value may lie behind
            if (lane == who && seen.best_vec >= end && seen.best_vec < w1) look_at(seen.best_vec);
            if (lane == 0 && t == 0 && w0 > v0) look_at(v0);
            if (lane == 0 && t == 1 && w1 < v1) look_at(v1 - 1);
        }
        __syncthreads();
        const int found = n_cand;
        uint64_t mine = 0;
        if (found <= LP_CAND) {
            if (found <= 32) {  // as a rule
                if (warp == 0) lists[0][lane] = warp_sort(lane < found ? cand[lane] : 0, lane);
                __syncthreads();
            } else {
                for (int b = warp * 32; b < found; b += LP_THREADS)
                    mine = warp_merge(mine, warp_sort(b + lane < found ? cand[b + lane] : 0, lane), lane);
                block_merge(mine, lists, warp, lane);
            }
        } else {
            // many values at or above the bound (a pattern of the row's order
            // that gives a few threads most of the largest values): one search
            // of the part for each of the k
            uint64_t below = ~0ull;
            for (int r = 0; r < k; ++r) {
                uint64_t top = 0;
                for (int v = v0 + (int)threadIdx.x; v < v1; v += LP_THREADS) {
                    float x[V];
                    load_run<T, V>(x, row, v, shift, n);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int e = v * V - shift + i;
                        const uint64_t o = e >= 0 && e < n ? top_key(x[i], (uint32_t)e) : 0;
                        if (o < below && o > top) top = o;
                    }
                }
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    const uint64_t o = shfl_xor64(top, d);
                    top = o > top ? o : top;
                }
                if (lane == 0) cand[warp] = top;
                __syncthreads();
                below = 0;
                for (int w = 0; w < LP_WARPS; ++w) below = cand[w] > below ? cand[w] : below;
                if (threadIdx.x == 0) lists[0][r] = below;
                __syncthreads();
            }
            if (threadIdx.x >= k && threadIdx.x < 32) lists[0][threadIdx.x] = 0;
        }
    }
    block_join(s, warp_soft, warp, lane, c);

    if (p.splits > 1) {
        LogprobPart* parts = reinterpret_cast<LogprobPart*>(p.partials) + (int64_t)row_i * p.splits;
        if (threadIdx.x == 0) parts[split].m = s.m, parts[split].z = s.z, parts[split].a = s.a;
        if (threadIdx.x < k) parts[split].top[threadIdx.x] = lists[0][threadIdx.x];
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(p.counters + row_i, 1u) == (uint32_t)p.splits - 1;
        __syncthreads();
        if (!last) return;
        __threadfence();
        if (threadIdx.x == 0) p.counters[row_i] = 0;  // as the next call expects it
        s = Softmax{-3.402823466e38f, 0.f, 0.f};
        for (int i = threadIdx.x; i < p.splits; i += LP_THREADS) {
            const LogprobPart* q = parts + i;
            s = join(s, Softmax{__ldcg(&q->m), __ldcg(&q->z), __ldcg(&q->a)}, c);
        }
        uint64_t mine = 0;
        if (k > 0) {
            const unsigned long long* q = reinterpret_cast<const unsigned long long*>(parts->top);
            constexpr int STEP = sizeof(LogprobPart) / 8;
            for (int i = warp; i < p.splits; i += LP_WARPS * 4) {
                uint64_t key[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    key[u] = i + u * LP_WARPS < p.splits && lane < k ? __ldcg(q + (int64_t)(i + u * LP_WARPS) * STEP + lane) : 0;
                mine = warp_merge(mine, warp_merge(warp_merge(key[0], key[1], lane), warp_merge(key[2], key[3], lane), lane), lane);
            }
            block_merge(mine, lists, warp, lane);
        }
        block_join(s, warp_soft, warp, lane, c);
    }
    // z = 0: nothing but -inf. NaN (or +inf) among the logits makes z NaN.
    const float ln_z = logf(s.z);
    if (threadIdx.x == 0 && p.entropy)
        p.entropy[row_i] = s.z == 0.f ? 0.f : ln_z - 0.6931471805599453f * s.a / s.z;
    const float none = __int_as_float(0xff800000);
    for (int g = threadIdx.x; g < p.n_given; g += LP_THREADS) {
        const int tok = p.tokens[(int64_t)row_i * p.n_given + g];
        float lp = 0.f;
        if (tok >= 0 && tok < n) lp = s.z == 0.f ? none : (to_f32(row[tok]) - s.m) * p.scale - ln_z;
        p.logprob[(int64_t)row_i * p.n_given + g] = lp;
    }
    if (threadIdx.x < k) {
        const uint64_t key = lists[0][threadIdx.x];
        p.top_ids[(int64_t)row_i * k + threadIdx.x] = (int32_t)key_index(key);
        p.top_lp[(int64_t)row_i * k + threadIdx.x] =
            s.z == 0.f ? none : (key_value(key) - s.m) * p.scale - ln_z;
    }
}

}  // namespace bh

extern "C" int bh_token_logprobs(bh_ctx* ctx, bh_workspace* ws, const void* logits, int type, int n_rows, int n_vocab,
                                 int64_t row_stride, float scale, const int32_t* tokens, int n_given, float* logprob,
                                 float* entropy_opt, int k, int32_t* top_ids, float* top_logprob, void* stream) {
    using bh::is_aligned;
    if (!ctx || !ws || ws->device != ctx->device || !bh::is_type(type)) return BH_EINVAL;
    if (n_rows < 0 || n_vocab < 1 || n_vocab > 1 << 30 || n_given < 0 || k < 0 || k > BH_MAX_TOP || k > n_vocab)
        return BH_EINVAL;
    if (n_rows > 1 && row_stride < n_vocab) return BH_EINVAL;
    if (!(scale > 0.f) || scale > 3.402823466e38f) return BH_EINVAL;
    if (n_rows == 0) return BH_OK;
    if (!logits || !is_aligned(logits, bh::type_bytes(type))) return BH_EINVAL;
    if ((n_given > 0 && (!tokens || !logprob)) || (k > 0 && (!top_ids || !top_logprob))) return BH_EINVAL;
    for (const void* q : {(const void*)tokens, (const void*)logprob, (const void*)entropy_opt, (const void*)top_ids,
                          (const void*)top_logprob})
        if (!is_aligned(q, 4)) return BH_EINVAL;
    bh::CallDevice dev(ctx->device);
    if (!dev.ok) return BH_ENODEV;
    // Rows are split until the machine is full (four CTAs an SM), parts of at
    // least four vectors a thread: the number that makes the waves of CTAs, each
    // as long as its bytes and an end worth about 96 KB of them, the shortest
    // (2048 rows of 304 KB: 122 us unsplit, 157 in halves; 8 rows of 608 KB: 10.7
    // us in 37 parts, 12.8 in 74, 15.7 unsplit).
    const int64_t bytes = (int64_t)n_vocab * bh::type_bytes(type), room = (int64_t)ctx->num_sms * 4;
    const int64_t most = bytes / 16 / (bh::LP_THREADS * 4);
    int64_t splits = 1, least = INT64_MAX;
    for (int64_t s = 1; s <= most && s <= room / n_rows + 4; ++s) {
        const int64_t cost = (n_rows * s + room - 1) / room * (bytes / s + (96 << 10));
        if (cost < least) least = cost, splits = s;
    }
    if (n_rows > bh::WS_COUNTERS) splits = 1;
    while (splits > 1 && (size_t)n_rows * splits * sizeof(bh::LogprobPart) > ws->bytes) --splits;
    if (splits < 1) splits = 1;
    if ((int64_t)n_rows * splits > INT_MAX) return BH_EINVAL;
    bh::LogprobParams p{logits,     tokens, logprob, entropy_opt, top_logprob, top_ids, ws->counters, ws->partials,
                        row_stride, scale,  n_rows,  n_vocab,     n_given,     k,       (int)splits};
    const unsigned grid = (unsigned)(n_rows * splits);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == BH_F32) bh::token_logprobs_kernel<float><<<grid, bh::LP_THREADS, 0, s>>>(p);
    else if (type == BH_F16) bh::token_logprobs_kernel<__half><<<grid, bh::LP_THREADS, 0, s>>>(p);
    else bh::token_logprobs_kernel<__nv_bfloat16><<<grid, bh::LP_THREADS, 0, s>>>(p);
    return bh::launch_result();
}
