// qk_norm_rope.cu — per-head RMSNorm of q and k, their rotation, and the append
// of k and v to the paged cache, in one pass over the projected q|k|v rows
// (bh_qk_norm_rope_append).
//
// y = x * rsqrt(mean(x^2) + eps) * w; pairs (a, b) of the first rot values turn
// into (a cos - b sin, a sin + b cos); everything in fp32, rounded once to the
// type it is stored in. Every value is read and written once: HBM bound at
// prompt sizes, latency bound at one token.
//
// A group of lanes owns one head, a lane the two runs of V consecutive values
// whose elements are each other's rotation partners (NeoX: i and i + rot / 2;
// interleaved partners lie within a run), so loads and stores are 16 bytes, the
// rotation needs no exchange and the norm is one reduction over the group. A
// warp works the heads of a token, its (cos, sin) row in registers, with the
// runs of AHEAD groups of them on the way at once.
//
// Measured in a graph, 32 + 8 + 8 heads of 128 values: one token 3.1 us (launch
// and two dependent loads); 509 tokens of fp32 into an f16 cache 6.5 us, 3.5
// TB/s from the L2; 16384 of bf16 88 us, 4.65 TB/s, where warps wait for loads
// with the issue slots 43% busy: 64 bytes a lane are in flight (fp32 throughout,
// with 128 bytes a lane, 5.9 TB/s).
#include "paged_kv.cuh"

namespace bh {

struct RopeParams {
    const void* x;
    void* q_out;
    KvView kv;
    const float *q_norm, *k_norm, *rope;
    const int32_t* pos;
    const int64_t* slot;
    int* status;
    int64_t row_stride, q_stride;
    float eps;
    int n_tok, n_head, n_kv, dim, n_pos, rot, neox;
    int slices;  // warps that share a token's heads
    Divisor block;
};

constexpr int ROPE_THREADS = 128, ROPE_CTAS = 4;  // CTAs of an SM

// V consecutive floats as pairs; 16-byte aligned, V a multiple of 4.
template <int V>
__device__ __forceinline__ void load_pairs(uint64_t (&x)[V / 2], const float* p) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(p + i);
        x[i / 2] = pair(f.x, f.y), x[i / 2 + 1] = pair(f.z, f.w);
    }
}
// A run as pairs of floats, and back.
template <typename T, int V>
__device__ __forceinline__ void to_pairs(uint64_t (&x)[V / 2], const Pack<T, V>& p) {
#pragma unroll
    for (int i = 0; i < V; i += 2) x[i / 2] = pair(to_f32(p.v[i]), to_f32(p.v[i + 1]));
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> from_pairs(const uint64_t (&x)[V / 2]) {
    Pack<T, V> p;
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        float a, b;
        unpair(x[i / 2], a, b);
        if constexpr (std::is_same<T, float>::value) {
            p.v[i] = a, p.v[i + 1] = b;
        } else if constexpr (std::is_same<T, __half>::value) {
            *reinterpret_cast<__half2*>(&p.v[i]) = __floats2half2_rn(a, b);
        } else {
            *reinterpret_cast<__nv_bfloat162*>(&p.v[i]) = __floats2bfloat162_rn(a, b);
        }
    }
    return p;
}

// T: activations, C: cache, V: values of a run, L: lanes of a head.
template <typename T, typename C, int V, int L>
__global__ void __launch_bounds__(ROPE_THREADS, ROPE_CTAS) qk_norm_rope_kernel(const RopeParams p) {
    constexpr int HEADS = 32 / L, N = V / 2;  // heads of a warp at a time, pairs of a run
    constexpr int AHEAD = V == 8 ? 2 : 4;  // head groups on the way
    const int lane = threadIdx.x & 31, li = lane % L, hg = lane / L;
    // the lane's runs: pair li of the rotated part, else of the rest
    const int rot_pairs = p.rot / 2 / V, rest = (p.dim - p.rot) / V, rest_pairs = (rest + 1) / 2;
    int e0 = -1, e1 = -1;  // first elements
    const bool turned = li < rot_pairs;
    if (turned) {
        e0 = p.neox ? li * V : 2 * li * V;
        e1 = p.neox ? li * V + p.rot / 2 : 2 * li * V + V;
    } else if (li - rot_pairs < rest_pairs) {
        const int i = li - rot_pairs;
        e0 = p.rot + i * V;
        if (i + rest_pairs < rest) e1 = p.rot + (i + rest_pairs) * V;
    }
    const uint64_t one = pair(1.f, 1.f);
    uint64_t w0[N], w1[N];  // q's weights; k's come from the L1 at each use
#pragma unroll
    for (int i = 0; i < N; ++i) w0[i] = w1[i] = one;
    if (p.q_norm && e0 >= 0) load_pairs<V>(w0, p.q_norm + e0);
    if (p.q_norm && e1 >= 0) load_pairs<V>(w1, p.q_norm + e1);
    const int q_groups = (p.n_head + HEADS - 1) / HEADS, kv_groups = (p.n_kv + HEADS - 1) / HEADS;
    const int groups = q_groups + 2 * kv_groups;
    const float per_dim = 1.f / (float)p.dim;
    const int64_t units = (int64_t)p.n_tok * p.slices, step = (int64_t)gridDim.x * (ROPE_THREADS / 32);
    for (int64_t unit = (int64_t)blockIdx.x * (ROPE_THREADS / 32) + (threadIdx.x >> 5); unit < units; unit += step) {
        const int t = p.slices == 1 ? (int)unit : (int)(unit / p.slices), slice = (int)(unit - (int64_t)t * p.slices);
        const T* x = static_cast<const T*>(p.x) + (int64_t)t * p.row_stride;
        const int pos = p.pos[t];
        int64_t slot = p.slot[t], page = 0;
        bool live = pos >= 0;
        if (live && ((p.rot && pos >= p.n_pos) || slot >= (int64_t)p.kv.n_blocks * p.kv.block_size)) {
            if (lane == 0) set_status(p.status, ST_BADARG);
            live = false;
        }
        if (!live) slot = -1;
        if (slot >= 0) {
            const uint32_t b = p.block.div((uint32_t)slot), o = (uint32_t)slot - b * p.block.d;
            page = (int64_t)b * p.kv.block_stride + (int64_t)o * p.kv.token_stride;
        }
        uint64_t cs[N], sn[N];  // cos and sin of the lane's V pairs
#pragma unroll
        for (int i = 0; i < N; ++i) cs[i] = one, sn[i] = 0;
        if (live && turned) {
            const float4* row = reinterpret_cast<const float4*>(p.rope + ((int64_t)pos * (p.rot / 2) + li * V) * 2);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float4 f = row[i];
                cs[i] = pair(f.x, f.z), sn[i] = pair(f.y, f.w);
            }
        }
        // the slice's head groups, AHEAD of them on the way; a group is q, k or v as a whole
        for (int g0 = slice; g0 < groups; g0 += p.slices * AHEAD) {
            Pack<T, V> a[AHEAD], b[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int g = g0 + u * p.slices, kind = g < q_groups ? 0 : g < q_groups + kv_groups ? 1 : 2;
                const int h = (kind == 0 ? g : g - q_groups - (kind - 1) * kv_groups) * HEADS + hg;
                const T* src = x + (int64_t)((kind == 0 ? 0 : p.n_head + (kind - 1) * p.n_kv) + h) * p.dim;
                const bool in = g < groups && h < (kind == 0 ? p.n_head : p.n_kv);
                if (in && e0 >= 0) a[u] = *reinterpret_cast<const Pack<T, V>*>(src + e0);
                if (in && e1 >= 0) b[u] = *reinterpret_cast<const Pack<T, V>*>(src + e1);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int g = g0 + u * p.slices, kind = g < q_groups ? 0 : g < q_groups + kv_groups ? 1 : 2;
                if (g >= groups) break;
                const int h = (kind == 0 ? g : g - q_groups - (kind - 1) * kv_groups) * HEADS + hg;
                const bool mine = h < (kind == 0 ? p.n_head : p.n_kv);
                uint64_t y0[N], y1[N];
                to_pairs<T, V>(y0, a[u]);
                to_pairs<T, V>(y1, b[u]);
                if (kind < 2) {
                    const float* norm = kind == 0 ? p.q_norm : p.k_norm;
                    if (norm) {
                        uint64_t s0 = 0, s1 = 0;
#pragma unroll
                        for (int i = 0; i < N; ++i) s0 = fma2(y0[i], y0[i], s0), s1 = fma2(y1[i], y1[i], s1);
                        float f0, f1, f2, f3;
                        unpair(s0, f0, f1);
                        unpair(s1, f2, f3);
                        float ss = (mine && e0 >= 0 ? f0 + f1 : 0.f) + (mine && e1 >= 0 ? f2 + f3 : 0.f);
#pragma unroll
                        for (int d = 1; d < L; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                        const float r = rsqrtf(ss * per_dim + p.eps);
                        const uint64_t r2 = pair(r, r);
#pragma unroll
                        for (int i = 0; i < N; ++i) y0[i] = mul2(y0[i], r2), y1[i] = mul2(y1[i], r2);
                        if (kind == 0) {
#pragma unroll
                            for (int i = 0; i < N; ++i) y0[i] = mul2(y0[i], w0[i]), y1[i] = mul2(y1[i], w1[i]);
                        } else {
                            uint64_t k0[N], k1[N];
                            load_pairs<V>(k0, norm + max(e0, 0));
                            load_pairs<V>(k1, norm + max(e1, 0));
#pragma unroll
                            for (int i = 0; i < N; ++i) y0[i] = mul2(y0[i], k0[i]), y1[i] = mul2(y1[i], k1[i]);
                        }
                    }
                    if (turned) {
                        if (p.neox) {
#pragma unroll
                            for (int i = 0; i < N; ++i) {
                                const uint64_t u0 = y0[i], u1 = y1[i];
                                y0[i] = sub2(mul2(u0, cs[i]), mul2(u1, sn[i]));
                                y1[i] = fma2(u0, sn[i], mul2(u1, cs[i]));
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < V; ++i) {  // the runs' 2 V consecutive values are V pairs
                                uint64_t& y = i < N ? y0[i] : y1[i - N];
                                float u0, u1, c0, c1, s0, s1;
                                unpair(y, u0, u1);
                                unpair(cs[i / 2], c0, c1);
                                unpair(sn[i / 2], s0, s1);
                                const float c = i & 1 ? c1 : c0, s = i & 1 ? s1 : s0;
                                y = pair(__fmaf_rn(u0, c, -(u1 * s)), __fmaf_rn(u0, s, u1 * c));
                            }
                        }
                    }
                }
                if (!mine) continue;
                if (kind == 0) {
                    if (!live) {
#pragma unroll
                        for (int i = 0; i < N; ++i) y0[i] = y1[i] = 0;
                    }
                    T* dst = static_cast<T*>(p.q_out) + (int64_t)t * p.q_stride + h * p.dim;
                    if (e0 >= 0) *reinterpret_cast<Pack<T, V>*>(dst + e0) = from_pairs<T, V>(y0);
                    if (e1 >= 0) *reinterpret_cast<Pack<T, V>*>(dst + e1) = from_pairs<T, V>(y1);
                } else if (slot >= 0) {
                    C* dst = static_cast<C*>(kind == 1 ? p.kv.k : p.kv.v) + page + (int64_t)h * p.kv.head_stride;
                    if (e0 >= 0) *reinterpret_cast<Pack<C, V>*>(dst + e0) = from_pairs<C, V>(y0);
                    if (e1 >= 0) *reinterpret_cast<Pack<C, V>*>(dst + e1) = from_pairs<C, V>(y1);
                }
            }
        }
    }
}

template <typename T, typename C, int V, int L>
static int launch_rope(RopeParams& p, int num_sms, cudaStream_t s) {
    // One wave of warps: each works the heads of several tokens, or, of few
    // tokens, a share of a token's head groups (one token 3.1 us, by one warp 11.7;
    // 509 tokens 6.5 and 12.0).
    const int groups = (p.n_head + 32 / L - 1) / (32 / L) + 2 * ((p.n_kv + 32 / L - 1) / (32 / L));
    const int64_t most = (int64_t)num_sms * ROPE_CTAS, fit = most * (ROPE_THREADS / 32) / p.n_tok;
    p.slices = (int)(fit < 1 ? 1 : fit < groups ? fit : groups);
    const int64_t warps = (int64_t)p.n_tok * p.slices, ctas = (warps + ROPE_THREADS / 32 - 1) / (ROPE_THREADS / 32);
    qk_norm_rope_kernel<T, C, V, L><<<(unsigned)(ctas < most ? ctas : most), ROPE_THREADS, 0, s>>>(p);
    return launch_result();
}

template <typename T, typename C, int V>
static int launch_rope_lanes(RopeParams& p, int num_sms, cudaStream_t s) {
    // rotated pairs of runs, then those of the rest
    const int lanes = p.rot / 2 / V + ((p.dim - p.rot) / V + 1) / 2;
    if (lanes <= 4) return launch_rope<T, C, V, 4>(p, num_sms, s);
    if (lanes <= 8) return launch_rope<T, C, V, 8>(p, num_sms, s);
    if (lanes <= 16) return launch_rope<T, C, V, 16>(p, num_sms, s);
    return launch_rope<T, C, V, 32>(p, num_sms, s);
}

template <typename T, typename C>
static int launch_rope_types(RopeParams& p, int num_sms, cudaStream_t s) {
    // 16-byte runs of the activations; 8-byte ones of 16-bit types when half
    // of the rotated part is not a whole number of 8-value runs (16384 tokens of
    // bf16: 88 us, with 8-byte runs 140)
    if (sizeof(T) == 2 && p.rot % 16 == 0) return launch_rope_lanes<T, C, 8>(p, num_sms, s);
    return launch_rope_lanes<T, C, 4>(p, num_sms, s);
}

}  // namespace bh

extern "C" int bh_qk_norm_rope_append(bh_ctx* ctx, const void* qkv, int act_type, int n_tok, int64_t row_stride,
                                      int n_head, const bh_paged_kv* kv, const float* q_norm, const float* k_norm,
                                      float eps, const float* rope, int n_pos, int rot_dim, int neox,
                                      const int32_t* tok_pos, const int64_t* tok_slot, void* q_out, int64_t q_stride,
                                      void* stream) {
    using bh::is_aligned;
    if (!ctx || !bh::kv_valid(kv) || !bh::is_type(act_type) || n_tok < 0 || n_head < 1) return BH_EINVAL;
    if (act_type != kv->dtype && act_type != BH_F32) return BH_EINVAL;
    if (n_head > 1 << 16 || kv->n_head_kv > 1 << 16) return BH_EINVAL;
    if (rot_dim < 0 || rot_dim > kv->head_dim || rot_dim % 8 || !(eps >= 0.f)) return BH_EINVAL;
    if (rot_dim && (!rope || n_pos < 1)) return BH_EINVAL;
    const int64_t per = 16 / bh::type_bytes(act_type);
    const int64_t row = (int64_t)(n_head + 2 * kv->n_head_kv) * kv->head_dim;
    if (row_stride % per || q_stride % per) return BH_EINVAL;
    if (n_tok > 1 && (row_stride < row || q_stride < (int64_t)n_head * kv->head_dim)) return BH_EINVAL;
    if (n_tok == 0) return BH_OK;
    if (!qkv || !q_out || !tok_pos || !tok_slot) return BH_EINVAL;
    if (!is_aligned(qkv, 16) || !is_aligned(q_out, 16) || !is_aligned(rope, 16) || !is_aligned(q_norm, 16) ||
        !is_aligned(k_norm, 16) || !is_aligned(tok_pos, 4) || !is_aligned(tok_slot, 8))
        return BH_EINVAL;
    bh::CallDevice dev(ctx->device);
    if (!dev.ok) return BH_ENODEV;
    bh::RopeParams p{qkv,        q_out,    bh::kv_view(kv), q_norm,        k_norm,       rope,  tok_pos, tok_slot, ctx->d_status,
                     row_stride, q_stride, eps,             n_tok,         n_head,       kv->n_head_kv, kv->head_dim,
                     n_pos,      rot_dim,  neox != 0,       1,             bh::Divisor(kv->block_size)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (act_type == BH_F16) return bh::launch_rope_types<__half, __half>(p, ctx->num_sms, s);
    if (act_type == BH_BF16) return bh::launch_rope_types<__nv_bfloat16, __nv_bfloat16>(p, ctx->num_sms, s);
    if (kv->dtype == BH_F16) return bh::launch_rope_types<float, __half>(p, ctx->num_sms, s);
    if (kv->dtype == BH_BF16) return bh::launch_rope_types<float, __nv_bfloat16>(p, ctx->num_sms, s);
    return bh::launch_rope_types<float, float>(p, ctx->num_sms, s);
}
