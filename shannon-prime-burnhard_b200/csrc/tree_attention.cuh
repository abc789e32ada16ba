// tree_attention.cuh — the kernel of bh_tree_attention, instantiated for one
// pair of types in each tree_attention_*.cu.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(x_j - m), x_j = scale log2(e) q.k_j
// and m the running maximum: one pass over the positions, the sums rescaled
// when m grows.
//
// Rows. The query rows of a KV head are its sequence's new tokens times the
// heads of its group; MT of them form a row tile, so that K and V are read once
// for all of them and the products run on the tensor cores (mma.sync
// m16n8k16). What bounds it is the read of the cache: 16 rows do 16 flops a
// byte, the tensor cores pay from about 100 on. Measured in a graph, 32 heads
// over 8 of 128 values: 48 sequences up to 8192 long, fp32 over f16, 152 us, 5.4
// TB/s; f16 throughout 139 us, 5.9 TB/s; one token over 127 positions of fp32 16
// us, all of it latency (launch, three dependent loads, the join).
//
// Work. Positions come in tiles of TN. All tiles of all (sequence, row tile, KV
// head) form one line, of which every CTA takes an equal, contiguous part
// (ragged lengths need no plan on the host). A row tile that lies in several
// CTAs is joined from their parts, in order, by a second small kernel, launched
// programmatically, that finds them in a record which every CTA leaves. (The
// last CTA of a row tile to arrive did this before: its loads took 4 us each,
// queued behind the other CTAs' tiles.)
//
// A CTA is one warp that copies and RG x KG that compute. The copying warp
// fetches the tiles' rows at the block table's addresses by 16-byte cp.async
// into a ring of STAGES tiles (rows of 256 bytes by cp.async.bulk measured 2.5
// TB/s for the whole GPU, one such copy about every 30 cycles an SM; one warp's
// cp.async, two CTAs an SM, 6.4). 16-byte chunks are permuted by row so that
// ldmatrix (16-bit caches) or 16-byte loads (fp32) meet no bank conflict. The
// computing warps are RG groups of rows times KG groups of a tile's positions;
// position groups keep sums of their own until the row tile ends.
//
// Precision. m and the sums are fp32. 16-bit activations over their own type:
// the probabilities are rounded to that type for the product with V (its error
// is the output type's own). fp32 activations: q and the probabilities are
// split into NS parts of the cache's type (f16: 2 x 11 bits of values scaled
// into f16's range, bf16: 3 x 8 bits), or, with K and V as well, into two TF32
// parts of which three products are kept (22 bits). The tensor core's own
// accumulation rounds toward zero, so there the small parts have accumulators
// of their own and a tile's products with V are added to the sums in fp32.
#pragma once

#include <atomic>

#include "paged_kv.cuh"

namespace bh {

struct AttnParams {
    const void* q;
    void* out;
    float* lse;
    KvView kv;
    const int32_t *tables, *ctx_lens, *q_start;
    const int64_t* mask;
    float* partials;
    int* status;
    int64_t q_stride, out_stride;
    float scale;
    int n_tok, n_head, n_kv, dim, max_blocks, n_seq, max_new, num_sms;
    Divisor group, block;  // query heads of a KV head, tokens of a block
};

constexpr int TA_MIN_TILES = 2;  // a CTA's least share of the line

template <int TA_, int TC_, int DP_, int RG_, int KG_>
struct AttnShape {
    static constexpr int TA = TA_, TC = TC_, DP = DP_, RG = RG_, KG = KG_;
    using T = typename ValueOf<TA>::type;
    using C = typename ValueOf<TC>::type;
    static constexpr bool F = TC == BH_F32;
    static constexpr int MT = 16 * RG, WARPS = RG * KG, COMPUTE = WARPS * 32, THREADS = COMPUTE + 32;
    static constexpr int NS = F ? 1 : TA == TC ? 1 : TC == BH_F16 ? 2 : 3;  // parts of q kept in shared memory
    static constexpr bool EXACT = TA == BH_F32;
    // exponent added to probabilities that f16 holds, which would lose those below
    // 2^-25 of the largest: a long row has much of its sum there
    static constexpr float OFF = TC == BH_F16 ? 12.f : 0.f;
    static constexpr int NT = DP / 8;  // accumulator tiles of 8 values
    static constexpr int ROW = DP * (int)sizeof(C);
    // 16 positions a warp (8 of fp32), more of short rows: 32 KB of K and V in a stage (64 KB for 256 values)
    static constexpr int TN = KG * (DP == 64 ? 32 : 16) / (F ? 2 : 1);
    static constexpr int WN = TN / KG;
    static constexpr int TILE = TN * ROW;
    // the query rows, and in their place the sums when the row tile ends
    static constexpr int Q_BYTES = NS * MT * ROW, EPI_BYTES = MT * DP * 4;
    static constexpr int SHARED_Q = Q_BYTES > EPI_BYTES ? Q_BYTES : EPI_BYTES;
    // CTAs an SM: three of two stages where 128 registers do, else two (three stages if they fit) or one
    static constexpr int MORE = 2048 + 64 * MT;  // static shared memory and the system's
    static constexpr int room(int stages) { return 228 * 1024 / (stages * 2 * TILE + SHARED_Q + MORE); }
    static constexpr int CTAS = THREADS > 160 ? 1 : NT <= 16 && room(2) >= 3 ? 3 : room(2) >= 2 ? 2 : 1;
    static constexpr int STAGES = room(3) >= CTAS ? 3 : 2;
    static constexpr size_t BYTES = (size_t)STAGES * 2 * TILE + SHARED_Q;
    static constexpr int SLOT = MT * (DP + 4);  // floats of a partial result
    // lengths on the line: of a tile, and of a row tile's begin and end, which cost about two tiles
    static constexpr int BEGIN = 2;
    __device__ static __forceinline__ int weight(int) { return 1; }
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// c += a b on 16 x 8 x 16 values of type C (f16 or bf16)
template <typename C>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<C, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c += a b on 16 x 8 x 8 TF32 values
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same products alone (c = a b)
template <typename C>
__device__ __forceinline__ void mma16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<C, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_tf32_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// the leading 11 bits of a value and the rest (exact; the tensor core reads its leading 11)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
template <typename C>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<C, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <typename C>
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b) {
    if constexpr (std::is_same<C, __half>::value) {
        const __half2 h = *reinterpret_cast<const __half2*>(&u);
        a = __low2float(h), b = __high2float(h);
    } else {
        a = __uint_as_float(u << 16), b = __uint_as_float(u & 0xffff0000u);
    }
}

// byte offsets of a 16-byte chunk in a tile's row
template <class S>
__device__ __forceinline__ int k_chunk(int row, int c) {
    return row * S::ROW + ((S::F ? c ^ ((row & 1) << 2) : c ^ (row & 7)) << 4);
}
template <class S>
__device__ __forceinline__ int v_chunk(int row, int c) {
    return row * S::ROW + ((S::F ? c ^ (((row >> 1) & 3) << 1) : c ^ (row & 7)) << 4);
}

// One sequence's part of the line: for each row tile and head its begin, then
// its tiles, `weight` each. A tile is the CTA's whose share holds its first place.
struct SeqWork {
    int ctx, start, n_new, tiles, row_tiles, weight;
};
template <class S>
__device__ __forceinline__ SeqWork seq_work(const AttnParams& p, int s) {
    SeqWork w;
    w.ctx = max(p.ctx_lens[s], 0);
    w.start = p.q_start[s];
    w.n_new = p.q_start[s + 1] - w.start;
    if (w.n_new > 0 && (w.n_new > p.max_new || w.start < 0 || w.start > p.n_tok - w.n_new ||
                        w.ctx > INT_MAX - 1024 || (int64_t)w.ctx + w.n_new > (int64_t)p.max_blocks * p.kv.block_size)) {
        set_status(p.status, ST_BADARG);
        w.n_new = 0;
    }
    if (w.n_new <= 0) {
        w.n_new = w.tiles = w.row_tiles = w.weight = 0;
        return w;
    }
    w.tiles = (int)(((uint32_t)w.ctx + (uint32_t)w.n_new + S::TN - 1) / S::TN);
    w.row_tiles = (w.n_new * (int)p.group.d + S::MT - 1) / S::MT;
    w.weight = S::weight(w.n_new * (int)p.group.d);
    return w;
}

// A place on the line.
struct Cursor {
    SeqWork w;
    int seq, row_tile, head, tile;
    int64_t first;  // the place of the row tile's first tile
    __device__ __forceinline__ int64_t place() const { return first + (int64_t)tile * w.weight; }
    __device__ __forceinline__ int64_t last() const { return first + (int64_t)(w.tiles - 1) * w.weight; }
};
template <class S>
__device__ __forceinline__ void next_tile(Cursor& c, const AttnParams& p) {
    if (++c.tile < c.w.tiles) return;
    c.tile = 0;
    c.first += (int64_t)c.w.tiles * c.w.weight + S::BEGIN;
    if (++c.head < p.n_kv) return;
    c.head = 0;
    if (++c.row_tile < c.w.row_tiles) return;
    c.row_tile = 0;
    do {
        if (++c.seq >= p.n_seq) return;
        c.w = seq_work<S>(p, c.seq);
    } while (c.w.tiles == 0);
}

// The place of the tile after `c`.
template <class S>
__device__ __forceinline__ int64_t next_place(const Cursor& c) {
    return c.place() + c.w.weight + (c.tile + 1 < c.w.tiles ? 0 : S::BEGIN);
}

// Sum over the CTA of one value a thread, and the sum of the threads before.
template <int WARPS>
__device__ __forceinline__ int64_t cta_scan(int64_t v, int64_t* warp_sums, int64_t& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int64_t inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, (long long)inc, d);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 31) warp_sums[w] = inc;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        if (i < w) before += warp_sums[i];
        total += warp_sums[i];
    }
    return before + inc - v;
}

template <class S>
struct AttnShared {
    uint64_t full[S::STAGES], empty[S::STAGES];
    uint32_t valid[S::STAGES][(S::TN + 31) / 32];  // rows of the tile that exist
    int whole[S::STAGES];                          // all of them, and none a draft
    uint32_t bad[(S::TN + 31) / 32];               // drafts of the tile whose V is not finite
    uint64_t mask[S::MT];
    float row_scale[S::MT];
    float part_m[S::KG][S::MT], part_l[S::KG][S::MT];
    float row_m[S::MT], row_l[S::MT];
    int64_t scan[S::WARPS + 1];
    Cursor first;
    int sees_all[S::WARPS];
    int given_up;
};

// The CTA's part [f0, f1) of the line cut into equal shares, and, in `sh`, the
// row tile and tile that it begins with.
template <class S, class Shared>
__device__ __forceinline__ void find_part(const AttnParams& p, Shared& sh, int64_t& per, int64_t& f0, int64_t& f1) {
    constexpr int THREADS = S::THREADS;
    const int tid = threadIdx.x;
    int64_t total = 0, at = 0, mine = 0;
    SeqWork w;
    for (int base = 0; base < p.n_seq; base += THREADS) {
        int64_t sum;
        mine = 0;
        if (base + tid < p.n_seq) {
            w = seq_work<S>(p, base + tid);
            if (w.tiles) mine = ((int64_t)w.tiles * w.weight + S::BEGIN) * w.row_tiles * p.n_kv;
        }
        at = total + cta_scan<THREADS / 32>(mine, sh.scan, sum);
        total += sum;
    }
    per = (total + gridDim.x - 1) / gridDim.x;
    const int least = S::BEGIN + TA_MIN_TILES * S::weight(p.max_new * (int)p.group.d);
    if (per < least) per = least;
    f0 = per * blockIdx.x;
    f1 = f0 + per < total ? f0 + per : total;
    if (f0 >= total) return;
    int64_t before = 0;
    for (int base = 0; base < p.n_seq; base += THREADS) {
        if (p.n_seq > THREADS) {  // more sequences than the first scan left in registers
            int64_t sum;
            mine = 0;
            if (base + tid < p.n_seq) {
                w = seq_work<S>(p, base + tid);
                if (w.tiles) mine = ((int64_t)w.tiles * w.weight + S::BEGIN) * w.row_tiles * p.n_kv;
            }
            at = before + cta_scan<THREADS / 32>(mine, sh.scan, sum);
            before += sum;
        }
        if (mine && at <= f0 && f0 < at + mine) {
            const int64_t in = f0 - at, length = (int64_t)w.tiles * w.weight + S::BEGIN;
            const int item = (int)(in / length);
            const int64_t inside = in - item * length - S::BEGIN;
            // at the begin, the tile that starts there or the next one (which may be the next row tile's first)
            Cursor c{w, base + tid, item / p.n_kv, item % p.n_kv, 0, f0 - inside};
            if (inside > 0) {
                c.tile = (int)((inside + w.weight - 1) / w.weight);
                if (c.tile == w.tiles) {
                    --c.tile;
                    next_tile<S>(c, p);
                }
            }
            sh.first = c;
        }
        if (before > f0) break;
    }
}

// A part's place among the partial results: maxima, sums and score scales of
// its rows, then its values, four of every row next to each other. A CTA has
// two: of a row tile that began before it, and of one that ends after it.
template <class S>
__device__ __forceinline__ float* part_slot(const AttnParams& p, int cta, bool begins) {
    return p.partials + ((int64_t)cta * 2 + begins) * S::SLOT;
}
template <class S>
__device__ __forceinline__ int part_value(int row, int d) {
    return 4 * S::MT + (d / 4 * S::MT + row) * 4;
}
// A row tile's row in q, out and lse: token and head.
template <class S>
__device__ __forceinline__ void row_of(const AttnParams& p, const Cursor& c, int r, int& tok, int& head) {
    const uint32_t row = c.row_tile * S::MT + r, i = p.group.div(row);
    tok = c.w.start + (int)i;
    head = c.head * (int)p.group.d + (int)(row - i * p.group.d);
}
// ln of a row's sum: m in units of the scores, rs log2 of e a unit
__device__ __forceinline__ float log_sum(float m, float rs, float off, float sum) {
    return sum == 0.f ? __int_as_float(0xff800000)
                      : (float)(((double)m * rs - off) * 0.6931471805599453 + (double)logf(sum));
}

// What a CTA leaves about the row tile that it began and others end.
struct Split {
    int rows, last_cta;  // rows 0: there is none
    int row_tile, head, start;
};
template <class S>
__device__ __forceinline__ Split* split_of(const AttnParams& p, int cta) {
    return reinterpret_cast<Split*>(p.partials + (int64_t)S::CTAS * p.num_sms * 2 * S::SLOT) + cta;
}
template <class S>
__device__ __forceinline__ void leave_split(const AttnParams& p, const Cursor& c, bool is_split, int64_t per) {
    Split x{0, 0, c.row_tile, c.head, c.w.start};
    if (is_split) {
        x.rows = min(S::MT, c.w.n_new * (int)p.group.d - c.row_tile * S::MT);
        x.last_cta = (int)(c.last() / per);
    }
    *split_of<S>(p, blockIdx.x) = x;
}

// Joins the row tile that CTA blockIdx.x of the attention began and others ended.
constexpr int JOIN_THREADS = 256;
template <class S>
__global__ void __launch_bounds__(JOIN_THREADS, 4) tree_attention_join_kernel(const AttnParams p) {
    using T = typename S::T;
    __shared__ float tops[S::MT], invs[S::MT], scales[S::MT];
    pdl_wait();
    const Split x = *split_of<S>(p, blockIdx.x);
    if (x.rows == 0) return;
    const int c0 = blockIdx.x, c1 = x.last_cta, rows = x.rows;
    Cursor cur;
    cur.row_tile = x.row_tile, cur.head = x.head, cur.w.start = x.start;
    // the rows' maxima and sums, in one pass over the parts
    for (int r = threadIdx.x; r < rows; r += JOIN_THREADS) {
        const float rs = __ldcg(part_slot<S>(p, c0, true) + 2 * S::MT + r);
        float top = __int_as_float(0xff800000), sum = 0.f;
#pragma unroll 8
        for (int c = c0; c <= c1; ++c) {
            const float* q = part_slot<S>(p, c, c == c0);
            const float m = __ldcg(q + r), l = __ldcg(q + S::MT + r), t = fmaxf(top, m);
            const float base = t == __int_as_float(0xff800000) ? 0.f : t;
            sum = sum * ex2((top - base) * rs) + l * ex2((m - base) * rs);
            top = t;
        }
        tops[r] = top == __int_as_float(0xff800000) ? 0.f : top;
        invs[r] = sum == 0.f ? 0.f : 1.f / sum;
        scales[r] = rs;
        if (p.lse && blockIdx.y == 0) {
            int tok, head;
            row_of<S>(p, cur, r, tok, head);
            p.lse[(int64_t)tok * p.n_head + head] = log_sum(top, rs, S::OFF, sum);
        }
    }
    __syncthreads();
    // the values: four places a thread and two parts in flight
    const int n = rows * (p.dim / 4), stride = gridDim.y * JOIN_THREADS;
    for (int i0 = blockIdx.y * JOIN_THREADS + threadIdx.x; i0 < n; i0 += 4 * stride) {
        float4 o[4];
        int row[4], at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + u * stride, n - 1), d = i / rows;
            row[u] = i - d * rows;
            at[u] = part_value<S>(row[u], d * 4);
            o[u] = float4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll 2
        for (int c = c0; c <= c1; ++c) {
            const float* q = part_slot<S>(p, c, c == c0);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(q + at[u]));
                const float w = ex2((__ldcg(q + row[u]) - tops[row[u]]) * scales[row[u]]);
                o[u].x = __fmaf_rn(x.x, w, o[u].x), o[u].y = __fmaf_rn(x.y, w, o[u].y);
                o[u].z = __fmaf_rn(x.z, w, o[u].z), o[u].w = __fmaf_rn(x.w, w, o[u].w);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (i0 + u * stride >= n) break;
            const float inv = invs[row[u]];
            const int d = (i0 + u * stride) / rows * 4;
            int tok, head;
            row_of<S>(p, cur, row[u], tok, head);
            Pack<T, 4> y;
            y.v[0] = from_f32<T>(o[u].x * inv), y.v[1] = from_f32<T>(o[u].y * inv);
            y.v[2] = from_f32<T>(o[u].z * inv), y.v[3] = from_f32<T>(o[u].w * inv);
            *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(p.out) + (int64_t)tok * p.out_stride + (int64_t)head * p.dim + d) = y;
        }
    }
}

// The attention's launch and the join's after it.
template <class S, class... Args>
int launch_and_join(void (*kernel)(const AttnParams, Args...), const AttnParams& p, int ctas, cudaStream_t s, Args... args) {
    // the attribute is the device's: set on the first call there
    static std::atomic<uint64_t> set{0};
    int device = 0;
    cudaGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (!(set.load() & bit)) {
        const void* f = reinterpret_cast<const void*>(kernel);
        if (cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::BYTES) != cudaSuccess) return BH_EIO;
        if (device < 64) set.fetch_or(bit);
    }
    kernel<<<(unsigned)ctas, S::THREADS, S::BYTES, s>>>(p, args...);
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    // one wave: up to four CTAs an SM share a row tile's values
    c.gridDim = dim3((unsigned)ctas, (unsigned)(S::MT * S::DP / 4 > JOIN_THREADS * 4 ? 4 / S::CTAS : 1));
    c.blockDim = dim3(JOIN_THREADS);
    c.stream = s;
    c.attrs = &pdl;
    c.numAttrs = 1;
    if (cudaGetLastError() != cudaSuccess) return BH_EIO;
    return cudaLaunchKernelEx(&c, tree_attention_join_kernel<S>, p) == cudaSuccess ? BH_OK : BH_EIO;
}

// A ring's wait. One that runs out sets the status word, and every later wait
// of the CTA gives up at once, so the CTA still comes to its end.
template <class Shared>
__device__ __forceinline__ void ring_wait(Shared& sh, uint64_t* bar, uint32_t parity, int* status) {
    if (mbar_try_wait(bar, parity)) return;
    if (*(volatile int*)&sh.given_up) return;
    if (!mbar_wait_bounded(bar, parity)) {
        sh.given_up = 1;
        set_status(status, ST_TIMEOUT);
    }
}

// The copying warp: tiles f0 .. f1 of the line into the ring.
template <class S>
__device__ __forceinline__ void copy_tiles(const AttnParams& p, AttnShared<S>& sh, uint32_t tiles_a, int64_t f1) {
    using C = typename S::C;
    constexpr int TN = S::TN, STAGES = S::STAGES, CPR = S::ROW / 16;
    constexpr int RPP = CPR <= 32 ? 32 / CPR : 1;  // rows of one pass of the warp
    constexpr int CPL = CPR <= 32 ? 1 : CPR / 32;  // chunks of a row a lane copies
    constexpr int NR = (TN + 31) / 32;
    const int lane = threadIdx.x & 31;
    const int used = p.dim * (int)sizeof(C) / 16;
    const bool runs = p.block.d % 8 == 0;
    Cursor at = sh.first;
    uint32_t next_pos[NR];
    int32_t next_id[NR];
    // the rows' block ids are fetched a tile ahead
    auto fetch = [&] {
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const uint32_t r = j * 32 + lane, pos = (uint32_t)at.tile * TN + r;
            next_pos[j] = pos;
            next_id[j] = -2;  // no such position
            if (r < TN && pos < (uint32_t)(at.w.ctx + at.w.n_new))
                next_id[j] = p.tables[(int64_t)at.seq * p.max_blocks + p.block.div(pos)];
        }
    };
    fetch();
    int stage = 0;
    uint32_t turn = 1;  // parity of the stage's last release; the first pass waits for none
    for (bool more = at.place() < f1; more;) {
        int64_t off[NR];
        uint32_t ok[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            off[j] = -1;
            if ((uint32_t)next_id[j] < p.kv.n_blocks)
                off[j] = (next_id[j] * p.kv.block_stride + (next_pos[j] - p.block.div(next_pos[j]) * p.block.d) * p.kv.token_stride +
                          at.head * p.kv.head_stride) * (int)sizeof(C);
            else if (next_id[j] != -2)
                set_status(p.status, ST_BADARG);
            ok[j] = __ballot_sync(0xffffffffu, off[j] >= 0);
        }
        const bool history = (uint32_t)at.tile * TN + TN <= (uint32_t)at.w.ctx;
        more = next_place<S>(at) < f1;
        if (more) {
            next_tile<S>(at, p);
            fetch();
        }
        ring_wait(sh, &sh.empty[stage], turn, p.status);
        if (lane == 0) {
            bool all = history;
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                sh.valid[stage][j] = ok[j];
                all = all && ok[j] == (TN < 32 ? (1u << TN % 32) - 1 : 0xffffffffu);
            }
            sh.whole[stage] = all;
        }
        const uint32_t k_to = tiles_a + stage * 2 * S::TILE, v_to = k_to + S::TILE;
        const uint8_t* kb = static_cast<const uint8_t*>(p.kv.k);
        const uint8_t* vb = static_cast<const uint8_t*>(p.kv.v);
        bool every = true;
#pragma unroll
        for (int j = 0; j < NR; ++j) every = every && ok[j] == (TN < 32 ? (1u << TN % 32) - 1 : 0xffffffffu);
        if (every && runs) {
            // eight rows at a time lie at one distance from one another: an
            // address for each run, not for each row (a tile's 64 copies took
            // 3200 cycles to issue row by row)
            const int64_t next_row = p.kv.token_stride * (int)sizeof(C) * RPP;
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
                for (int q = 0; q < (TN < 32 ? TN : 32) / 8; ++q) {
                    const int64_t run = __shfl_sync(0xffffffffu, (long long)off[j], q * 8);
#pragma unroll
                    for (int i = 0; i < CPL; ++i) {
                        const int c = lane % CPR + 32 * i;
                        if (c >= used) continue;
                        int64_t at_row = run + lane / CPR * (next_row / RPP) + c * 16;
#pragma unroll
                        for (int e = 0; e < 8; e += RPP, at_row += next_row) {
                            const int r = j * 32 + q * 8 + e + lane / CPR;
                            cp_async16(k_to + k_chunk<S>(r, c), kb + at_row);
                            cp_async16(v_to + v_chunk<S>(r, c), vb + at_row);
                        }
                    }
                }
        } else {
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll 4
                for (int q = 0; q < (TN < 32 ? TN : 32) / RPP; ++q) {
                    const int in = q * RPP + lane / CPR, r = j * 32 + in;
                    const int64_t row = __shfl_sync(0xffffffffu, (long long)off[j], in);
#pragma unroll
                    for (int i = 0; i < CPL; ++i) {
                        const int c = lane % CPR + 32 * i;
                        if (c < used) {
                            const int64_t src = (row < 0 ? 0 : row) + c * 16;
                            cp_async16(k_to + k_chunk<S>(r, c), kb + src, row < 0 ? 0 : 16);
                            cp_async16(v_to + v_chunk<S>(r, c), vb + src, row < 0 ? 0 : 16);
                        }
                    }
                }
        }
        // 32 arrivals when the lanes' copies have landed, one for `valid`
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sh.full[stage])) : "memory");
        if (lane == 0) mbar_arrive(&sh.full[stage]);
        if (++stage == STAGES) stage = 0, turn ^= 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class S>
__global__ void __launch_bounds__(S::THREADS, S::CTAS) tree_attention_kernel(const AttnParams p) {
    using T = typename S::T;
    using C = typename S::C;
    constexpr int MT = S::MT, TN = S::TN, WN = S::WN, NT = S::NT, STAGES = S::STAGES, ROW = S::ROW;
    constexpr int SN = WN / 8;     // score tiles of a warp
    constexpr int CPR = ROW / 16;  // chunks of a row
    constexpr int NC = S::COMPUTE;
    constexpr int RPP = NC / CPR;  // rows a pass of the computing warps covers
    constexpr float OFF = S::OFF;
    const float NONE = __int_as_float(0xff800000);
    extern __shared__ __align__(1024) uint8_t tiles[];
    __shared__ AttnShared<S> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int rg = warp % S::RG, kg = warp / S::RG;
    const int group = (int)p.group.d;
    uint8_t* q_mem = tiles + STAGES * 2 * S::TILE;
    const uint32_t tiles_a = smem_u32(tiles), q_a = smem_u32(q_mem);

    int64_t per, f0, f1;
    pdl_trigger();
    find_part<S>(p, sh, per, f0, f1);
    __syncthreads();
    if (f0 >= f1 || sh.first.place() >= f1) {  // no tile begins in the share
        if (tid == 0) leave_split<S>(p, sh.first, false, per);
        return;
    }
    // columns behind the head's own are zero throughout
    if (p.dim < S::DP)
        for (int i = tid; i < STAGES * 2 * TN * CPR; i += S::THREADS)
            if ((i % CPR) * 16 >= p.dim * (int)sizeof(C)) {
                const int r = i / CPR % TN, which = i / CPR / TN;
                const int o = (which & 1) ? v_chunk<S>(r, i % CPR) : k_chunk<S>(r, i % CPR);
                *reinterpret_cast<uint4*>(tiles + which * S::TILE + o) = uint4{0, 0, 0, 0};
            }
    if (tid < STAGES) {
        mbar_init(&sh.full[tid], 33);
        mbar_init(&sh.empty[tid], S::WARPS);
        fence_mbar_init();
    }
    if (tid == 0) sh.given_up = 0;
    __syncthreads();
    if (warp == S::WARPS) {
        copy_tiles<S>(p, sh, tiles_a, f1);
        return;
    }
    Cursor cur = sh.first;
    auto sync = [] { named_bar(1, NC); };

    float acc[NT][4], m[2], l[2];
    bool fresh = true;  // a row tile begins
    bool sees_all = true;
    int stage = 0;
    uint32_t turn = 0;
    // lane's places in the query rows, K and V: the tile's offset and the step's chunk are added by xor
    const int ar = (lane & 7) + (lane & 8), ac = lane >> 4;              // A and V: rows, then chunks
    const int br = (lane & 7) + ((lane >> 4) << 3), bc = lane >> 3 & 1;  // K: chunks, then rows
    const uint32_t q_lane = q_a + k_chunk<S>(rg * 16 + ar, ac);
    const uint32_t k_lane = k_chunk<S>(kg * WN + br, bc), v_lane = v_chunk<S>(kg * WN + ar, ac);

    // tiles until the line position f1
    while (cur.place() < f1) {
        const int rows = min(MT, cur.w.n_new * group - cur.row_tile * MT);
        if (fresh) {
            // the rows of q, split and swizzled, a warp's in turn
            bool all = true;
            for (int r = warp; r < MT; r += S::WARPS) {
                const bool live = r < rows;
                const int row = cur.row_tile * MT + r, i = (int)p.group.div(row), h = cur.head * group + row - i * group;
                const T* src = static_cast<const T*>(p.q) + (int64_t)(cur.w.start + i) * p.q_stride + (int64_t)h * p.dim;
                // scores are q.k times rs >= 0: a negative scale turns q
                float rs = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-30f);
                float up = p.scale < 0.f ? -1.f : p.scale == 0.f ? 0.f : 1.f;
                if constexpr (S::NS == 2) {
                    // a power of two that brings the row's largest value to 2^10 .. 2^11
                    float top = 0.f;
                    if (live)
                        for (int d = lane; d < p.dim; d += 32) top = fmaxf(top, fabsf(to_f32(src[d])));
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const int e = top > 0.f && top < 3e38f ? max(-90, min(110, ilogbf(top))) : 10;
                    up *= ldexpf(1.f, 10 - e);
                    rs = fmaxf(rs * ldexpf(1.f, e - 10), 1e-37f);
                }
                for (int c = lane; c < CPR; c += 32) {
                    constexpr int V = 16 / sizeof(C), VT = 16 / sizeof(T);
                    float x[V];
#pragma unroll
                    for (int b = 0; b < V / VT; ++b) {
                        Pack<T, VT> y;
                        const bool in = live && c * V < p.dim;
                        if (in) y = *reinterpret_cast<const Pack<T, VT>*>(src + c * V + b * VT);
#pragma unroll
                        for (int e = 0; e < VT; ++e) x[b * VT + e] = in ? to_f32(y.v[e]) * up : 0.f;
                    }
                    uint8_t* dst = q_mem + k_chunk<S>(r, c);
#pragma unroll
                    for (int part = 0; part < S::NS; ++part) {
                        Pack<C, V> y;
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            y.v[e] = from_f32<C>(x[e]);
                            x[e] -= to_f32(y.v[e]);
                        }
                        *reinterpret_cast<Pack<C, V>*>(dst + part * MT * ROW) = y;
                    }
                }
                const uint64_t drafts = cur.w.n_new >= 64 ? ~0ull : (1ull << cur.w.n_new) - 1;
                uint64_t see = 0;
                if (live) see = (p.mask ? (uint64_t)p.mask[cur.w.start + i] : i >= 63 ? ~0ull : (2ull << i) - 1) & drafts;
                all = all && (!live || see == drafts);
                if (lane == 0) sh.mask[r] = see, sh.row_scale[r] = rs;
            }
            if (lane == 0) sh.sees_all[warp] = all;
            sync();
            sees_all = true;
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) sees_all = sees_all && sh.sees_all[w];
            m[0] = m[1] = NONE;
            l[0] = l[1] = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
            fresh = false;
        }
        ring_wait(sh, &sh.full[stage], turn, p.status);

        const int pos0 = cur.tile * TN;
        const uint32_t k_at = tiles_a + stage * 2 * S::TILE, v_at = k_at + S::TILE;
        const uint8_t* v_mem = tiles + stage * 2 * S::TILE + S::TILE;
        // drafts: by the lengths alone, the same in every warp also after a wait that
        // ran out, when `whole` may not be: barriers depend on it
        const bool whole = sh.whole[stage], drafts = pos0 + TN > cur.w.ctx;

        // A draft that some row does not see must not reach that row's sums:
        // the products would make NaN of 0 times an infinity. Rows of V that
        // hold one are zeroed here and added by themselves below.
        bool mend = false;
        if (drafts && !sees_all) {
            sync();  // a warp may still be adding rows of the tile before
            if (tid < (TN + 31) / 32) sh.bad[tid] = 0;
            sync();
#pragma unroll
            for (int i = 0; i < (TN + RPP - 1) / RPP; ++i) {
                const int r = tid / CPR + i * RPP;
                if (r >= TN || pos0 + r < cur.w.ctx) continue;
                const uint4 x = *reinterpret_cast<const uint4*>(v_mem + v_chunk<S>(r, tid % CPR));
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t u = e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w;
                    if constexpr (S::F) {
                        bad = bad || (u & 0x7f800000u) == 0x7f800000u;
                    } else {
                        constexpr uint32_t ex = S::TC == BH_F16 ? 0x7c00u : 0x7f80u;
                        bad = bad || (u & ex) == ex || (u >> 16 & ex) == ex;
                    }
                }
                if (bad) atomicOr(&sh.bad[r / 32], 1u << (r & 31));
            }
            sync();
#pragma unroll
            for (int i = 0; i < (TN + 31) / 32; ++i) mend = mend || sh.bad[i];
            if (mend) {
#pragma unroll
                for (int i = 0; i < (TN + RPP - 1) / RPP; ++i) {
                    const int r = tid / CPR + i * RPP;
                    if (r < TN && sh.bad[r / 32] >> (r & 31) & 1)
                        *reinterpret_cast<uint4*>(tiles + stage * 2 * S::TILE + S::TILE +
                                                  v_chunk<S>(r, tid % CPR)) = uint4{0, 0, 0, 0};
                }
                sync();
            }
        }

        // scores; with small parts or TF32 terms in accumulators of their own, even and odd steps apart
        constexpr int CH = S::F ? 3 : S::NS == 1 ? 1 : S::NS;
        float sc[CH][SN][4];
        if constexpr (S::F) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int n = 0; n < SN; ++n) sc[c][n][0] = sc[c][n][1] = sc[c][n][2] = sc[c][n][3] = 0.f;
            // 16 values of a head at a time: a lane's four consecutive ones are two pairs of contraction indexes
            const float* qf = reinterpret_cast<const float*>(q_mem);
            const float* kf = reinterpret_cast<const float*>(tiles + stage * 2 * S::TILE);
#pragma unroll 4
            for (int d = 0; d < S::DP / 16; ++d) {
                uint32_t ah[2][4], al[2][4];
                const int r = rg * 16 + g;
                const float4 x = *reinterpret_cast<const float4*>(qf + k_chunk<S>(r, d * 4 + t4) / 4);
                const float4 y = *reinterpret_cast<const float4*>(qf + k_chunk<S>(r + 8, d * 4 + t4) / 4);
                split_tf32(x.x, ah[0][0], al[0][0]);
                split_tf32(y.x, ah[0][1], al[0][1]);
                split_tf32(x.y, ah[0][2], al[0][2]);
                split_tf32(y.y, ah[0][3], al[0][3]);
                split_tf32(x.z, ah[1][0], al[1][0]);
                split_tf32(y.z, ah[1][1], al[1][1]);
                split_tf32(x.w, ah[1][2], al[1][2]);
                split_tf32(y.w, ah[1][3], al[1][3]);
#pragma unroll
                for (int n = 0; n < SN; ++n) {
                    const float4 k4 = *reinterpret_cast<const float4*>(kf + k_chunk<S>(kg * WN + n * 8 + g, d * 4 + t4) / 4);
                    uint32_t hi[4], lo[4];
                    split_tf32(k4.x, hi[0], lo[0]);
                    split_tf32(k4.y, hi[1], lo[1]);
                    split_tf32(k4.z, hi[2], lo[2]);
                    split_tf32(k4.w, hi[3], lo[3]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_tf32(sc[2][n], al[j], hi[2 * j], hi[2 * j + 1]);
                        mma_tf32(sc[2][n], ah[j], lo[2 * j], lo[2 * j + 1]);
                        mma_tf32(sc[j][n], ah[j], hi[2 * j], hi[2 * j + 1]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int d = 0; d < S::DP / 16; ++d) {
                uint32_t b[SN / 2][4];
#pragma unroll
                for (int n = 0; n < SN / 2; ++n) ldsm4(b[n], ((k_at + k_lane) ^ (d << 5)) + n * 16 * ROW);
#pragma unroll
                for (int part = 0; part < S::NS; ++part) {
                    uint32_t a[4];
                    ldsm4(a, (q_lane ^ (d << 5)) + part * MT * ROW);
#pragma unroll
                    for (int n = 0; n < SN / 2; ++n) {
                        if (d == 0) {
                            mma16_first<C>(sc[part][2 * n], a, b[n][0], b[n][1]);
                            mma16_first<C>(sc[part][2 * n + 1], a, b[n][2], b[n][3]);
                        } else {
                            mma16<C>(sc[part][2 * n], a, b[n][0], b[n][1]);
                            mma16<C>(sc[part][2 * n + 1], a, b[n][2], b[n][3]);
                        }
                    }
                }
            }
        }
        float (&s)[SN][4] = sc[0];
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (CH == 2) s[n][e] += sc[CH - 1][n][e];
                if constexpr (CH == 3) s[n][e] += sc[CH - 2][n][e] + sc[CH - 1][n][e];
            }
        // probabilities
        float alpha[2];
        bool grew = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = rg * 16 + g + 8 * h;
            const float rs = sh.row_scale[r];
            float top = m[h];
            if (!whole) {
                const uint64_t mask = sh.mask[r];
#pragma unroll
                for (int n = 0; n < SN; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int in = kg * WN + n * 8 + 2 * t4 + e, j = pos0 + in - cur.w.ctx;
                        const bool see = (sh.valid[stage][in / 32] >> (in & 31) & 1) && (j < 0 || (j < 64 && (mask >> j & 1)));
                        if (!see) s[n][2 * h + e] = NONE;
                    }
            }
#pragma unroll
            for (int n = 0; n < SN; ++n) top = fmaxf(top, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float base = top == NONE ? 0.f : top;
            alpha[h] = ex2((m[h] - base) * rs);
            grew = grew || top > m[h];
            m[h] = top;
            const float shift = OFF - base * rs;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < SN; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = s[n][2 * h + e];
                    // exact differences where the sums are; one operation where a 16-bit result hides base's rounding
                    x = ex2(S::EXACT ? __fmaf_rn(x - base, rs, OFF) : __fmaf_rn(x, rs, shift));
                    sum += x;
                }
            l[h] = __fmaf_rn(l[h], alpha[h], sum);
        }
        if constexpr (!S::EXACT) {
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[n][e] *= alpha[e >> 1];
                    }
            }
        }
        // the sums with V
        constexpr bool APART = S::EXACT;  // this tile's products by themselves
        if constexpr (S::F) {
            const float* vf = reinterpret_cast<const float*>(v_mem);
            uint32_t ah[SN][4], al[SN][4];
#pragma unroll
            for (int n = 0; n < SN; ++n) {
                split_tf32(s[n][0], ah[n][0], al[n][0]);
                split_tf32(s[n][2], ah[n][1], al[n][1]);
                split_tf32(s[n][1], ah[n][2], al[n][2]);
                split_tf32(s[n][3], ah[n][3], al[n][3]);
            }
            // a lane's columns of four accumulator tiles are four consecutive values of V
#pragma unroll
            for (int d = 0; d < S::DP / 32; ++d) {
                float o[4][4];
#pragma unroll
                for (int n = 0; n < SN; ++n) {
                    const int r = kg * WN + n * 8 + 2 * t4;
                    const float4 x = *reinterpret_cast<const float4*>(vf + v_chunk<S>(r, d * 8 + g) / 4);
                    const float4 y = *reinterpret_cast<const float4*>(vf + v_chunk<S>(r + 1, d * 8 + g) / 4);
                    uint32_t xh[4], xl[4], yh[4], yl[4];
                    split_tf32(x.x, xh[0], xl[0]);
                    split_tf32(x.y, xh[1], xl[1]);
                    split_tf32(x.z, xh[2], xl[2]);
                    split_tf32(x.w, xh[3], xl[3]);
                    split_tf32(y.x, yh[0], yl[0]);
                    split_tf32(y.y, yh[1], yl[1]);
                    split_tf32(y.z, yh[2], yl[2]);
                    split_tf32(y.w, yh[3], yl[3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (n == 0) mma_tf32_first(o[j], al[n], xh[j], yh[j]);
                        else mma_tf32(o[j], al[n], xh[j], yh[j]);
                        mma_tf32(o[j], ah[n], xl[j], yl[j]);
                        mma_tf32(o[j], ah[n], xh[j], yh[j]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[4 * d + j][e] = __fmaf_rn(acc[4 * d + j][e], alpha[e >> 1], o[j][e]);
            }
        } else {
            uint32_t a[SN / 2][S::NS][4];
#pragma unroll
            for (int n = 0; n < SN / 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = s[2 * n + (i >> 1)][2 * (i & 1)], y = s[2 * n + (i >> 1)][2 * (i & 1) + 1];
#pragma unroll
                    for (int part = 0; part < S::NS; ++part) {
                        a[n][part][i] = pack2<C>(x, y);
                        if (part + 1 < S::NS) {
                            float u, v;
                            unpack2<C>(a[n][part][i], u, v);
                            x -= u, y -= v;
                        }
                    }
                }
#pragma unroll
            for (int d = 0; d < NT; d += 2) {
                float o[2][4];
#pragma unroll
                for (int n = 0; n < SN / 2; ++n) {
                    uint32_t b[4];
                    ldsm4_t(b, ((v_at + v_lane) ^ (d << 4)) + n * 16 * ROW);
#pragma unroll
                    for (int part = S::NS - 1; part >= 0; --part)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float (&to)[4] = APART ? o[j] : acc[d + j];
                            if (APART && n == 0 && part == S::NS - 1)
                                mma16_first<C>(to, a[n][part], b[2 * j], b[2 * j + 1]);
                            else
                                mma16<C>(to, a[n][part], b[2 * j], b[2 * j + 1]);
                        }
                }
                if constexpr (APART) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[d + j][e] = __fmaf_rn(acc[d + j][e], alpha[e >> 1], o[j][e]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[stage]);
        // the value of a head that accumulator (tile n, column e of 2) holds
        auto dim_of = [&](int n, int e) {
            return S::F ? (n / 4) * 32 + 8 * t4 + 4 * e + n % 4 : n * 8 + 2 * t4 + e;
        };
        if (mend) {  // from memory: the ring's copy may be gone
#pragma unroll
            for (int n = 0; n < SN; ++n)
                for (int in = kg * WN + n * 8; in < kg * WN + n * 8 + 8; ++in) {
                    if (!(sh.bad[in / 32] >> (in & 31) & 1)) continue;
                    const uint32_t pos = (uint32_t)(pos0 + in), blk = p.block.div(pos);
                    const int32_t id = p.tables[(int64_t)cur.seq * p.max_blocks + blk];
                    const C* v = static_cast<const C*>(p.kv.v) + id * p.kv.block_stride +
                                 (pos - blk * p.kv.block_size) * p.kv.token_stride + cur.head * p.kv.head_stride;
                    const int src = (lane & ~3) | (in & 7) >> 1;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float p0 = __shfl_sync(0xffffffffu, s[n][2 * h], src);
                        const float p1 = __shfl_sync(0xffffffffu, s[n][2 * h + 1], src);
                        const float pr = in & 1 ? p1 : p0;
                        const int j = (int)pos - cur.w.ctx;
                        if (j < 64 && (sh.mask[rg * 16 + g + 8 * h] >> j & 1)) {
#pragma unroll
                            for (int d = 0; d < NT; ++d)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    if (dim_of(d, e) < p.dim)
                                        acc[d][2 * h + e] =
                                            __fmaf_rn(pr, to_f32(v[dim_of(d, e)]), acc[d][2 * h + e]);
                        }
                    }
                }
        }

        if (++stage == STAGES) stage = 0, turn ^= 1;
        const bool row_tile_ends = cur.tile == cur.w.tiles - 1;
        const bool ends = next_place<S>(cur) >= f1;
        if (row_tile_ends || ends) {
            // join the position groups: maxima, then sums in their order
            float* epi = reinterpret_cast<float*>(q_mem);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                const int r = rg * 16 + g + 8 * h;
                if (t4 == 0) sh.part_m[kg][r] = m[h], sh.part_l[kg][r] = l[h];
            }
            sync();
            float f2[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = rg * 16 + g + 8 * h;
                float top = sh.part_m[0][r];
#pragma unroll
                for (int k = 1; k < S::KG; ++k) top = fmaxf(top, sh.part_m[k][r]);
                const float base = top == NONE ? 0.f : top;
                const float rs = sh.row_scale[r];
                f2[h] = ex2((m[h] - base) * rs);
                if (kg == 0 && t4 == 0) {
                    float sum = 0.f;
#pragma unroll
                    for (int k = 0; k < S::KG; ++k) sum += sh.part_l[k][r] * ex2((sh.part_m[k][r] - base) * rs);
                    sh.row_m[r] = top;
                    sh.row_l[r] = sum;
                }
            }
            // few rows: a place for every group; else one place, the groups in turn
            const bool side = rows * S::KG <= MT;
#pragma unroll
            for (int k = 0; k < S::KG; ++k) {
                if (kg == k) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = rg * 16 + g + 8 * h;
                        if (r >= rows) continue;
                        float* row = epi + (side ? k * rows + r : r) * S::DP;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float x = acc[n][2 * h + e] * f2[h];
                                row[dim_of(n, e)] = k == 0 || side ? x : row[dim_of(n, e)] + x;
                            }
                    }
                }
                if (!side && k + 1 < S::KG) sync();
            }
            sync();
            auto joined = [&](int r, int d) {
                float4 o = *reinterpret_cast<const float4*>(epi + r * S::DP + d);
                if (side)
#pragma unroll
                    for (int k = 1; k < S::KG; ++k) {
                        const float4 x = *reinterpret_cast<const float4*>(epi + (k * rows + r) * S::DP + d);
                        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
                    }
                return o;
            };
            const int dv = p.dim / 4;
            if (cur.first >= f0 && row_tile_ends) {
                for (int i = tid; i < rows * dv; i += NC) {
                    const int r = i / dv, d = i % dv * 4;
                    const float4 o = joined(r, d);
                    const float sum = sh.row_l[r], inv = sum == 0.f ? 0.f : 1.f / sum;
                    int tok, head;
                    row_of<S>(p, cur, r, tok, head);
                    Pack<T, 4> y;
                    y.v[0] = from_f32<T>(o.x * inv), y.v[1] = from_f32<T>(o.y * inv);
                    y.v[2] = from_f32<T>(o.z * inv), y.v[3] = from_f32<T>(o.w * inv);
                    *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(p.out) + (int64_t)tok * p.out_stride + (int64_t)head * p.dim + d) = y;
                    if (p.lse && d == 0) p.lse[(int64_t)tok * p.n_head + head] = log_sum(sh.row_m[r], sh.row_scale[r], OFF, sum);
                }
            } else {
                float* to = part_slot<S>(p, blockIdx.x, cur.first >= f0);
                if (tid < rows) to[tid] = sh.row_m[tid], to[MT + tid] = sh.row_l[tid], to[2 * MT + tid] = sh.row_scale[tid];
                for (int i = tid; i < rows * dv; i += NC) {
                    const int r = i % rows, d = i / rows * 4;
                    *reinterpret_cast<float4*>(to + part_value<S>(r, d)) = joined(r, d);
                }
            }
            sync();  // the sums' place is the next query rows'
            fresh = true;
        }
        if (ends) {
            if (tid == 0) leave_split<S>(p, cur, cur.first >= f0 && !row_tile_ends, per);
            break;
        }
        next_tile<S>(cur, p);
    }
}

template <class S>
int launch_attention_shape(const AttnParams& p, int num_sms, cudaStream_t s) {
    static_assert(sizeof(AttnShared<S>) + 1024 <= S::MORE, "the static shared memory is as small as its share");
    static_assert(S::BYTES + sizeof(AttnShared<S>) <= 227 * 1024, "an SM's shared memory holds a CTA");
    static_assert(S::CTAS * (2 * S::SLOT * sizeof(float) + sizeof(Split)) <= WS_CTAS_PER_SM * WS_CTA_BYTES, "partials fit the workspace");
    return launch_and_join<S>(&tree_attention_kernel<S>, p, num_sms * S::CTAS, s);
}

// Row tiles of 16 rows up to heads of 128 values, and rows beyond them in further
// tiles, whose reads of the cache meet the first one's in the L2: 48 sequences up
// to 2048 long, 8 heads of 128 values, fp32 over f16, 32 / 64 / 256 rows a head
// 122 / 199 / 656 us (row tiles of 32 and 64: 207 / 366 / 1040, for want of
// registers and CTAs; fp32, bf16 and heads of 64 alike). Heads of 256 leave room
// for one CTA an SM in any case: 32 / 64 / 256 rows in tiles of as many, up to 64,
// 291 / 461 / 1386 us (in tiles of 16: 319 / 602 / 2056).
template <int TA, int TC>
int launch_attention(const AttnParams& p, int num_sms, cudaStream_t s) {
    const int rows = p.max_new * (p.n_head / p.n_kv);
    if (p.dim <= 64) return launch_attention_shape<AttnShape<TA, TC, 64, 1, 4>>(p, num_sms, s);
    if (p.dim <= 128) return launch_attention_shape<AttnShape<TA, TC, 128, 1, 4>>(p, num_sms, s);
    if (rows <= 16) return launch_attention_shape<AttnShape<TA, TC, 256, 1, 4>>(p, num_sms, s);
    if (rows <= 32) return launch_attention_shape<AttnShape<TA, TC, 256, 2, 2>>(p, num_sms, s);
    return launch_attention_shape<AttnShape<TA, TC, 256, 4, 2>>(p, num_sms, s);
}

// one for each pair of types, in files of their own
int launch_attention_f32_f32(const AttnParams& p, int num_sms, cudaStream_t s);
int launch_attention_f32_f16(const AttnParams& p, int num_sms, cudaStream_t s);
int launch_attention_f32_bf16(const AttnParams& p, int num_sms, cudaStream_t s);
int launch_attention_f16(const AttnParams& p, int num_sms, cudaStream_t s);
int launch_attention_bf16(const AttnParams& p, int num_sms, cudaStream_t s);

}  // namespace bh
