// tree_attention_wide.cuh — bh_tree_attention for many query rows of a KV head
// in 16-bit types: the same sums over the same line of tiles as
// tree_attention.cuh, with the products on the fifth-generation tensor cores.
//
// From about 100 rows on, the products bound the mma.sync kernel (550 TFLOP/s
// measured for the whole GPU: 84 flops a byte of cache at full bandwidth).
// tcgen05.mma does a tile's 128 x 128 scores and sums in 512 cycles each, and
// the read of a tile takes about 2800 at full bandwidth, so up to 128 rows the
// cache's read is the bound again, and near it up to 256. Measured in a graph, 32
// heads over 8 of 128 values in bf16: 24 sequences up to 12000 long with trees of
// up to 13 (one stream) 115 us, 5.4 TB/s; 16 up to 32768 with trees of up to 64
// (two streams) 273 us, 4.2 TB/s and 570 TFLOP/s, of which a tile of 128
// positions takes 4500 cycles: scores, softmax and sums of a stream follow one
// another, and two streams hide half of it. (Tiles of 64 with two score buffers
// for each of two streams, so that nothing waits: 326 us, bound by the issue of
// twice as many groups of products.)
//
// Two shapes of CTA. Rows of a stream lie on the 128 lanes of tensor memory, a
// thread each: scores S (in whose place the 16-bit probabilities P go) and sums.
//
// One stream (at most 128 rows in the call): two CTAs an SM, so that one's row
// tile can begin or end (query rows, output: microseconds behind the copies that
// are queued) while the other's products run. Tiles of 64 positions; two score
// buffers, so that S(n + 1) = Q K^T runs under the softmax of S(n).
//
// Two streams: a CTA has an SM, and tiles of 128 positions. More than 128 rows:
// both streams work on every tile, each with rows of its own. Fewer: both have
// the same rows and take every other tile, and are joined at the end.
//   4 warps a stream  a row a thread; maxima, probabilities, output
//   2 warps           copy K, V into rings of tiles, in the 128-byte swizzle that
//                     the tensor core reads (K with the contraction along the row,
//                     V across the rows): boxes of `box` tokens by tensor copies
//                     where the block size is a multiple of 8 and the tile is all
//                     history, else rows by 16-byte cp.async
//   1 warp            issues the products; P(n - 2) V goes before S(n) for two
//                     streams, so that one's products run under the other's softmax
// Rows' maxima grow by more than 2^8 before the sums are rescaled (rarely after
// the first tiles); the sums stay exact relative to the maximum in use.
#pragma once

#include "tree_attention.cuh"

namespace bh {

template <int TC_, int DP_, int STREAMS_>
struct WideShape {
    static constexpr int TC = TC_, DP = DP_, STREAMS = STREAMS_;
    using C = typename ValueOf<TC>::type;
    using T = C;
    // exponent added to f16 probabilities (2^6, and 2^8 that the maximum in use may
    // lag, of 2^16), so that what is above 2^-31 of the largest reaches the sums
    static constexpr float OFF = TC == BH_F16 ? 6.f : 0.f;
    static constexpr int TN = 64 * STREAMS, MT = 128 * STREAMS;
    static constexpr int SOFT = 128 * STREAMS, THREADS = SOFT + 96, CTAS = 3 - STREAMS;
    static constexpr int ROW = DP * 2, TILE = TN * ROW, BLOCK = TN * 128;  // 64 values of every row make a block
    static constexpr int K_STAGES = DP == 128 ? 3 : 5, V_STAGES = DP == 128 ? 2 : 5;
    static constexpr int Q_BYTES = MT * ROW;  // as large as the sums of 128 rows that pass between two streams
    static constexpr size_t BYTES = (size_t)(K_STAGES + V_STAGES) * TILE + Q_BYTES;
    static constexpr int SLOT = MT * (DP + 4);
    // tensor memory: scores of a stream (or buffer) every TN columns, sums behind them
    static constexpr int SUMS = 2 * TN, COLUMNS = 256 * STREAMS;
    // lengths on the line, from measured times: tiles of one stream's rows are
    // bound by the cache's read, those of two by the products between them, and
    // a row tile's begin and end, each load of which queues behind the other
    // CTAs' tiles, take as long as ten tiles of 128 or 14 of 64
    static constexpr int BEGIN = STREAMS == 2 ? 30 : 14;
    __device__ static __forceinline__ int weight(int rows) { return STREAMS == 1 ? 1 : rows > 128 ? 4 : 3; }
    static constexpr int META = 8;  // tiles whose descriptions are kept: more than the rings run ahead
};

template <class S>
struct WideShared {
    uint64_t k_full[S::K_STAGES], k_empty[S::K_STAGES], v_full[S::V_STAGES], v_empty[S::V_STAGES];
    uint64_t q_full, done;
    // by stream, or, of one stream, by turns: whoever waits for a phase has
    // seen the one before it on the same word, and the one after needs the waiter
    uint64_t s_full[2], p_full[2], o_full[2];
    uint32_t valid[S::META][S::TN / 32];  // rows of the tile that exist
    uint32_t bad[2][S::TN / 32];        // rows of a tile whose V is not finite, by stream or, if both work on it, by turns
    int whole[S::META];          // all rows exist, and none is a draft
    float part_m[S::STREAMS == 2 ? 128 : 1], part_l[S::STREAMS == 2 ? 128 : 1];
    int64_t scan[S::THREADS / 32];
    Cursor first;
    uint32_t tmem;
    int keep[2];  // the stream's sums hold something before its first product
    int given_up;
};

__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// arrival without a wait at a named barrier
__device__ __forceinline__ void named_bar_arrive(int id, int nthreads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}
// 32 columns of the warp's 32 lanes, a lane's row a thread
__device__ __forceinline__ void tm_load(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tm_store(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tm_store16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tm_load16(uint32_t (&r)[16], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tm_load8(uint32_t (&r)[8], uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
}
__device__ __forceinline__ void tm_store8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// box at (x, token, head, block) of the cache's tensor map
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int token, int head, int block,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(token), "r"(head), "r"(block), "r"(smem_u32(bar))
        : "memory");
}
// Shared-memory operand in 128-byte swizzled blocks of 64 values, as its
// descriptor's low word: the address, and `lead`, the bytes from one block to
// the next where the rows are the contraction (V; not used for Q and K). Moving
// the address by n bytes adds n / 16. The high word, OPERAND, is the same for
// all: 8-row groups 1024 bytes apart, 128-byte swizzle.
__device__ __forceinline__ uint32_t operand(uint32_t addr, uint32_t lead) {
    return (addr & 0x3ffffu) >> 4 | (lead >> 4) << 16;
}
constexpr uint32_t OPERAND = (1024 >> 4) | 1u << 14 | 2u << 29;
// 128 x n products of 16-bit values with fp32 sums; `across`: B's rows are the contraction
template <int TC>
__host__ __device__ constexpr uint32_t product(int n, bool across) {
    return 1u << 4 | (TC == BH_BF16 ? 1u << 7 | 1u << 10 : 0u) | (across ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 |
           (uint32_t)(128 >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t kind, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(kind), "r"((uint32_t)add), "r"(OPERAND)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t kind, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(kind), "r"((uint32_t)add), "r"(OPERAND)
        : "memory");
}
// one lane of a converged warp
__device__ __forceinline__ bool elected() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
// byte offset of a 16-byte chunk of a row in swizzled blocks of `rows` rows
template <int ROWS>
__device__ __forceinline__ int swizzled(int r, int c) {
    return (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// A row tile's part that a CTA has: its tiles from `cur` on.
struct WidePart {
    int rows, tiles;
    bool both;  // more than 128 rows: both streams work on every tile
    bool ends;  // with it the row tile
};
template <class S>
__device__ __forceinline__ WidePart wide_part(const AttnParams& p, const Cursor& cur, int64_t f1) {
    WidePart x;
    x.rows = min(S::MT, cur.w.n_new * (int)p.group.d - cur.row_tile * S::MT);
    x.both = S::STREAMS == 2 && x.rows > 128;
    x.ends = cur.last() < f1;
    x.tiles = x.ends ? cur.w.tiles - cur.tile : (int)((f1 - cur.place() + cur.w.weight - 1) / cur.w.weight);
    return x;
}
// To the next row tile; false where the CTA has none of it.
template <class S>
__device__ __forceinline__ bool next_part(Cursor& c, const AttnParams& p, int64_t f1) {
    c.tile = c.w.tiles - 1;
    if (next_place<S>(c) >= f1) return false;
    next_tile<S>(c, p);
    return true;
}

// One of the copying warps. box: tokens of a tensor copy, a power of two that
// divides the block size, or 0.
template <class S, bool V>
__device__ __forceinline__ void copy_wide(const AttnParams& p, const CUtensorMap* map, int box, WideShared<S>& sh,
                                          uint32_t ring, int64_t f1) {
    using C = typename S::C;
    constexpr int TN = S::TN, NR = TN / 32, CPR = S::ROW / 16, RPP = 32 / CPR;
    constexpr int STAGES = V ? S::V_STAGES : S::K_STAGES;
    const int lane = threadIdx.x & 31;
    const uint32_t used = (uint32_t)p.dim / 8;
    const uint8_t* base = static_cast<const uint8_t*>(V ? p.kv.v : p.kv.k);
    const int boxes = box ? TN / box : 0;
    Cursor at = sh.first;
    // a tile ahead: the block of the lane's box, or the blocks of its rows
    uint32_t next_pos = 0;
    int32_t next_id[NR];
    bool boxed = false;
    auto fetch = [&] {
        boxed = boxes > 0 && (uint32_t)at.tile * TN + TN <= (uint32_t)at.w.ctx;
        if (boxed) {
            if (lane < boxes) {
                next_pos = (uint32_t)at.tile * TN + lane * box;
                next_id[0] = p.tables[(int64_t)at.seq * p.max_blocks + p.block.div(next_pos)];
            }
        } else {
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                const uint32_t pos = (uint32_t)at.tile * TN + j * 32 + lane;
                next_id[j] = -2;  // no such position
                if (pos < (uint32_t)(at.w.ctx + at.w.n_new))
                    next_id[j] = p.tables[(int64_t)at.seq * p.max_blocks + p.block.div(pos)];
            }
        }
    };
    fetch();
    int stage = 0, count = 0;
    uint32_t turn = 1;
    named_bar(4, S::SOFT + 64);  // behind the first query rows' loads
    for (bool more = at.place() < f1; more; ++count) {
        uint64_t* full = V ? &sh.v_full[stage] : &sh.k_full[stage];
        uint64_t* empty = V ? &sh.v_empty[stage] : &sh.k_empty[stage];
        const uint32_t to = ring + stage * S::TILE;
        more = next_place<S>(at) < f1;
        const int meta = count % S::META;
        bool whole = boxed;
        if (boxed && !__all_sync(0xffffffffu, lane >= boxes || (uint32_t)next_id[0] < p.kv.n_blocks)) {
            // a block outside the cache: row by row
#pragma unroll
            for (int j = 0; j < NR; ++j)
                next_id[j] = p.tables[(int64_t)at.seq * p.max_blocks + p.block.div((uint32_t)at.tile * TN + j * 32 + lane)];
            whole = false;
        }
        if (whole) {
            const int token = (int)(next_pos - p.block.div(next_pos) * p.block.d), block = next_id[0], head = at.head;
            if (more) {
                next_tile<S>(at, p);
                fetch();
            }
            ring_wait(sh, empty, turn, p.status);
            __syncwarp();
            if (lane == 0) {
                if (!V) sh.whole[meta] = 1;
                mbar_arrive_expect_tx(full, S::TILE);
            }
            __syncwarp();
            if (lane < boxes) {
#pragma unroll
                for (int x = 0; x < S::DP / 64; ++x)
                    copy_box(to + x * S::BLOCK + lane * box * 128, map, x * 64, token, head, block, full);
            }
            mbar_arrive(full);
        } else {
            // the end of a sequence, or blocks that boxes do not fit
            int64_t off[NR];
            uint32_t ok[NR];
            const int first_draft = at.w.ctx - at.tile * TN;  // row of the tile
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                const uint32_t pos = (uint32_t)at.tile * TN + j * 32 + lane;
                off[j] = -1;
                if ((uint32_t)next_id[j] < p.kv.n_blocks)
                    off[j] = (next_id[j] * p.kv.block_stride + (pos - p.block.div(pos) * p.block.d) * p.kv.token_stride +
                              at.head * p.kv.head_stride) * (int)sizeof(C);
                else if (next_id[j] != -2)
                    set_status(p.status, ST_BADARG);
                ok[j] = __ballot_sync(0xffffffffu, off[j] >= 0);
            }
            if (more) {
                next_tile<S>(at, p);
                fetch();
            }
            ring_wait(sh, empty, turn, p.status);
            __syncwarp();
            if (!V && lane == 0) {
                bool all = first_draft >= TN;
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    sh.valid[meta][j] = ok[j];
                    all = all && ok[j] == 0xffffffffu;
                }
                sh.whole[meta] = all;
            }
            const int c = lane % CPR;
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
                for (int q = 0; q < 32 / RPP; ++q) {
                    const int in = q * RPP + lane / CPR;
                    const int64_t row = __shfl_sync(0xffffffffu, (long long)off[j], in);
                    cp_async16(to + swizzled<TN>(j * 32 + in, c), base + (row < 0 ? 0 : row) + (c < used ? c * 16 : 0),
                               row < 0 || c >= used ? 0 : 16);
                }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
            if (lane == 0) mbar_arrive(full);
        }
        if (++stage == STAGES) stage = 0, turn ^= 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // Tensor copies too have landed when the CTA ends, also one that gave up.
    for (int i = 0; i < STAGES && i < count; ++i) {
        if (--stage < 0) stage = STAGES - 1, turn ^= 1;
        mbar_wait_bounded(V ? &sh.v_full[stage] : &sh.k_full[stage], turn ^ 1);
    }
}

// The warp that issues the products, one of its lanes at a time; the others go
// along so that the operands stay in uniform registers (a single thread's own
// address arithmetic took 120 cycles a product, the product takes 64).
template <class S>
__device__ __forceinline__ void issue_products(const AttnParams& p, WideShared<S>& sh, uint32_t k_ring, uint32_t v_ring,
                                               uint32_t q_at, int64_t f1) {
    constexpr uint32_t QK = product<S::TC>(S::TN, false), PV = product<S::TC>(S::DP, true);
    constexpr int STEPS = S::DP / 16;
    const uint32_t tm = sh.tmem;
    Cursor cur = sh.first;
    int ks = 0, vs = 0;
    uint32_t kt = 0, vt = 0, qt = 0, pt[2] = {0, 0};
    while (cur.place() < f1) {
        const WidePart part = wide_part<S>(p, cur, f1);
        ring_wait(sh, &sh.q_full, qt, p.status);
        qt ^= 1;
        const int n_steps = part.both ? 2 * part.tiles : part.tiles;
        auto sums = [&](int m) {  // P V of step m
            const int w = m & 1;
            const bool first = !part.both || w == 0, last = !part.both || w == 1;  // of the tile's products
            ring_wait(sh, &sh.p_full[w], pt[w], p.status);
            pt[w] ^= 1;
            if (first) ring_wait(sh, &sh.v_full[vs], vt, p.status);
            __syncwarp();
            fence_proxy_async_smem();
            tm_fence_after();
            const int o = S::STREAMS == 2 ? w : 0;
            const uint32_t add = m >= S::STREAMS || *(volatile int*)&sh.keep[o];
            const uint32_t v = operand(v_ring + vs * S::TILE, S::BLOCK), pr = tm + w * S::TN;
            if (elected()) {
#pragma unroll
                for (int k = 0; k < S::TN / 16; ++k)  // 16 positions a step
                    mma_ts(tm + S::SUMS + o * S::DP, pr + k * 8, v + k * (2048 >> 4), PV, k > 0 ? true : add);
                tm_commit(&sh.o_full[w]);
                if (last) tm_commit(&sh.v_empty[vs]);
            }
            __syncwarp();
            if (last && ++vs == S::V_STAGES) vs = 0, vt ^= 1;
        };
        for (int n = 0; n < n_steps + 2; ++n) {
            if (S::STREAMS == 2 && n >= 2) sums(n - 2);
            if (n < n_steps) {
                const int w = n & 1;
                const bool first = !part.both || w == 0, last = !part.both || w == 1;
                if (first) ring_wait(sh, &sh.k_full[ks], kt, p.status);
                __syncwarp();
                fence_proxy_async_smem();
                tm_fence_after();
                const uint32_t k = operand(k_ring + ks * S::TILE, 0), q = operand(q_at + (part.both ? w * 128 * 128 : 0), 0);
                if (elected()) {
#pragma unroll
                    for (int i = 0; i < STEPS; ++i)  // 16 values of a head a step, four steps a block
                        mma_ss(tm + w * S::TN, q + (i / 4) * (S::MT * 128 >> 4) + (i % 4) * 2,
                               k + (i / 4) * (S::BLOCK >> 4) + (i % 4) * 2, QK, i > 0);
                    tm_commit(&sh.s_full[w]);
                    if (last) tm_commit(&sh.k_empty[ks]);
                }
                __syncwarp();
                if (last && ++ks == S::K_STAGES) ks = 0, kt ^= 1;
            }
            if (S::STREAMS == 1 && n >= 1 && n <= n_steps) sums(n - 1);
        }
        if (!next_part<S>(cur, p, f1)) break;
    }
    if (elected()) tm_commit(&sh.done);
    __syncwarp();
    if (!mbar_wait_bounded(&sh.done, 0)) set_status(p.status, ST_TIMEOUT);
    __syncwarp();
}

template <class S>
__global__ void __launch_bounds__(S::THREADS, S::CTAS)
    tree_attention_wide_kernel(const AttnParams p, const __grid_constant__ CUtensorMap k_map,
                               const __grid_constant__ CUtensorMap v_map, int box) {
    using C = typename S::C;
    constexpr int DP = S::DP, TN = S::TN, MT = S::MT, CPR = S::ROW / 16, SOFT = S::SOFT;
    constexpr int NC = TN / 32, K_WARP = SOFT / 32, V_WARP = K_WARP + 1, MMA_WARP = K_WARP + 2;
    const float NONE = __int_as_float(0xff800000);
    extern __shared__ __align__(1024) uint8_t mem[];
    __shared__ WideShared<S> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint8_t* q_mem = mem + (S::K_STAGES + S::V_STAGES) * S::TILE;
    const uint32_t k_ring = smem_u32(mem), v_ring = k_ring + S::K_STAGES * S::TILE, q_at = smem_u32(q_mem);

    int64_t per, f0, f1;
    pdl_trigger();
    find_part<S>(p, sh, per, f0, f1);
    __syncthreads();
    if (f0 >= f1 || sh.first.place() >= f1) {  // no tile begins in the share
        if (tid == 0) leave_split<S>(p, sh.first, false, per);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < S::K_STAGES; ++i) mbar_init(&sh.k_full[i], 33), mbar_init(&sh.k_empty[i], 1);
        for (int i = 0; i < S::V_STAGES; ++i) mbar_init(&sh.v_full[i], 33), mbar_init(&sh.v_empty[i], 1);
        mbar_init(&sh.q_full, SOFT);
        for (int w = 0; w < 2; ++w) {
            mbar_init(&sh.s_full[w], 1);
            mbar_init(&sh.p_full[w], 128);
            mbar_init(&sh.o_full[w], 1);
        }
        mbar_init(&sh.done, 1);
        fence_mbar_init();
        sh.given_up = 0;
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(S::COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_proxy_async_smem();
    tm_fence_before();
    __syncthreads();
    tm_fence_after();

    if (warp == K_WARP) {
        copy_wide<S, false>(p, &k_map, box, sh, k_ring, f1);
    } else if (warp == V_WARP) {
        copy_wide<S, true>(p, &v_map, box, sh, v_ring, f1);
    } else if (warp == MMA_WARP) {
        issue_products<S>(p, sh, k_ring, v_ring, q_at, f1);
    } else {
        const int w = S::STREAMS == 2 ? warp >> 2 : 0, lane_row = (warp & 3) * 32 + lane;
        const uint32_t tm_lane = sh.tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_at = tm_lane + S::SUMS + w * DP;
        const float rs = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-30f);
        const float turn_q = p.scale < 0.f ? -1.f : p.scale == 0.f ? 0.f : 1.f;
        const uint32_t q_and = p.scale == 0.f ? 0u : ~0u, q_xor = p.scale < 0.f ? 0x80008000u : 0u;
        auto sync = [] { named_bar(1, SOFT); };
        Cursor cur = sh.first;
        bool started = false;
        uint32_t st[2] = {0, 0}, ot[2] = {0, 0};  // parities of the next scores and sums
        int count = 0;  // tiles before this part
        while (cur.place() < f1) {
            const WidePart part = wide_part<S>(p, cur, f1);
            const int my = part.both ? w * 128 + lane_row : lane_row;  // the thread's row of the tile
            int my_tok, my_head;
            row_of<S>(p, cur, my, my_tok, my_head);
            const bool warp_live = my - lane < part.rows;
            uint64_t see = 0;
            if (my < part.rows)
                see = p.mask ? (uint64_t)p.mask[my_tok] : my_tok - cur.w.start >= 63 ? ~0ull : (2ull << (my_tok - cur.w.start)) - 1;
            if (cur.w.n_new < 64) see &= (1ull << cur.w.n_new) - 1;
            // The query rows, in blocks of 64 values. (What runs once a row tile
            // is kept short: its instructions are fetched anew, behind the copies;
            // sixteen loads and stores in a row took 7 us to get through.)
            constexpr int AHEAD = 4;
            const int c = tid % CPR;
#pragma unroll 1
            for (int base = 0; base < part.rows; base += SOFT / CPR * AHEAD) {  // as often in every thread
                uint4 x[AHEAD];
#pragma unroll
                for (int b = 0; b < AHEAD; ++b) {
                    int tok, head;
                    row_of<S>(p, cur, min(base + tid / CPR + b * (SOFT / CPR), part.rows - 1), tok, head);
                    x[b] = uint4{0, 0, 0, 0};  // also values behind the head's own
                    if (c * 8 < p.dim)
                        x[b] = *reinterpret_cast<const uint4*>(static_cast<const C*>(p.q) + (int64_t)tok * p.q_stride +
                                                               (int64_t)head * p.dim + c * 8);
                }
                __syncwarp();
                if (!started) named_bar_arrive(4, SOFT + 64);  // the tiles' copies queue up behind them
                started = true;
#pragma unroll
                for (int b = 0; b < AHEAD; ++b) {
                    // a negative scale turns the sign of every value, zero makes it zero
                    x[b].x = (x[b].x & q_and) ^ q_xor, x[b].y = (x[b].y & q_and) ^ q_xor;
                    x[b].z = (x[b].z & q_and) ^ q_xor, x[b].w = (x[b].w & q_and) ^ q_xor;
                    const int r = base + tid / CPR + b * (SOFT / CPR);
                    if (r < part.rows) *reinterpret_cast<uint4*>(q_mem + swizzled<MT>(r, c)) = x[b];
                }
            }
            if (lane_row == 0) sh.keep[w] = 0;
            // The issuing warp orders these writes, as those of cp.async, before
            // the tensor core's reads: it fences after it has seen their arrival.
            mbar_arrive(&sh.q_full);

            float m = NONE, l = 0.f;
            bool begun = false;
            // the products of the stream's tile `t` have reached the sums
            auto sums_done = [&](int t) {
                const int i = S::STREAMS == 2 ? w : t & 1;
                ring_wait(sh, &sh.o_full[i], ot[i] ^ 1, p.status);
                __syncwarp();
                tm_fence_after();
            };
            for (int t = part.both ? 0 : w; t < part.tiles; t += part.both || S::STREAMS == 1 ? 1 : 2) {
                const int meta = (count + t) % S::META, pos0 = (cur.tile + t) * TN;
                const int buf = S::STREAMS == 2 ? w : t & 1;
                const uint32_t s_at = tm_lane + buf * TN;
                ring_wait(sh, &sh.s_full[buf], st[buf], p.status);
                st[buf] ^= 1;
                __syncwarp();
                tm_fence_after();
                const bool whole = *(volatile int*)&sh.whole[meta];
                if (pos0 + TN > cur.w.ctx) {  // by the lengths: barriers depend on it, also after a wait that ran out
                    // A draft that some row does not see must not reach that
                    // row's sums: the products would make NaN of 0 times an
                    // infinity. Rows of V that hold one become zero in the ring
                    // and are added below. The tile's streams look together.
                    const int vn = count + t;
                    ring_wait(sh, &sh.v_full[vn % S::V_STAGES], vn / S::V_STAGES & 1, p.status);
                    __syncwarp();
                    const uint32_t v_at = v_ring + vn % S::V_STAGES * S::TILE;
                    bool b = false;
                    if ((!part.both || w == 0) && lane_row < TN && pos0 + lane_row >= cur.w.ctx) {
                        constexpr uint32_t ex = S::TC == BH_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll 2
                        for (int i = 0; i < CPR; ++i) {
                            uint4 v;
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                         : "r"(v_at + swizzled<TN>(lane_row, i)));
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t u = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
                                b = b || (u & ex) == ex || (u >> 16 & ex) == ex;
                            }
                        }
                        if (b) {
#pragma unroll 1
                            for (int i = 0; i < CPR; ++i)
                                asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(v_at + swizzled<TN>(lane_row, i)), "r"(0) : "memory");
                            fence_proxy_async_smem();
                        }
                    }
                    const uint32_t any = __ballot_sync(0xffffffffu, b);
                    if (lane == 0 && (!part.both || w == 0) && (warp & 3) < NC) sh.bad[part.both || S::STREAMS == 1 ? t & 1 : w][warp & 3] = any;
                    if (part.both) sync();
                    else named_bar(2 + w, 128);
                }
                if (warp_live) {
                    uint32_t vis[NC];
                    uint32_t bad_any = 0;
                    const volatile uint32_t* bad = sh.bad[part.both || S::STREAMS == 1 ? t & 1 : w];
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            const int rel = pos0 + 32 * c - cur.w.ctx;  // the first column's draft
                            uint32_t bits = ~0u;
                            if (rel > -32)
                                bits = rel >= 64 ? 0u : rel >= 0 ? (uint32_t)(see >> rel) : (uint32_t)(see << -rel) | ((1u << -rel) - 1);
                            if (pos0 + TN > cur.w.ctx) bad_any |= bad[c];
                            vis[c] = bits & *(volatile uint32_t*)&sh.valid[meta][c];
                        }
                        __syncwarp();
                    }
                    uint32_t x[NC][32];
#pragma unroll
                    for (int c = 0; c < NC; ++c) tm_load(x[c], s_at + c * 32);
                    tm_wait_ld();
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < NC; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!(vis[c] >> i & 1)) x[c][i] = 0xff800000u;
                    }
                    float tops[4] = {m, m, m, m};
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            tops[i / 2 & 3] = max3(tops[i / 2 & 3], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
                    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    const bool grow = my < part.rows && (top - m) * rs > 8.f;  // also from nothing to something
                    float alpha = 1.f;
                    if (grow) {
                        alpha = ex2((m - top) * rs);
                        m = top;
                        l *= alpha;
                    }
                    if (begun && __any_sync(0xffffffffu, grow)) {
                        sums_done(t - 1);
#pragma unroll 1
                        for (int c = 0; c < DP / 8; ++c) {
                            uint32_t o[8];
                            tm_load8(o, o_at + c * 8);
                            tm_wait_ld();
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tm_store8(o_at + c * 8, o);
                        }
                        tm_wait_st();
                    }
                    const float base = m == NONE ? 0.f : m, shift = S::OFF - base * rs;
                    const uint64_t rs2 = pair(rs, rs), shift2 = pair(shift, shift);
                    uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        uint32_t y[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float a, b;
                            unpair(fma2(pair(__uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1])), rs2, shift2), a, b);
                            a = ex2(a);
                            b = ex2(b);
                            sum[i / 2 & 3] = add2(sum[i / 2 & 3], pair(a, b));
                            y[i / 2] = pack2<C>(a, b);
                        }
                        tm_store16(s_at + c * 16, y);  // in the scores' own place, which has been read
                    }
                    float la, lb;
                    unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), la, lb);
                    l += la + lb;
                    tm_wait_st();
                    if (bad_any) {
                        // rows of V that the ring holds as zeros, from memory, before the tile's products
                        if (begun) sums_done(t - 1);
                        else {
                            uint32_t z[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) z[i] = 0;
                            for (int c = 0; c < DP / 32; ++c) tm_store(o_at + c * 32, z);
                            tm_wait_st();
                            *(volatile int*)&sh.keep[w] = 1;
                        }
                        for (int r = max(0, cur.w.ctx - pos0); r < TN; ++r) {
                            if (!(bad[r / 32] >> (r & 31) & 1)) continue;
                            const uint32_t pos = (uint32_t)(pos0 + r), blk = p.block.div(pos);
                            const int32_t id = p.tables[(int64_t)cur.seq * p.max_blocks + blk];
                            const int64_t at = id * p.kv.block_stride + (pos - blk * p.kv.block_size) * p.kv.token_stride +
                                               cur.head * p.kv.head_stride;
                            const C* v = static_cast<const C*>(p.kv.v) + at;
                            const C* k = static_cast<const C*>(p.kv.k) + at;
                            const bool mine = see >> (pos - cur.w.ctx) & 1;
                            // the score again: its place holds probabilities now
                            float x = 0.f;
                            if (mine) {
                                const C* q = static_cast<const C*>(p.q) + (int64_t)my_tok * p.q_stride + (int64_t)my_head * p.dim;
                                for (int d = 0; d < p.dim; ++d) x = __fmaf_rn(to_f32(q[d]) * turn_q, to_f32(k[d]), x);
                            }
                            const float pr = mine ? ex2(__fmaf_rn(x, rs, shift)) : 0.f;
                            __syncwarp();
                            for (int c = 0; c < DP / 32; ++c) {
                                uint32_t o[32];
                                tm_load(o, o_at + c * 32);
                                tm_wait_ld();
                                if (mine) {
#pragma unroll
                                    for (int i = 0; i < 32; ++i)
                                        if (c * 32 + i < p.dim)
                                            o[i] = __float_as_uint(__fmaf_rn(pr, to_f32(v[c * 32 + i]), __uint_as_float(o[i])));
                                }
                                __syncwarp();
                                tm_store(o_at + c * 32, o);
                                tm_wait_st();
                            }
                        }
                    }
                }
                begun = true;
                tm_fence_before();
                mbar_arrive(&sh.p_full[buf]);
                ot[buf] ^= 1;
            }
            if (begun) sums_done(part.tiles - 1);
            const int rows = part.rows;
            float* swap = reinterpret_cast<float*>(q_mem);  // the query rows have served
            auto swap_at = [&](int c) { return swap + lane_row * DP + ((c ^ lane_row & (DP / 4 - 1)) << 2); };
            float m1 = NONE, l1 = 0.f;
            if (S::STREAMS == 2 && !part.both) {
                // the second stream's rows to the first
                if (w == 1) sh.part_m[lane_row] = m, sh.part_l[lane_row] = l;
                sync();
                if (w == 1 && warp_live && begun) {
#pragma unroll 1
                    for (int c = 0; c < DP / 32; ++c) {
                        uint32_t x[32];
                        tm_load(x, o_at + c * 32);
                        tm_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4*>(swap_at(c * 8 + i)) = uint4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
                    }
                }
                sync();
                if (part.tiles > 1) m1 = sh.part_m[lane_row], l1 = sh.part_l[lane_row];
            }
            const bool complete = cur.first >= f0 && part.ends;
            float* const slot = part_slot<S>(p, blockIdx.x, cur.first >= f0);
            if (warp_live && (part.both || w == 0)) {
                const float top = fmaxf(m, m1), base = top == NONE ? 0.f : top;
                const bool two = S::STREAMS == 2 && !part.both && part.tiles > 1;
                const float a0 = two ? ex2((m - base) * rs) : 1.f, a1 = two ? ex2((m1 - base) * rs) : 0.f;
                const float sum = __fmaf_rn(l, a0, l1 * a1);
                const float inv = !complete ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
                for (int d = 0; d < DP; d += 16) {
                    uint32_t x[16];
                    tm_load16(x, o_at + d);
                    tm_wait_ld();
                    if (my < rows) {
                        float y[16];
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            float4 z{0.f, 0.f, 0.f, 0.f};
                            if (two) z = *reinterpret_cast<const float4*>(swap_at((d + i) / 4));
                            y[i] = __fmaf_rn(__uint_as_float(x[i]), a0, z.x * a1) * inv;
                            y[i + 1] = __fmaf_rn(__uint_as_float(x[i + 1]), a0, z.y * a1) * inv;
                            y[i + 2] = __fmaf_rn(__uint_as_float(x[i + 2]), a0, z.z * a1) * inv;
                            y[i + 3] = __fmaf_rn(__uint_as_float(x[i + 3]), a0, z.w * a1) * inv;
                        }
                        if (complete) {
                            C* to = static_cast<C*>(p.out) + (int64_t)my_tok * p.out_stride + (int64_t)my_head * p.dim + d;
#pragma unroll
                            for (int i = 0; i < 16; i += 8) {
                                const uint4 v{pack2<C>(y[i], y[i + 1]), pack2<C>(y[i + 2], y[i + 3]), pack2<C>(y[i + 4], y[i + 5]),
                                              pack2<C>(y[i + 6], y[i + 7])};
                                if (d + i < p.dim) *reinterpret_cast<uint4*>(to + i) = v;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i += 4)
                                *reinterpret_cast<float4*>(slot + part_value<S>(my, d + i)) = float4{y[i], y[i + 1], y[i + 2], y[i + 3]};
                        }
                    }
                    __syncwarp();
                }
                if (my < rows) {
                    if (!complete) slot[my] = top, slot[MT + my] = sum, slot[2 * MT + my] = rs;
                    else if (p.lse) p.lse[(int64_t)my_tok * p.n_head + my_head] = log_sum(top, rs, S::OFF, sum);
                }
            }
            sync();  // the next query rows take their place
            count += part.tiles;
            const bool is_split = cur.first >= f0 && !part.ends;
            if (!next_part<S>(cur, p, f1)) {
                if (tid == 0) leave_split<S>(p, cur, is_split, per);
                break;
            }
        }
    }
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    if (warp == MMA_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "n"(S::COLUMNS));
}

// cuTensorMapEncodeTiled through the runtime (the library does not link the
// driver), null where it has none; defined in tree_attention.cu.
typedef CUresult (*TensorMapEncoder)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                     const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                     CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
TensorMapEncoder tensor_map_encoder();

// The cache's tensor map with boxes of 64 values x `box` tokens, and `box` (0:
// the block size has no factor of 8, or the strides fit no map).
inline int wide_map(CUtensorMap* map, const AttnParams& p, void* base, bool bf16, int most) {
    const uint32_t bs = p.kv.block_size;
    int box = (int)(bs & (~bs + 1));
    if (box > most) box = most;
    const TensorMapEncoder encode = tensor_map_encoder();
    if (box < 8 || !encode) return 0;
    // where there is one head or block its stride is never taken
    const int64_t token = p.kv.token_stride * 2, head = (p.n_kv > 1 ? p.kv.head_stride : p.kv.token_stride) * 2,
                  block = (p.kv.n_blocks > 1 ? p.kv.block_stride : p.kv.token_stride) * 2;
    if (token >= 1ll << 40 || head >= 1ll << 40 || block >= 1ll << 40) return 0;
    const cuuint64_t size[4] = {(cuuint64_t)p.dim, bs, (cuuint64_t)p.n_kv, p.kv.n_blocks};
    const cuuint64_t stride[3] = {(cuuint64_t)token, (cuuint64_t)head, (cuuint64_t)block};
    const cuuint32_t part[4] = {64, (cuuint32_t)box, 1, 1}, step[4] = {1, 1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base,
                                  size, stride, part, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? box
               : 0;
}

template <class S>
int launch_wide_shape(const AttnParams& p, int num_sms, cudaStream_t s) {
    static_assert(S::BYTES + sizeof(WideShared<S>) <= 227 * 1024, "an SM's shared memory holds a CTA");
    static_assert(S::CTAS * (S::BYTES + sizeof(WideShared<S>) + 1024) <= 228 * 1024, "an SM holds its CTAs");
    static_assert(S::CTAS * (2 * S::SLOT * sizeof(float) + sizeof(Split)) <= WS_CTAS_PER_SM * WS_CTA_BYTES, "partials fit the workspace");
    CUtensorMap k_map{}, v_map{};
    int box = wide_map(&k_map, p, p.kv.k, S::TC == BH_BF16, S::TN);
    if (box && !wide_map(&v_map, p, p.kv.v, S::TC == BH_BF16, S::TN)) box = 0;
    return launch_and_join<S, CUtensorMap, CUtensorMap, int>(&tree_attention_wide_kernel<S>, p, num_sms * S::CTAS, s, k_map,
                                                             v_map, box);
}

// One stream where its 128 rows hold every sequence's rows of a head, else two:
// 128 rows, 16 sequences up to 32768 long, heads of 128 values, 204 us (two
// streams 209), 160 rows 252 us (one stream in two row tiles 255).
template <int TC, int DP>
int launch_wide(const AttnParams& p, int num_sms, cudaStream_t s) {
    if (p.max_new * (int)p.group.d <= 128) return launch_wide_shape<WideShape<TC, DP, 1>>(p, num_sms, s);
    return launch_wide_shape<WideShape<TC, DP, 2>>(p, num_sms, s);
}

// Either kernel, of 16-bit types: up to 16 rows of a head fill one row tile of
// mma.sync, whose row tiles begin and end sooner. bf16, 8 heads of 128 values, 16
// rows: 8 sequences up to 1000 long 22.7 us (wide 28.5), 24 up to 12000 133 us
// (wide 114; 8 rows 116); heads of 64: 19 and 80 us (wide 88 of the long). 20
// rows, 24 sequences: wide 114 us, mma.sync 138, and 32 rows 116 and 187.
template <int TC>
int launch_attention_16bit(const AttnParams& p, int num_sms, cudaStream_t s) {
    const int rows = p.max_new * (int)p.group.d;
    if (rows > 16 && p.dim <= 64) return launch_wide<TC, 64>(p, num_sms, s);
    if (rows > 16 && p.dim <= 128) return launch_wide<TC, 128>(p, num_sms, s);
    return launch_attention<TC, TC>(p, num_sms, s);
}

}  // namespace bh
