// attn_tile.cu -- attention of many query rows over one stretch of the paged
// KV cache: token runs that attend causally, and sequences that share a prefix.
//
// A query row of context length L attends o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(q . k_j / 16 - m) over what attended_range(L) keeps, then
// o *= sigmoid(gate).
//
// A CTA takes a tile of up to 32 tokens (or sequences) x the 4 query heads of
// one kv head = 128 rows, and walks position tiles of K and V:
//   S = Q K^T   tcgen05, A and B from shared memory
//   P = exp2(S c - m c + 7)   8 warps, two per 32 rows, S and P in TMEM
//   O += P V    tcgen05, A from TMEM, B from shared memory
// so that K and V are read once for all 128 rows.  TMEM holds O (256 columns)
// and two S buffers: the score product of tile j + 1 runs while the softmax
// warps work on tile j; P takes the place of its own S.  Chunks lie at arbitrary
// addresses, which a tensor map cannot span, so producer warps copy K and V with
// cp.async (or turn q8_0 blocks into f16) into a ring of stages in the 128-byte
// swizzled layout, a stage a K or a V tile.
//
// What the ring holds decides the speed: a V tile waits in it for its softmax,
// and the rest has to cover the latency of L2 or HBM.  Hence
//   single CTAs   64 positions a tile; 5 stages of 32 KB beside Q (64 KB);
//   CTA pairs     (runs of more than 32 tokens) 256 rows share one K/V tile of
//                 128 positions, each CTA holding half of it (cta_group::2): half
//                 the L2 reads and twice the tiles in the ring.
// f32 calls (HL) carry q and p as f16 hi + lo pairs, two products each, ~22
// bits: 0.3e-6 to 3e-6 of the output in the 2-norm, over q8_0 up to 4.3e-6 (plain
// f32 0.4e-6 to 3.5e-6).  Q's lo half sits in TMEM for single CTAs, where
// 64-position S buffers leave 128 columns and the ring keeps its size; for pairs, bound by the products
// and so better off with 128 positions a product, beside Q (3 stages remain).
// q8_0 values d * code (18 bits) then enter as hi + lo stages as well.  f16 calls
// round p to f16 once, and q8_0 values once, the rounding their type implies.
//
// The running maximum is lazy: O is rescaled only when a row's maximum grows by
// more than 2^8 over the one in use, so P reaches at most 2^15 (its 2^7 offset
// keeps small probabilities out of f16's denormals).  Sums and O are f32; O leaves
// TMEM in pieces (kAwayF32), as the tensor cores truncate what they add.
//
// Work is split along the positions where there are few row tiles; the parts'
// (m, l, O) go through the workspace and attn_join_kernel merges them.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "kvcache.cuh"
#include "ops.h"
#include "tc.cuh"

namespace qw35 {

namespace {

constexpr int TM_ROWS = 128;             // rows of a CTA: 32 tokens x 4 heads
constexpr int TM_TOK = TM_ROWS / AGRP;   // tokens (sequences) of a CTA
constexpr int SOFT_WARPS = 8;
constexpr uint32_t QBYTES = TM_ROWS * AHD * 2;
constexpr int kPlanSMs = 148;
constexpr int kPlanTile = 128;           // positions by which work is divided: a whole number of any variant's tiles
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kShift = 7.0f, kSlack = 8.0f;  // log2: offset of P, growth of the maximum before O is rescaled
constexpr float kNoScore = -3.0e38f;  // the maximum that a part leaves which has values but no finite score (an empty one: -infinity)

// Positions that one O in TMEM sums up before the softmax warps put it away, adding it, rounded to nearest, to the row's sum
// in the workspace, and the next product starts anew.  The tensor cores' adder truncates, step by step of 16 positions and
// operand half.  f32 in one chain: off by 2.1e-5 (2-norm) after 8,192 positions, by 8.7e-5 after 32,768 (q8_0 17e-5); in
// pieces 6e-6 (10e-6), with what was cut added back 3e-6 (4e-6).  For that a prompt of 4,096 takes 317 us instead of 296, of 8,192 853 instead
// of 779, of 32,768 13.0 ms instead of 12.4; pieces of 1,024 (1.5e-6) took 64 tokens at 32,704 from 64 us to 70.  f16 has
// half the steps and 24e-5 of its own rounding, so its pieces are longer.  Parts no longer than a piece take a kernel that
// cannot put away (AWAY false): f16 8192 tokens 435 us against 443 with one that can.
constexpr int kAwayF32 = 2048, kAwayF16 = 65536;

// A step of 16 products cuts 0 to 2^-23 of the sum so far, 0.72 x 2^-24 on average over mantissas, which is added back.  For
// O the row's probabilities tell how far the sum had come at each step, and whether its products reach the sum's last place
// at all (2^-24 each of it; the lo halves are 2^-11 of that): where they do not, nothing is cut.  A constant half of the
// steps was off by 5.6e-6 behind a first position with all the weight.  A score is taken to be half there on average.
constexpr float kCut = 4.3e-8f, kFelt = 0x1p-20f;

template <bool HL, bool Q8, bool PAIR>
struct TileGeo {
    static constexpr int CTAS = PAIR ? 2 : 1;
    static constexpr int TK = PAIR ? 128 : 64;           // positions of a tile; divides a chunk
    static constexpr int KR = TK / CTAS;                 // positions of K a CTA holds
    static constexpr int VP = 32 / CTAS;                 // 16-byte pieces of a V row a CTA holds
    static constexpr uint32_t STAGE = (uint32_t)TK * AHD * 2 / CTAS;
    static constexpr bool LO_SMEM = HL && PAIR, LO_TMEM = HL && !PAIR;  // where Q's lo half is
    static constexpr uint32_t QB = LO_SMEM ? 2 * QBYTES : QBYTES;
    static constexpr int NST = LO_SMEM ? 3 : 5;          // stages: what 227 KB hold beside Q
    // f16 planes: four warps issue the copies; q8_0: eight convert, each an eighth of a stage (at six, with two
    // batches for some, a stage took 1.7 us and the products waited)
    static constexpr int LOADERS = Q8 ? 8 : 4;
    // f16 over q8_0: 18 warps leave 96 registers a thread and softmax needs more (8192-token prompt 607 us with the split,
    // 673 without).  f32 over q8_0 spills 50 to 160 bytes of a thread at 96 and has not been measured with a split.  The 14
    // warps over f16 planes have 128 (449 us; split 463).
    static constexpr bool SPLIT = Q8 && !HL;
    static constexpr int THREADS = (SOFT_WARPS + LOADERS + (SPLIT ? 4 : 2)) * 32;  // and products, relay (two idle: whole groups of four)
    // registers a thread of softmax warps, loaders and the last four warps, within the launch's 96 a thread
    static constexpr int SOFT_REGS = 136, LOAD_REGS = 80, REST_REGS = 48;
    static_assert(!SPLIT || SOFT_WARPS * SOFT_REGS + LOADERS * LOAD_REGS + 4 * REST_REGS <= THREADS / 32 * 96, "registers");
    static constexpr int PARTS = HL && Q8 ? 2 : 1;       // stages of a tile: values, or their hi and lo halves
    static constexpr uint32_t RING = NST * STAGE, SMEM = QB + RING;
    static constexpr uint32_t S0 = 256;                  // TMEM columns: O, then the S buffers, then (LO_TMEM) Q's lo half
    static constexpr int STEPS = HL ? (Q8 ? 3 : 2) : 1;  // products of 16 positions onto O
    static constexpr int AWAY = (HL ? kAwayF32 : kAwayF16) / TK;  // tiles after which O is put away
    // a lo half bound for TMEM passes through the last 64 KB of the ring
    static constexpr int FREE_AT_START = LO_TMEM ? (int)((RING - QBYTES) / STAGE) : NST;
};

struct TilePlan {
    int pair;       // row tiles of two CTAs
    int tiles;      // row tiles (upper bound)
    int ns;         // position splits of a row tile (upper bound)
    int own_tiles;  // shared prefixes: sequences with a tail of their own, else 0
    int ns_own;     // position splits of a tail (upper bound)
    int each;       // kPlanTile tiles of a split
    int room;       // the workspace has room for O that is put away
};

constexpr uint32_t kQlo = 384;  // TMEM columns of the lo half of Q
constexpr int kMaxStages = 5;
struct __align__(16) TileShared {
    uint64_t full[kMaxStages], ready[kMaxStages], empty[kMaxStages];
    uint64_t s_full[2], p_full[2], pv_done, q_full, q_moved, o_full, looked;
    uint32_t tmem;
    int abort;
    int row0, nrow, kvh, table, part;  // this CTA's rows, kv head, chunk-table row, part number
    int lo, hi_max, hi_min, rs_max;    // positions [lo, hi) of the rows
    int hi_all, rs_all;                // of a pair: hi_min and rs_max over both CTAs
    int bad;                           // a V value that some row must not see is not finite
    int a0, n1, t2, begin, end;        // tile list: a0 .. a0+n1-1, then t2 ..; this CTA's share of it
    int hi[TM_TOK], sk[TM_TOK], rs[TM_TOK];
    float ex[2][2][TM_ROWS];           // row maxima (then sums) exchanged between the two column halves
};

template <bool SPLIT, int REGS, bool MORE>
__device__ __forceinline__ void set_regs() {
    if constexpr (!SPLIT) return;
    else if constexpr (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// ---- two CTAs ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// arrive on a CTA's copy of a barrier; MEM: this thread's (and its warp's) writes to memory go before it, else only
// what a tcgen05 fence orders
template <bool MEM>
__device__ __forceinline__ void arrive_at(uint64_t *bar, int rank) {
    if constexpr (MEM)
        asm volatile(
            "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\t"
            "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)), "r"(rank)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\t"
            "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)), "r"(rank)
            : "memory");
}
template <bool MEM>
__device__ __forceinline__ void arrive_leader(uint64_t *bar) { arrive_at<MEM>(bar, 0); }
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t *bar) {  // to both CTAs' copies
    if constexpr (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((unsigned short)3)
            : "memory");
    else
        tc_commit(bar);
}
// D (+)= A B with A from shared memory / from TMEM, one CTA or the pair
template <bool PAIR>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
    else
        tc_mma_f16(d, a, b, idesc, acc);
}
template <bool PAIR>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
    else
        tc_mma_f16_ts(d, a, b, idesc, acc);
}
template <bool PAIR>
__device__ __forceinline__ void tmem_take(uint32_t *dst) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(dst, 512);
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_give(uint32_t tmem) {
    if constexpr (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    else
        tmem_dealloc(tmem, 512);
}

// Bounded wait (2 s, as mbar_wait) that sees the other CTA's writes too; after one has run out, none waits any more.
__device__ __forceinline__ bool try_wait_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ void tw(uint64_t *bar, uint32_t parity, TileShared &s, unsigned code) {
    if (try_wait_cluster(bar, parity)) return;
    unsigned long long t0 = 0;
    while (!*(volatile int *)&s.abort) {
        for (int i = 0; i < 16; ++i)  // (a look at the clock costs more than one at the barrier)
            if (try_wait_cluster(bar, parity)) return;
        const unsigned long long t = globaltimer();
        if (t0 == 0) t0 = t;
        if (t - t0 > kTimeoutNs) {
            atomicOr(&g_dev_error, code);
            *(volatile int *)&s.abort = 1;
        }
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cpa16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// V stage as the B operand of O += P V: dims contiguous ("MN-major"), rows of 128 bytes (64 dims) per position,
// 128-byte swizzle; 64-dim blocks `block` bytes apart (LBO), 8-position groups 1 KB apart (SBO)
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr, uint32_t block) {
    const uint64_t d = smem_desc_sw128(saddr);
    return (d & ~((uint64_t)0x3FFFu << 16)) | ((uint64_t)(block >> 4) << 16);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = pack2(a, b);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    lo = pack2(a - f.x, b - f.y);
}

// 1 / (1 + e^-x): f32 to 2^-21 (expf 2 units, quotient 2^-22; sigmoid_f's exact division cost an epilogue 4 us), f16, by
// ex2 of a rounded argument, to 2^-18 at gates of -80.  0 below the smallest normal number (__fdividef by 2^126 and more),
// NaN for NaN: no clamp, which would take the bound for a NaN.
template <typename T>
__device__ __forceinline__ float sigmoid_fast(float x) {
    const float e = std::is_same<T, float>::value ? expf(-x) : ex2(-x * kLog2e);
    return __fdividef(1.0f, 1.0f + e);
}

// 8 consecutive values of a row, 16-byte aligned
__device__ __forceinline__ void get8(const float *p, float *v) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void get8(const __half *p, float *v) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = t.x;
        v[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ void put8(float *p, const float *v) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void put8(__half *p, const float *v) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
}
__device__ __forceinline__ void red_add4(float4 *p, const float *v) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
__device__ __forceinline__ int warp_min_i(int v) { return __reduce_min_sync(0xffffffffu, v); }
__device__ __forceinline__ int warp_max_i(int v) { return __reduce_max_sync(0xffffffffu, v); }

// Run (group) of row r, by one converged warp: the last u with off[u] <= r, if r < off[u + 1]; else -1.
__device__ __forceinline__ int run_of_row(const AttnTileArgs &p, int r) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int u = 0; u < p.n_run; u += 32) {
        const bool le = u + lane < p.n_run && p.off[u + lane] <= r;
        n += __popc(__ballot_sync(0xffffffffu, le));
    }
    return n > 0 && r < p.off[n] ? n - 1 : -1;
}

struct RunRows {
    int run, begin, end, len, row0;  // run (group), its rows, len[run] (or shared_len[run]), the tile's first row
};
// Row tile `tile` of `toks` rows -> its run, by one converged warp; run = -1 behind the last tile.  What is needed of
// a run is loaded in one go: the latency counts, not the bytes.
__device__ __forceinline__ RunRows find_tile(const AttnTileArgs &p, int tile, int toks) {
    const int lane = threadIdx.x & 31;
    const int32_t *lens = p.shared_len ? p.shared_len : p.len;
    int before = 0;
    for (int u = 0; u < p.n_run; u += 32) {
        const bool in = u + lane < p.n_run;
        const int a = in ? p.off[u + lane] : 0, b = in ? p.off[u + lane + 1] : 0, len = in ? lens[u + lane] : 0;
        const int n = b > a ? (b - a + toks - 1) / toks : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + sum > tile);
        if (hit) {
            const int w = __ffs(hit) - 1;
            const int first = a + (tile - (before + sum - n)) * toks;
            return RunRows{u + w, __shfl_sync(0xffffffffu, a, w), __shfl_sync(0xffffffffu, b, w),
                           __shfl_sync(0xffffffffu, len, w), __shfl_sync(0xffffffffu, first, w)};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return RunRows{-1, 0, 0, 0, 0};
}

// What this CTA does, by warp 0; false when there is no such unit (for both CTAs of a pair).
template <int CTAS, int TK>
__device__ __forceinline__ bool find_work(const AttnTileArgs &p, const TilePlan &pl, TileShared &s, int rank) {
    const int lane = threadIdx.x & 31;
    int id = blockIdx.x / CTAS, nrow = 0, ns = pl.ns, split, kvh;
    const int n_first = pl.tiles * AKV * pl.ns;
    const bool tail = id >= n_first;
    RunRows w{-1, 0, 0, 0, 0};
    if (!tail) {
        split = id % ns;
        kvh = (id / ns) % AKV;
        int tile = id / (AKV * ns);
        if (!p.shared_len) tile = pl.tiles - 1 - tile;  // the last tokens of a run have the most to do: first
        w = find_tile(p, tile, TM_TOK * CTAS);
        if (w.run >= 0) nrow = min(TM_TOK * CTAS, w.end - w.row0);
    } else {
        id -= n_first;
        ns = pl.ns_own;
        split = id % ns;
        kvh = (id / ns) % AKV;
        w.row0 = id / (AKV * ns);
        w.run = run_of_row(p, w.row0);
        if (w.run >= 0) {
            nrow = 1;
            w.len = p.shared_len[w.run];
        }
    }
    const int row0 = w.row0;
    if (w.begin < 0 || row0 < 0 || row0 + nrow > p.n_row) nrow = 0;  // (offsets that make no sense)
    // lane = token of the CTA's tile; a pair walks the positions that either of its tiles needs
    int lo = 0, hi_max = 0, rs_min = 0x7fffffff, sk_max = 0, hi_all = 0x7fffffff, rs_all = 0;
    for (int e = 0; e < CTAS; ++e) {
        const int tok = e * TM_TOK + lane;
        const bool real = tok < nrow;
        int hi = 0, sk = 0, rs = 0;
        if (real) {
            const int r = row0 + tok;
            int L = p.shared_len ? p.len[r] : w.len - (w.end - r) + 1;
            L = max(0, min(L, p.max_chunks * ACHUNK));
            int total;
            attended_range(L, p.window, p.sink, total, sk, rs);
            hi = L;
            if (p.shared_len) {
                const int sh = max(0, w.len);
                if (tail) lo = sh;
                else hi = min(L, sh);
            }
        }
        hi_max = max(hi_max, warp_max_i(hi));
        rs_min = min(rs_min, warp_min_i(real && hi > 0 ? rs : 0x7fffffff));
        sk_max = max(sk_max, warp_max_i(sk));
        const int hi_min = warp_min_i(real ? hi : 0x7fffffff), rs_max = warp_max_i(rs);
        hi_all = min(hi_all, hi_min);
        rs_all = max(rs_all, rs_max);
        if (e == rank) {
            s.hi[lane] = hi;
            s.sk[lane] = sk;
            s.rs[lane] = rs;
            if (lane == 0) {
                s.hi_min = hi_min;
                s.rs_max = rs_max;
            }
        }
    }
    lo = warp_max_i(lo);
    const int sk_end = min(sk_max, hi_max);
    const int end = (hi_max + TK - 1) / TK, a0 = lo / TK;
    const int a1 = sk_end > lo ? (sk_end + TK - 1) / TK : a0;
    int t2 = max(lo, min(rs_min, hi_max)) / TK, n1 = a1 - a0;
    if (a1 >= t2) {  // one stretch (always so without a window: rs_min is 0)
        n1 = 0;
        t2 = min(t2, a0);
    }
    const int total = hi_max > lo ? n1 + max(0, end - t2) : 0;
    if (lane == 0) {
        s.row0 = row0 + rank * TM_TOK;
        s.nrow = max(0, min(TM_TOK, nrow - rank * TM_TOK));
        s.kvh = kvh;
        s.table = p.shared_len ? (tail ? row0 : w.begin) : max(w.run, 0);
        s.part = tail ? pl.ns + split : split;
        s.lo = lo; s.hi_max = hi_max; s.hi_all = hi_all; s.rs_all = rs_all; s.bad = 0;
        s.a0 = a0; s.n1 = n1; s.t2 = t2;
        const int each = pl.each * (kPlanTile / TK);
        s.begin = min(total, split * each);
        s.end = split == ns - 1 ? total : min(total, (split + 1) * each);
    }
    return nrow > 0;
}

__device__ __forceinline__ int tile_at(const TileShared &s, int i) { return i < s.n1 ? s.a0 + i : s.t2 + (i - s.n1); }

// 8 codes of a q8_0 block (quarter j of the block at blk, 34 b bytes into its row) as they lie in memory: the
// codes start 2 or 0 bytes past a 4-byte border by the block's parity, and only the words they touch are read.  An
// even block's words hold its own d (first quarter) and the next block's (last quarter).
struct Q8Raw {
    uint32_t w0, w1, w2;
};
__device__ __forceinline__ Q8Raw q8_fetch(const uint8_t *blk, int j, bool odd) {
    Q8Raw r;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(blk + 2 + 8 * j - (odd ? 0 : 2));
    r.w0 = w[0];
    r.w1 = w[1];
    r.w2 = odd ? 0u : w[2];
    return r;
}
// The block's d, by the whole warp; piece c of a row in lane c (or c and 16 + c, of two rows)
__device__ __forceinline__ __half2 q8_scale(const Q8Raw &r, int c, bool odd) {
    const int lane = threadIdx.x & 31;
    const uint32_t v = __shfl_sync(0xffffffffu, (c & 7) == 3 ? r.w2 : r.w0, odd ? (lane & ~3) - 1 : lane & ~3);
    return __half2half2(__ushort_as_half((unsigned short)(odd ? v >> 16 : v)));
}
// d * code in f16: h rounded, l the remainder, exact (18 bits of product, 11 in h)
__device__ __forceinline__ void q8_halves(const Q8Raw &r, __half2 d, bool odd, uint4 &h, uint4 &l) {
    const uint32_t sh = odd ? 0u : 16u;
    const uint32_t x[2] = {__funnelshift_r(r.w0, r.w1, sh) ^ 0x80808080u, __funnelshift_r(r.w1, r.w2, sh) ^ 0x80808080u};
    const __half2 bias = __half2half2(__ushort_as_half((unsigned short)0x6480));
    uint32_t hw[4], lw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // bytes of code + 128 in halves 1024 + byte; - 1152 is exact
        const uint32_t v = __byte_perm(x[i >> 1], 0x64646464u, (i & 1) ? 0x4342u : 0x4140u);
        const __half2 q = __hsub2(*reinterpret_cast<const __half2 *>(&v), bias);
        const __half2 hi = __hmul2(q, d), lo = __hfma2(q, d, __hneg2(hi));
        hw[i] = *reinterpret_cast<const uint32_t *>(&hi);
        lw[i] = *reinterpret_cast<const uint32_t *>(&lo);
    }
    h = make_uint4(hw[0], hw[1], hw[2], hw[3]);
    l = make_uint4(lw[0], lw[1], lw[2], lw[3]);
}

__device__ __forceinline__ void sts16(uint32_t dst, const uint4 &v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ void lds16(uint32_t src, uint32_t *v) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src) : "memory");
}

// ---- producers ------------------------------------------------------------------
// Stages in the order in which the products consume them: K(0), then K(j + 1) before V(j).  A pair's CTA holds half
// of each: K by positions, V by dims.  Rows outside [lo, hi) (and of a chunk that is missing) come in as zeros.
struct TileRef {
    uint64_t plane;    // this layer's K or V plane of the chunk; 0: missing
    int pos0, row0;    // position and plane row of the stage's first row
    bool v;
};

template <bool HL, bool Q8, bool PAIR>
struct Loader {
    using G = TileGeo<HL, Q8, PAIR>;
    const AttnTileArgs &p;
    TileShared &s;
    uint32_t ring;
    int tid, rank, lo, hi, n, rs_all, hi_all, slot = 0;
    uint32_t phase = 1;  // parity that the slot's last release has; the first round waits for none

    __device__ __forceinline__ TileRef ref(int i) const {  // 0: K(0); 2 j + 1: K(j + 1); 2 j + 2: V(j); the last: V(n - 1)
        TileRef h;
        h.v = i == 2 * n - 1 || (i > 0 && !(i & 1));
        const int j = i == 2 * n - 1 ? n - 1 : (h.v ? i / 2 - 1 : (i + 1) / 2);
        const int t = tile_at(s, s.begin + j);
        const uint64_t base = p.chunk_ptrs[(size_t)s.table * p.max_chunks + t / (ACHUNK / G::TK)];
        h.plane = base ? base + (h.v ? p.v_off : p.k_off) : 0;
        h.pos0 = t * G::TK + (h.v ? 0 : rank * G::KR);
        h.row0 = s.kvh * ACHUNK + h.pos0 % ACHUNK;
        return h;
    }
    // A probability of 0 does not keep an infinity or NaN out of a product, so V tiles that some row does not see all
    // of are looked through; what is found sends the unit to attend_exactly().
    __device__ __forceinline__ bool some_masked(int pos0) const { return pos0 < rs_all || min(pos0 + G::TK, hi) > hi_all; }
    static __device__ __forceinline__ bool not_finite(const uint4 &v) {  // of 8 halves: an exponent of all ones
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) any |= (w[i] & 0x7c007c00u) + 0x04000400u;
        return (any & 0x80008000u) != 0;
    }
    __device__ __forceinline__ void report() {  // in both CTAs: each one's dims reach the other's rows
        *(volatile int *)&s.bad = 1;
        if constexpr (PAIR)
            asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.u32 [a], %2;\n\t}" ::"r"(
                             smem_u32(&s.bad)),
                         "r"(rank ^ 1), "r"(1)
                         : "memory");
    }
    // Once all loads are under way, from the cache again (looking tile by tile on the way cost a prompt 5%)
    __device__ __forceinline__ void look(int t) {
        const uint64_t base = p.chunk_ptrs[(size_t)s.table * p.max_chunks + t / (ACHUNK / G::TK)];
        if (base == 0) return;
        if constexpr (Q8) {
            for (int i = tid; i < G::TK * 8; i += G::LOADERS * 32) {  // the d of block i % 8 of a position
                const int pos = t * G::TK + i / 8;
                if (pos < lo || pos >= hi) continue;
                const uint8_t *row = reinterpret_cast<const uint8_t *>(base + p.v_off) + (size_t)(s.kvh * ACHUNK + pos % ACHUNK) * kKvQ8Row;
                const uint32_t d = *reinterpret_cast<const unsigned short *>(row + 34 * (i % 8)) & 0x7fffu;
                if (d >= 0x6000u) report();  // from 512 on, 127 d leaves the f16 range
            }
            return;
        }
        constexpr int RP = G::LOADERS * 32 / G::VP, N = G::TK / RP;
        const int r0 = tid / G::VP, pos0 = t * G::TK;
        const uint8_t *src = reinterpret_cast<const uint8_t *>(base + p.v_off) +
                             (size_t)(s.kvh * ACHUNK + pos0 % ACHUNK + r0) * (AHD * 2) + (rank * G::VP + tid % G::VP) * 16;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int pos = pos0 + r0 + i * RP;
            if (pos >= lo && pos < hi) bad |= not_finite(*reinterpret_cast<const uint4 *>(src + (size_t)i * RP * AHD * 2));
        }
        if (bad) report();
    }
    __device__ __forceinline__ void look_through() {  // (tiles ascend: what is masked lies at the ends of the list)
        int j = 0;
        for (; j < n && tile_at(s, s.begin + j) * G::TK < rs_all; ++j) look(tile_at(s, s.begin + j));
        for (int e = n - 1; e >= j && some_masked(tile_at(s, s.begin + e) * G::TK); --e) look(tile_at(s, s.begin + e));
    }
    // next free stage
    __device__ __forceinline__ int acquire(int stage) {
        const int k = slot;
        if (stage >= G::NST) tw(&s.empty[k], phase, s, 1u);
        else if (stage >= G::FREE_AT_START) tw(&s.q_moved, 0, s, 512u);
        if (++slot == G::NST) {
            slot = 0;
            phase ^= 1u;
        }
        return k;
    }

    // f16 planes: asynchronous copies of 16 bytes; the last to land signals the stage
    template <bool V>
    __device__ __forceinline__ void copy(const TileRef &h, int stage) {
        constexpr int PC = V ? G::VP : 32;  // pieces of a row of the stage
        constexpr int ROWS = V ? G::TK : G::KR, RP = G::LOADERS * 32 / PC, N = ROWS / RP;
        const int c = tid % PC, r0 = tid / PC;
        const uint8_t *src = reinterpret_cast<const uint8_t *>(h.plane) + (size_t)(h.row0 + r0) * (AHD * 2) + ((V ? rank * G::VP : 0) + c) * 16;
        const int k = acquire(stage);
        const uint32_t dst = ring + k * G::STAGE + (uint32_t)(c >> 3) * (ROWS * 128u);
        const int a = lo - h.pos0, b = (h.plane ? hi : 0) - h.pos0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = r0 + i * RP;
            const bool ok = r >= a && r < b;
            cpa16(dst + sw128_off(r, c & 7), ok ? static_cast<const void *>(src + (size_t)i * RP * AHD * 2) : p.q, ok);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&s.full[k])) : "memory");
    }

    // q8_0 planes: a warp takes 8 rows of K, or 8 (of a pair, 16 half) rows of V, a piece a lane and row; the words of
    // a stage are fetched while the one before it is converted
    enum : int { Q8_ROWS = 8 };
    __device__ __forceinline__ int piece(bool v) const { return v ? rank * G::VP + (tid & 31) % G::VP : tid & 31; }
    __device__ __forceinline__ int first_row(bool v) const {
        return (tid >> 5) * (v ? 8 * G::CTAS : 8) + (v && PAIR ? 8 * ((tid & 31) >> 4) : 0);
    }
    __device__ __forceinline__ void fetch(const TileRef &h, Q8Raw *raw) const {
        const int c = piece(h.v), r0 = first_row(h.v);
        const bool odd = (c >> 2) & 1;
        const uint8_t *src = reinterpret_cast<const uint8_t *>(h.plane) + (size_t)(h.row0 + r0) * kKvQ8Row + 34 * (c >> 2);
        const int a = lo - h.pos0 - r0, b = (h.plane ? hi : 0) - h.pos0 - r0;
        if (a <= 0 && b >= Q8_ROWS) {
#pragma unroll
            for (int i = 0; i < Q8_ROWS; ++i) raw[i] = q8_fetch(src + i * kKvQ8Row, c & 3, odd);
        } else {
#pragma unroll
            for (int i = 0; i < Q8_ROWS; ++i) raw[i] = i >= a && i < b ? q8_fetch(src + i * kKvQ8Row, c & 3, odd) : Q8Raw{0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ void convert(const TileRef &h, const Q8Raw *raw, int stage) {
        const int c = piece(h.v), cs = h.v ? c - rank * G::VP : c, r0 = first_row(h.v);
        const bool odd = (c >> 2) & 1;
        // (r0 is a multiple of 8: row r0 + i of an atom column has its pieces at c ^ i)
        const uint32_t at = (uint32_t)(cs >> 3) * (h.v ? G::TK * 128u : G::KR * 128u) + (uint32_t)(r0 >> 3) * 1024u + (uint32_t)(cs & 7) * 16u;
        const int k0 = acquire(stage * G::PARTS), k1 = HL ? acquire(stage * G::PARTS + 1) : 0;
        const uint32_t d0 = ring + k0 * G::STAGE + at, d1 = ring + k1 * G::STAGE + at;
#pragma unroll
        for (int i = 0; i < Q8_ROWS; ++i) {
            uint4 vh, vl;
            q8_halves(raw[i], q8_scale(raw[i], c, odd), odd, vh, vl);
            sts16((d0 ^ (i * 16u)) + i * 128u, vh);
            if constexpr (HL) sts16((d1 ^ (i * 16u)) + i * 128u, vl);
        }
        mbar_arrive(&s.full[k0]);
        if constexpr (HL) mbar_arrive(&s.full[k1]);
    }

    __device__ __forceinline__ void run() {
        if (n <= 0) return;
        if constexpr (Q8) {
            // (tile addresses come from memory, too: one stage further ahead)
            Q8Raw a[Q8_ROWS], b[Q8_ROWS];
            TileRef ha = ref(0), hb = ref(1);
            fetch(ha, a);
            for (int i = 0; i < 2 * n; i += 2) {
                fetch(hb, b);
                const TileRef hc = ref(min(i + 2, 2 * n - 1));
                convert(ha, a, i);
                if (i + 2 < 2 * n) fetch(hc, a);
                const TileRef hd = ref(min(i + 3, 2 * n - 1));
                convert(hb, b, i + 1);
                ha = hc;
                hb = hd;
            }
        } else {
            TileRef h = ref(0);
            for (int i = 0; i < 2 * n; ++i) {
                const TileRef next = ref(min(i + 1, 2 * n - 1));  // (its chunk address comes from memory)
                if (h.v) copy<true>(h, i);
                else copy<false>(h, i);
                h = next;
            }
        }
        look_through();
        if constexpr (!Q8) asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        if ((tid & 31) == 0) {
            mbar_arrive(&s.looked);
            if constexpr (PAIR) arrive_at<true>(&s.looked, rank ^ 1);
        }
    }
};

// ---- products (one warp; of a pair, the leader's) ------------------------------------
template <bool HL, bool Q8, bool PAIR, bool AWAY>
struct Products {
    using G = TileGeo<HL, Q8, PAIR>;
    TileShared &s;
    uint32_t q, ring, tmem;
    int slot = 0;
    uint32_t phase = 0;

    // stage `slot + ahead` is there (in both CTAs)
    __device__ __forceinline__ uint32_t stage(int ahead) {
        const int k = slot + ahead >= G::NST ? slot + ahead - G::NST : slot + ahead;
        tw(&s.ready[k], phase ^ (slot + ahead >= G::NST ? 1u : 0u), s, 2u);
        return ring + k * G::STAGE;
    }
    __device__ __forceinline__ void release() {
        if (elect_one()) commit<PAIR>(&s.empty[slot]);
        if (++slot == G::NST) {
            slot = 0;
            phase ^= 1u;
        }
    }
    // S = Q K^T; f32: the small products first, so that the accumulator is rounded at full size only 16 times
    __device__ __forceinline__ void scores(int j) {
        const uint32_t d = tmem + G::S0 + (j & 1) * G::TK;
        constexpr uint32_t idesc = idesc_f16_f32(TM_ROWS * G::CTAS, G::TK);
        const uint32_t k0 = stage(0), k1 = G::PARTS > 1 ? stage(1) : k0;
        const uint64_t kd0 = smem_desc_sw128(k0), kd1 = smem_desc_sw128(k1), qd = smem_desc_sw128(q);
        // descriptors hold addresses in units of 16 bytes: 32 bytes a step of 16 dims, a block every 64 dims
        auto kstep = [](int i) { return (uint64_t)((i >> 2) * (G::KR * 8) + (i & 3) * 2); };
        auto qstep = [](int i) { return (uint64_t)((i >> 2) * 1024 + (i & 3) * 2); };
        if (elect_one()) {
            if constexpr (HL) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if constexpr (G::LO_TMEM) mma_ts<PAIR>(d, tmem + kQlo + i * 8, kd0 + kstep(i), idesc, i > 0);
                    else mma_ss<PAIR>(d, qd + (QBYTES >> 4) + qstep(i), kd0 + kstep(i), idesc, i > 0);
                }
                if constexpr (Q8) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) mma_ss<PAIR>(d, qd + qstep(i), kd1 + kstep(i), idesc, 1);
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) mma_ss<PAIR>(d, qd + qstep(i), kd0 + kstep(i), idesc, HL || i > 0);
            commit<PAIR>(&s.s_full[j & 1]);
        }
        __syncwarp();
        for (int e = 0; e < G::PARTS; ++e) release();
    }
    // O += P V
    __device__ __forceinline__ void values(int j) {
        const uint32_t pa = tmem + G::S0 + (j & 1) * G::TK;
        constexpr uint32_t idesc = idesc_f16_f32(TM_ROWS * G::CTAS, AHD) | (1u << 16);  // B MN-major
        const uint32_t v0 = stage(0), v1 = G::PARTS > 1 ? stage(1) : v0;
        const uint64_t vd0 = desc_v(v0, G::TK * 128u), vd1 = desc_v(v1, G::TK * 128u);
        const bool on = AWAY ? j % G::AWAY > 0 : j > 0;  // onto what O holds
        if (elect_one()) {
#pragma unroll
            for (int i = 0; i < G::TK / 16; ++i) {  // 16 positions: 2048 bytes on
                if constexpr (HL) mma_ts<PAIR>(tmem, pa + G::TK / 2 + i * 8, vd0 + i * 128, idesc, on || i > 0);
                if constexpr (HL && Q8) mma_ts<PAIR>(tmem, pa + i * 8, vd1 + i * 128, idesc, 1);
                mma_ts<PAIR>(tmem, pa + i * 8, vd0 + i * 128, idesc, HL || on || i > 0);
            }
            commit<PAIR>(&s.pv_done);
        }
        __syncwarp();
        for (int e = 0; e < G::PARTS; ++e) release();
    }
    __device__ __forceinline__ void run() {
        const int n = s.end - s.begin;
        if (n <= 0) return;
        tw(&s.q_full, 0, s, 4u);
        tc_fence_after();
        scores(0);
        for (int j = 0; j < n; ++j) {
            if (j + 1 < n) scores(j + 1);  // into the buffer whose P the product before last has consumed, in order
            tw(&s.p_full[j & 1], (uint32_t)(j >> 1) & 1u, s, 8u);
            tc_fence_after();
            values(j);
        }
        if (elect_one()) commit<PAIR>(&s.o_full);
        __syncwarp();
        // after a timeout nobody else may be waiting: let the products end before TMEM is freed
        if (*(volatile int *)&s.abort) mbar_wait(&s.o_full, 0, 16u);
    }
};

// A thread of each CTA makes the producers' ordinary writes, seen through `full`, visible to the products and tells
// their warp: the fence costs the products' warp 0.1 us a stage otherwise.
template <bool HL, bool Q8, bool PAIR>
__device__ __forceinline__ void relay(TileShared &s, int rank) {
    using G = TileGeo<HL, Q8, PAIR>;
    const int n = 2 * G::PARTS * (s.end - s.begin);
    int slot = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n; ++i) {
        tw(&s.full[slot], phase, s, 2u);
        fence_async_smem();
        if (PAIR && rank) arrive_leader<true>(&s.ready[slot]);
        else mbar_arrive(&s.ready[slot]);
        if (++slot == G::NST) {
            slot = 0;
            phase ^= 1u;
        }
    }
}

// Row r of this CTA on the CUDA cores, from the cache itself and over the attended positions alone: the unit's values
// hold infinities or NaNs that the row may have to be kept from.  8 dims a lane; o unscaled, m in log2 units.
template <typename T, bool Q8>
__device__ __forceinline__ void attend_exactly(const AttnTileArgs &p, const TileShared &s, int r, int tk, float *o, float &m, float &l) {
    const int lane = threadIdx.x & 31, tok = r / AGRP;
    const int hi = s.hi[tok], sk = s.sk[tok], rs = s.rs[tok];
    const float c = p.scale * kLog2e;
    float q[8], k[8], v[8];
    get8(static_cast<const T *>(p.q) + ((size_t)(s.row0 + tok) * AH + s.kvh * AGRP + r % AGRP) * AHD + lane * 8, q);
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.0f;
    for (int j = s.begin; j < s.end; ++j) {
        const int t = tile_at(s, j);
        const uint64_t base = p.chunk_ptrs[(size_t)s.table * p.max_chunks + t * tk / ACHUNK];
        for (int pos = t * tk; pos < (t + 1) * tk; ++pos) {
            if (pos < s.lo || pos >= hi || (pos >= sk && pos < rs)) continue;
            const size_t row = (size_t)s.kvh * ACHUNK + pos % ACHUNK;
            auto values = [&](uint64_t plane, float *x) {  // (zeros of a chunk that is missing, as the tiles have them)
                if (base == 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
                } else if constexpr (Q8) {
                    const uint8_t *blk = reinterpret_cast<const uint8_t *>(plane) + row * kKvQ8Row + 34 * (lane >> 2);
                    const float d = __half2float(*reinterpret_cast<const __half *>(blk));
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = d * (float)(int8_t)blk[2 + 8 * (lane & 3) + i];
                } else {
                    get8(reinterpret_cast<const __half *>(plane) + row * AHD + lane * 8, x);
                }
            };
            values(base + p.k_off, k);
            values(base + p.v_off, v);
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) x = fmaf(q[i], k[i], x);
            x = warp_sum(x) * c;
            const float nm = fmaxf(m, x);
            // (before the first finite score l and o are 0, or NaN and have to stay so; nor may a weight of 0 hide one)
            const float a = m == -INFINITY ? 1.0f : ex2(m - nm), e = x == -INFINITY ? 0.0f : ex2(x - nm);
            l = l * a + e;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = o[i] * a + e * v[i];
            m = nm;
        }
    }
}

// ---- the kernel ---------------------------------------------------------------------
template <bool HL, bool Q8, bool PAIR, bool AWAY>
__global__ void __launch_bounds__(TileGeo<HL, Q8, PAIR>::THREADS, 1) attn_tile_kernel(AttnTileArgs p, TilePlan pl) {
    using G = TileGeo<HL, Q8, PAIR>;
    using T = typename std::conditional<HL, float, __half>::type;
    extern __shared__ __align__(1024) uint8_t smem[];
    TileShared &s = *reinterpret_cast<TileShared *>(smem + G::SMEM);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sbase = smem_u32(smem);
    const int rank = PAIR ? (int)cta_rank() : 0;
    constexpr int MMA_WARP = SOFT_WARPS + G::LOADERS;
    if (sbase & 1023u) {  // the swizzled layouts need 1024-byte aligned stages
        if (tid == 0) atomicOr(&g_dev_error, 256u);
        return;
    }
    int work = 0;
    if (warp == 0) work = find_work<G::CTAS, G::TK>(p, pl, s, rank);
    if (tid == 32) {
        for (int i = 0; i < G::NST; ++i) {
            mbar_init(&s.full[i], G::LOADERS * 32);
            mbar_init(&s.empty[i], 1);
            mbar_init(&s.ready[i], G::CTAS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], SOFT_WARPS * G::CTAS);
        }
        mbar_init(&s.pv_done, 1);
        mbar_init(&s.q_full, SOFT_WARPS * G::CTAS);
        mbar_init(&s.q_moved, SOFT_WARPS);
        mbar_init(&s.o_full, 1);
        mbar_init(&s.looked, G::LOADERS * G::CTAS);
        s.abort = 0;
        fence_barrier_init();
    }
    if (pl.ns + pl.ns_own > 1) pdl_trigger();  // (the join comes next)
    if (!__syncthreads_or(work)) return;
    if (s.begin == s.end && pl.ns + pl.ns_own > 1) {  // (both CTAs of a pair) nothing to attend in this part
        if (tid < s.nrow * AGRP) {
            const size_t g = (size_t)(s.row0 + tid / AGRP) * AH + s.kvh * AGRP + tid % AGRP;
            static_cast<float2 *>(p.ws)[g * (pl.ns + pl.ns_own) + s.part] = make_float2(-INFINITY, 0.0f);
        }
        return;
    }
    if (warp == MMA_WARP) tmem_take<PAIR>(&s.tmem);
    tc_fence_before();
    if constexpr (PAIR) cluster_sync();  // both CTAs' barriers exist
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;

    if (warp >= SOFT_WARPS && warp < MMA_WARP) {
        set_regs<G::SPLIT, G::LOAD_REGS, false>();
        Loader<HL, Q8, PAIR> ld{p, s, sbase + G::QB, tid - SOFT_WARPS * 32, rank, s.lo, s.hi_max, s.end - s.begin, s.rs_all, s.hi_all};
        ld.run();
    } else if (warp >= MMA_WARP) {
        set_regs<G::SPLIT, G::REST_REGS, false>();
        if (warp == MMA_WARP && rank == 0) {
            Products<HL, Q8, PAIR, AWAY> mm{s, sbase, sbase + G::QB, tmem};
            mm.run();
        } else if (warp == MMA_WARP + 1 && lane == 0) {
            relay<HL, Q8, PAIR>(s, rank);
        }
        __syncwarp();
    } else {
        set_regs<G::SPLIT, G::SOFT_REGS, true>();
        // softmax warps: row = TMEM lane; two groups of four, each a half of the columns (positions, then dims).
        // (Groups that take whole tiles in turn overlap better with each other, but each then holds an S buffer
        // twice as long, and with two buffers that is what the products wait for: 2.0 us a tile against 1.3.)
        const int quarter = warp & 3, grp = warp >> 2;
        const int row = quarter * 32 + lane, tok = row / AGRP;
        const bool real = tok < s.nrow;
        const bool busy = quarter * 32 / AGRP < s.nrow;  // some row of this warp is real
        const int n = s.end - s.begin;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        auto head_row = [&](int r) { return (size_t)(s.row0 + r / AGRP) * AH + s.kvh * AGRP + r % AGRP; };

        // stage Q: 16-byte pieces, 32 a row; a warp takes every eighth row, its loads first
        if (n > 0) {
            const T *qg = static_cast<const T *>(p.q) + lane * 8;
            const uint32_t qlo = sbase + (G::LO_TMEM ? G::SMEM - QBYTES : QBYTES);
            constexpr int NB = HL ? 8 : 16;  // rows a batch
            for (int r0 = warp; r0 < s.nrow * AGRP; r0 += SOFT_WARPS * NB) {
                uint4 v[16];
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const int r = r0 + i * SOFT_WARPS;
                    if (r < s.nrow * AGRP) {
                        const uint4 *src = reinterpret_cast<const uint4 *>(qg + head_row(r) * AHD);
                        if constexpr (HL) {
                            v[2 * i] = src[0];
                            v[2 * i + 1] = src[1];
                        } else {
                            v[i] = src[0];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const int r = r0 + i * SOFT_WARPS;
                    if (r >= s.nrow * AGRP) break;
                    const uint32_t dst = (lane >> 3) * 16384 + sw128_off(r, lane & 7);
                    if constexpr (HL) {
                        const float4 x = *reinterpret_cast<const float4 *>(&v[2 * i]), y = *reinterpret_cast<const float4 *>(&v[2 * i + 1]);
                        uint4 hi, lo;
                        split2(x.x, x.y, hi.x, lo.x);
                        split2(x.z, x.w, hi.y, lo.y);
                        split2(y.x, y.y, hi.z, lo.z);
                        split2(y.z, y.w, hi.w, lo.w);
                        sts16(sbase + dst, hi);
                        sts16(qlo + dst, lo);
                    } else {
                        sts16(sbase + dst, v[i]);
                    }
                }
            }
            fence_async_smem();
            if constexpr (G::LO_TMEM) {
                named_sync(9, SOFT_WARPS * 32);
                if (busy) {
#pragma unroll
                    for (int b = 0; b < 4; ++b) {  // 32 dims: 16 columns
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c = grp * 16 + b * 4 + i;
                            lds16(qlo + (c >> 3) * 16384 + sw128_off(row, c & 7), w + 4 * i);
                        }
                        tmem_st16(tmem + lanes + kQlo + grp * 64 + b * 16, w);
                    }
                    tmem_st_wait();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.q_moved);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR && rank) arrive_leader<true>(&s.q_full);
                else mbar_arrive(&s.q_full);
            }
        }

        const float c = p.scale * kLog2e * (1.0f + kCut * (AHD / 16 + 1) / 2);  // (lo products are too small to count)
        const int hi = real ? s.hi[tok] : 0x7fffffff, sk = real ? s.sk[tok] : 0, rs = real ? s.rs[tok] : 0;
        float m = -INFINITY, l = 0.0f;  // maximum in use; sum of this half's columns
        float way = 0.0f;               // sum of what l was at each step of this half's that O felt
        float gone = 0.0f;              // sum of both halves up to where O was put away
        constexpr int CW = G::TK / 2, NB = CW / 32;
        const int parts = pl.ns + pl.ns_own;
        float *acc = reinterpret_cast<float *>(static_cast<float2 *>(p.ws) + (size_t)p.n_row * AH * parts);
        float ma = -INFINITY;  // maximum in use when O was put away
        // Where this lane's 16 dims (16 b on) of O go, in four pieces: along its row or, for a full warp, in two heads' halves of
        // one of the warp's tokens, 512 bytes a store (a row a lane is 32 lines a store).  (Worked out where it is used: what
        // the tile loop would have to keep of it is spilled.)
        struct Place {
            float *at;
            int hop, half;
            __device__ __forceinline__ float4 *piece(int i) const { return reinterpret_cast<float4 *>(at + i / 2 * hop + i % 2 * half); }
        };
        auto place = [&](int b) {
            int r = row;
            asm volatile("" : "+r"(r));
            const int q = r & ~31, part = s.part;
            const bool full = q + 32 <= s.nrow * AGRP;
            const size_t h = head_row(full ? q + b / 2 * AGRP + b % 2 * 2 : r) * parts + part;
            return Place{acc + h * AHD + (full ? (r & 31) * 4 : b * 16), full ? parts * AHD : 8, full ? AHD / 2 : 4};
        };
        auto grown = [&]() { return ma == -INFINITY ? 1.0f : ex2((ma - m) * c); };  // (without a score so far: 0, or NaN and to stay so)
        // l becomes both halves' sum; what O is multiplied by for what was cut off it.  (No warp is in a tile: both rows of ex
        // are free.)
        auto both_halves = [&]() {
            s.ex[0][grp][row] = l;
            s.ex[1][grp][row] = way;
            named_sync(1 + quarter, 64);
            l += s.ex[0][grp ^ 1][row];
            way += s.ex[1][grp ^ 1][row];
            return l > 0.0f ? 1.0f + kCut * 2 * __fdividef(way, l) : 1.0f;  // (at a step either half is as far)
        };
        // O onto what was put away by additions in L2, which nothing waits for; no other thread has these values, so their
        // order is this one's.  Where a maximum grew since the last time, what is there takes its units first.
        auto put_away = [&](bool first) {
            const float f = first || !real ? 1.0f : grown(), whole = both_halves();
            if (__any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll 1
                for (int b = grp * 8; b < grp * 8 + 8 && real; ++b) {
                    const Place at = place(b);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 x = __ldcg(at.piece(i));
                        __stcg(at.piece(i), make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
                    }
                }
                __syncwarp();
            }
#pragma unroll 1
            for (int b = grp * 8; b < grp * 8 + 8; ++b) {
                const Place to = place(b);
                float o[16];
                tmem_ld16(tmem + lanes + b * 16, o);
                if (real) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] *= whole;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!first) red_add4(to.piece(i), o + 4 * i);
                        else __stcg(to.piece(i), make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
                    }
                }
                __syncwarp();
            }
            ma = m;
            gone += l;
            l = way = 0.0f;
            named_sync(1 + quarter, 64);  // (ex has been read)
        };
        auto tile = [&](int j) {
            const uint32_t sb = tmem + lanes + G::S0 + (j & 1) * G::TK;
            tw(&s.s_full[j & 1], (uint32_t)(j >> 1) & 1u, s, 32u);
            tc_fence_after();
            if (busy) {
                const int pos0 = tile_at(s, s.begin + j) * G::TK;
                const bool cut = pos0 < s.lo || pos0 + G::TK > s.hi_min || pos0 < s.rs_max;  // some row does not see all of it
                const int lo = s.lo;
                uint32_t u[NB][32];
                float mx = -INFINITY;
                tmem_ld32_async(sb + grp * CW, u[0]);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    tmem_ld_wait();
                    if (b + 1 < NB) tmem_ld32_async(sb + grp * CW + (b + 1) * 32, u[b + 1]);
                    if (cut) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int pos = pos0 + grp * CW + b * 32 + i;
                            if (pos >= hi || pos < lo || (pos >= sk && pos < rs)) u[b][i] = 0xff800000u;  // -inf
                        }
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(u[b][i]));
                    mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
                }
                s.ex[j & 1][grp][row] = mx;
                named_sync(1 + quarter, 64);  // also: both halves have read S, P may overwrite it
                mx = fmaxf(mx, s.ex[j & 1][grp ^ 1][row]);
                const bool grow = mx > m && (m == -INFINITY || (mx - m) * c > kSlack);
                if (__any_sync(0xffffffffu, grow)) {
                    const float nm = grow ? mx : m;
                    const float alpha = m == -INFINITY ? 0.0f : ex2((m - nm) * c);
                    if (j > 0) {
                        tw(&s.pv_done, (uint32_t)(j - 1) & 1u, s, 64u);
                        tc_fence_after();
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            uint32_t o[16];
                            const uint32_t ob = tmem + lanes + grp * 128 + b * 16;
                            tmem_ld16_async(ob, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st16(ob, o);
                        }
                    }
                    l *= alpha;
                    way *= alpha;
                    if (AWAY) gone *= alpha;
                    m = nm;
                }
                const float off = m == -INFINITY ? 0.0f : fmaf(m, c, -kShift);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t h[16];
                    [[maybe_unused]] uint32_t w[16];
                    float ls[2] = {0.0f, 0.0f};  // of the 16 positions of a step each
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float e0 = ex2(fmaf(__uint_as_float(u[b][2 * i]), c, -off));
                        const float e1 = ex2(fmaf(__uint_as_float(u[b][2 * i + 1]), c, -off));
                        ls[i >> 3] += e0 + e1;
                        if constexpr (HL) split2(e0, e1, h[i], w[i]);
                        else h[i] = pack2(e0, e1);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float at = fmaf(0.5f, ls[i], l);
                        if (ls[i] > kFelt * l) way += at;
                        if (G::STEPS > 1 && ls[i] > kFelt * 0x1p11f * l) way += (G::STEPS - 1) * at;
                        l += ls[i];
                    }
                    tmem_st16(sb + grp * (CW / 2) + b * 16, h);
                    if constexpr (HL) tmem_st16(sb + CW + grp * (CW / 2) + b * 16, w);
                }
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR && rank) arrive_leader<false>(&s.p_full[j & 1]);
                else mbar_arrive(&s.p_full[j & 1]);
            }
        };
        for (int j = 0, stop = 0; j < n;) {
            stop = AWAY ? min(n, stop + G::AWAY) : n;
            for (; j < stop; ++j) tile(j);
            if (AWAY && j < n && busy) {
                tw(&s.s_full[j & 1], (uint32_t)(j >> 1) & 1u, s, 32u);  // (so the product of j - 2 has ended: one parity bit tells j - 1)
                tw(&s.pv_done, (uint32_t)(j - 1) & 1u, s, 64u);
                tc_fence_after();
                put_away(j == G::AWAY);
            }
        }

        // O goes, scaled, to rows of the (free) ring and from there out coalesced, a warp per row; the gates of the
        // first rows are fetched before the last product ends
        const int rows = s.nrow * AGRP;
        const bool join = parts > 1;
        constexpr int EB = HL ? 4 : 8;  // rows a batch
        uint4 gates[EB][HL ? 2 : 1];
        auto fetch_gates = [&](int r0) {
            if (!p.gate || join) return;
#pragma unroll
            for (int i = 0; i < EB; ++i) {
                const int r = r0 + i * SOFT_WARPS;
                if (r < rows) {
                    const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(p.gate) + head_row(r) * AHD + lane * 8);
                    gates[i][0] = src[0];
                    if constexpr (HL) gates[i][1] = src[1];
                }
            }
        };
        fetch_gates(warp);
        if (n > 0) {
            tw(&s.o_full, 0, s, 128u);
            tw(&s.looked, 0, s, 128u);
            tc_fence_after();
        }
        float *buf = reinterpret_cast<float *>(smem);
        constexpr int BROW = AHD + 4;  // floats; 16-byte stores of 8 rows hit distinct banks
        const float whole = busy ? both_halves() : 1.0f;  // (of O's last piece)
        if (AWAY) l += gone;
        if (n > 0 && *(volatile int *)&s.bad) {
            for (int r = warp; r < rows; r += SOFT_WARPS) {
                float o[8], rm, rl;
                attend_exactly<T, Q8>(p, s, r, G::TK, o, rm, rl);
                const float inv = join ? 1.0f : (rl == 0.0f ? 0.0f : 1.0f / rl);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] *= inv;
                put8(buf + r * BROW + lane * 8, o);
                if (join && lane == 0) static_cast<float2 *>(p.ws)[head_row(r) * parts + s.part] = make_float2(fmaxf(rm, kNoScore), rl);
            }
        } else if (busy) {
            const float inv = join ? 1.0f : (l > 0.0f ? 1.0f / l : 0.0f);
            if (n > 0) {
                if (AWAY && n > G::AWAY) {
#pragma unroll 1
                    for (int b = grp * 8; b < grp * 8 + 8; ++b) {
                        const Place from = place(b);
                        const float f = grown();
                        float o[16];
                        float4 x[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (real) x[i] = __ldcg(from.piece(i));
                        __syncwarp();
                        tmem_ld16(tmem + lanes + b * 16, o);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<float4 *>(buf + row * BROW + b * 16 + 4 * i) =
                                make_float4(fmaf(x[i].x, f, o[4 * i] * whole) * inv, fmaf(x[i].y, f, o[4 * i + 1] * whole) * inv,
                                            fmaf(x[i].z, f, o[4 * i + 2] * whole) * inv, fmaf(x[i].w, f, o[4 * i + 3] * whole) * inv);
                    }
                } else {
                    const float times = whole * inv;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        float o[32];
                        tmem_ld32(tmem + lanes + grp * 128 + b * 32, o);
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<float4 *>(buf + row * BROW + grp * 128 + b * 32 + i) =
                                make_float4(o[i] * times, o[i + 1] * times, o[i + 2] * times, o[i + 3] * times);
                    }
                }
            }
            if (join && real && grp == 0)
                static_cast<float2 *>(p.ws)[head_row(row) * parts + s.part] = make_float2(m == -INFINITY ? kNoScore : fmaf(m, c, -kShift), l);
        }
        named_sync(9, SOFT_WARPS * 32);
        for (int r0 = warp; r0 < rows; r0 += SOFT_WARPS * EB) {
            if (r0 != warp) fetch_gates(r0);
#pragma unroll
            for (int i = 0; i < EB; ++i) {
                const int r = r0 + i * SOFT_WARPS;
                if (r >= rows) break;
                const size_t g = head_row(r);
                float y[8] = {};
                if (n > 0) get8(buf + r * BROW + lane * 8, y);
                if (join) {
                    if (n > 0) put8(acc + (g * parts + s.part) * AHD + lane * 8, y);
                    continue;
                }
                if (p.gate) {
                    float gv[8];
                    get8(reinterpret_cast<const T *>(&gates[i][0]), gv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] *= sigmoid_fast<T>(gv[e]);
                }
                put8(static_cast<T *>(p.out) + g * AHD + lane * 8, y);
            }
        }
    }
    tc_fence_before();
    if constexpr (PAIR) cluster_sync();  // (also: no CTA leaves while the other may still signal it)
    else __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_give<PAIR>(tmem);
    }
}

// Merges the parts of a (row, head): four warps take every fourth part, 8 dims a lane.  The loads of a warp's
// parts go out eight at a time: with few rows their latency is all there is.
constexpr int JOIN_WARPS = 4;
template <typename T>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attn_join_kernel(AttnTileArgs p, int parts) {
    const int row = blockIdx.x / AH, h = blockIdx.x % AH, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ __align__(16) float part_o[JOIN_WARPS][AHD];
    __shared__ float part_l[JOIN_WARPS];
    const bool mine = run_of_row(p, row) >= 0;
    const size_t g = (size_t)row * AH + h;
    float gv[8];
    if (warp == 0 && p.gate) get8(static_cast<const T *>(p.gate) + g * AHD + lane * 8, gv);
    pdl_wait();
    if (!mine) return;
    const float2 *ml = static_cast<const float2 *>(p.ws) + g * parts;
    const float *acc = reinterpret_cast<const float *>(static_cast<const float2 *>(p.ws) + (size_t)p.n_row * AH * parts) +
                       g * parts * AHD + lane * 8;
    float mx = -INFINITY;
    for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, ml[i].x);
    mx = warp_max(mx);
    float l = 0.0f, o[8] = {};
    constexpr int B = 8;
    for (int i0 = warp; i0 < parts; i0 += JOIN_WARPS * B) {
        float w[B], v[B][8];
        bool there[B];
#pragma unroll
        for (int k = 0; k < B; ++k) {
            const int i = i0 + k * JOIN_WARPS;
            there[k] = false;
            if (i < parts) {
                const float2 t = ml[i];
                if (t.x != -INFINITY) {  // (an empty part has no values)
                    there[k] = true;
                    w[k] = ex2(t.x - mx);
                    l = fmaf(w[k], t.y, l);
                    get8(acc + (size_t)i * AHD, v[k]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < B; ++k)
            if (there[k]) {  // (also with a weight of 0: it must not hide a NaN)
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = fmaf(w[k], v[k][e], o[e]);
            }
    }
    put8(&part_o[warp][lane * 8], o);
    if (lane == 0) part_l[warp] = l;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < JOIN_WARPS; ++w) {
        float t[8];
        get8(&part_o[w][lane * 8], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] += t[e];
        l += part_l[w];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        o[e] *= inv;
        if (p.gate) o[e] *= sigmoid_fast<T>(gv[e]);
    }
    put8(static_cast<T *>(p.out) + g * AHD + lane * 8, o);
}

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// The same plan for the workspace query and the launch.
TilePlan plan_for(int n_row, int n_run, int max_run, int max_len, int max_own, bool shared) {
    TilePlan pl{};
    // the most row tiles of `toks` tokens that the rows, divided into so many runs, can make
    const int runs = n_run < n_row ? n_run : n_row;
    auto row_tiles = [&](int toks) {
        const long long most = shared ? n_row : (long long)n_run * ceil_div(max_run, toks);
        return (int)std::min<long long>((n_row - runs) / toks + runs, most);
    };
    pl.tiles = row_tiles(TM_TOK);
    if (!shared) {
        // Pairs read and multiply with fewer pauses but take longer to set up: they pay from about two row tiles x
        // 128 positions an SM on.  f16, pairs against single CTAs: 4 runs of 64 tokens 13.8 against 11.4 us, 64
        // tokens at 4096 24.7 against 24.3, at 8128 28.1 against 31.2, at 32704 53.4 against 70.9, a prompt of 1024
        // 24.7 against 28.2, of 8192 441 against 601; f32 alike (64 tokens at 32704 62.7 against 74.8).
        const int kv = ceil_div(max_len, kPlanTile);
        pl.pair = max_run > TM_TOK && (long long)pl.tiles * AKV * kv > 2 * kPlanSMs;
        const int sms = kPlanSMs / (pl.pair ? 2 : 1);
        if (pl.pair) pl.tiles = row_tiles(2 * TM_TOK);
        const int units = pl.tiles * AKV;
        pl.ns = units >= sms ? 1 : sms / units;
        if (pl.ns > kv) pl.ns = kv;
        pl.each = ceil_div(kv, pl.ns);
        pl.ns = ceil_div(kv, pl.each);
        pl.room = pl.ns > 1 || max_len > kAwayF32;
        return pl;
    }
    // Shared prefixes.  Parts of one length: what one wave of CTAs would get each, a tail counting as its setup (a
    // tile's time) and half the longest.  Several groups may be much shorter than the longest, by which the host has
    // to plan, and leave SMs without a part: half the length then, two waves at most.
    const int kv = ceil_div(max_len, kPlanTile), kv_own = ceil_div(max_own, kPlanTile) + 1;
    const long long work = (long long)AKV * ((long long)pl.tiles * kv + (long long)n_row * (1 + kv_own / 2));
    const long long sms = (n_run > 1 ? 2 : 1) * kPlanSMs;
    pl.each = (int)std::min<long long>((work + sms - 1) / sms, std::max(kv, kv_own));  // (the quotient can pass 32 bits)
    pl.ns = kv > 0 ? ceil_div(kv, pl.each) : 1;
    pl.own_tiles = n_row;
    pl.ns_own = ceil_div(kv_own, pl.each);
    pl.room = 1;  // (a prefix and a tail: always joined)
    return pl;
}

size_t parts_bytes(int n_row, const TilePlan &pl) {
    const int parts = pl.ns + pl.ns_own;  // (f16 calls put away later than this allows for: the query has no type)
    return pl.room ? (size_t)n_row * AH * parts * (sizeof(float2) + AHD * sizeof(float)) : 256;
}

template <bool HL, bool Q8, bool PAIR, bool AWAY>
cudaError_t launch_one(const AttnTileArgs &a, const TilePlan &pl, cudaStream_t st) {
    using G = TileGeo<HL, Q8, PAIR>;
    auto kern = attn_tile_kernel<HL, Q8, PAIR, AWAY>;
    constexpr int smem = (int)(G::SMEM + sizeof(TileShared));
    static_assert(smem <= 227 * 1024, "stages and Q fit one SM");
    static_assert(G::NST <= kMaxStages, "a barrier for every stage");
    cudaError_t e = qw35h::smem_optin((const void *)kern, smem);
    if (e != cudaSuccess) return e;
    const long long grid = G::CTAS * ((long long)pl.tiles * AKV * pl.ns + (long long)pl.own_tiles * AKV * pl.ns_own);
    if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(G::THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = G::CTAS;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = PAIR ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a, pl);
}

template <bool HL, bool Q8, bool PAIR>
cudaError_t launch_tile(const AttnTileArgs &a, const TilePlan &pl, cudaStream_t st) {
    const bool away = pl.room && (long long)pl.each * kPlanTile > (HL ? kAwayF32 : kAwayF16);
    return away ? launch_one<HL, Q8, PAIR, true>(a, pl, st) : launch_one<HL, Q8, PAIR, false>(a, pl, st);
}

template <bool PAIR>
cudaError_t launch_type(const AttnTileArgs &a, const TilePlan &pl, cudaStream_t st) {
    return a.half ? (a.kv_q8 ? launch_tile<false, true, PAIR>(a, pl, st) : launch_tile<false, false, PAIR>(a, pl, st))
                  : (a.kv_q8 ? launch_tile<true, true, PAIR>(a, pl, st) : launch_tile<true, false, PAIR>(a, pl, st));
}

}  // namespace

size_t attn_tile_workspace_bytes(int n_row, int n_run, int max_run, int max_len, int max_own) {
    return parts_bytes(n_row, plan_for(n_row, n_run, max_run, max_len, max_own, max_run == 0));
}

cudaError_t attn_tile_run(const AttnTileArgs &a, cudaStream_t st) {
    if (a.n_row <= 0) return cudaSuccess;
    const TilePlan pl = plan_for(a.n_row, a.n_run, a.max_run, a.max_len, a.max_own, a.shared_len != nullptr);
    if (a.ws_bytes < parts_bytes(a.n_row, pl)) return cudaErrorInvalidValue;
    cudaError_t e = pl.pair ? launch_type<true>(a, pl, st) : launch_type<false>(a, pl, st);
    if (e != cudaSuccess) return e;
    const int parts = pl.ns + pl.ns_own;
    if (parts > 1) {
        // its launch, and the loads that do not depend on the parts, overlap the end of the kernel before
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)a.n_row * AH);
        cfg.blockDim = dim3(JOIN_WARPS * 32);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = getenv("QW35_NO_PDL") ? 0 : 1;
        e = a.half ? cudaLaunchKernelEx(&cfg, attn_join_kernel<__half>, a, parts)
                   : cudaLaunchKernelEx(&cfg, attn_join_kernel<float>, a, parts);
    }
    return e;
}

unsigned int attn_tile_error_read_and_clear() {
    unsigned int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(v));
    if (v) cudaMemcpyToSymbol(g_dev_error, &z, sizeof(z));
    return v;
}

}  // namespace qw35
