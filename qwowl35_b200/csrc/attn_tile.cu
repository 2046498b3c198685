// attn_tile.cu -- attention of many query rows over one stretch of the paged
// KV cache: token runs that attend causally, and sequences that share a prefix.
//
// A query row of context length L attends o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(q . k_j / 16 - m) over what attended_range(L) keeps, then
// o *= sigmoid(gate).
//
// One CTA takes a tile of up to 32 tokens (or sequences) x the 4 query heads of
// one kv head = 128 rows, and walks 128-position tiles of K and V:
//   S = Q K^T   128 x 128 x 256   tcgen05, A and B from shared memory
//   P = exp2(S c - m c + 7)       8 warps, two per 32 rows, S and P in TMEM
//   O += P V    128 x 256 x 128   tcgen05, A from TMEM, B from shared memory
// so that K and V are read once for all 128 rows.  TMEM holds O (256 columns)
// and two S buffers (128 each): the score product of tile j + 1 runs while the
// softmax warps work on tile j; P takes the place of its own S.  Chunks lie at
// arbitrary addresses, which a tensor map cannot span, so four producer warps
// copy K and V with cp.async (or turn q8_0 blocks into f16) into a ring of
// 32 KB stages in the 128-byte swizzled layout.
//
// The running maximum is lazy: O is rescaled only when a row's maximum grows by
// more than 2^8 over the one in use, so P reaches at most 2^15 (its 2^7 offset
// keeps small probabilities out of f16's denormals).  Sums and O are f32.
//
// f32 calls (HL) carry q and p as f16 hi + lo pairs, two products each, ~22
// bits; q8_0 values d * code (18 bits) then enter as hi + lo as well.  f16 calls
// round p to f16 once, and q8_0 values once, the rounding their type implies.
//
// Work is split along the positions where there are few row tiles; the parts'
// (m, l, O) go through the workspace and attn_join_kernel merges them.
#include <type_traits>

#include "kvcache.cuh"
#include "ops.h"
#include "tc.cuh"

namespace qw35 {

namespace {

constexpr int TM_ROWS = 128;             // rows of a tile: 32 tokens x 4 heads
constexpr int TM_TOK = TM_ROWS / AGRP;   // tokens (sequences) of a tile
constexpr int TK = 128;                  // positions of a K/V tile; divides a chunk
constexpr int SOFT_WARPS = 8, LOAD_WARPS = 4;
constexpr int TILE_THREADS = (SOFT_WARPS + LOAD_WARPS + 1) * 32;
constexpr uint32_t STAGE = 32768;        // 128 positions x 128 dims of K, or 64 x 256 of V
constexpr uint32_t QBYTES = TM_ROWS * AHD * 2;
constexpr int kPlanSMs = 148;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kShift = 7.0f, kSlack = 8.0f;  // log2: offset of P, growth of the maximum before O is rescaled

template <bool HL>
struct TileGeo {
    static constexpr int NST = HL ? 3 : 5;  // stages: what 227 KB hold beside Q (hi and lo)
    static constexpr int LAG = HL ? 1 : 2;  // copies of a producer thread in flight before it signals a stage
    static constexpr uint32_t QB = HL ? 2 * QBYTES : QBYTES;
    static constexpr uint32_t SMEM = QB + NST * STAGE;
};

struct TilePlan {
    int tiles;      // row tiles (upper bound)
    int ns;         // position splits of a row tile
    int own_tiles;  // shared prefixes: sequences with a tail of their own, else 0
    int ns_own;     // position splits of a tail
};

struct __align__(16) TileShared {
    uint64_t full[5], empty[5], s_full[2], p_full[2], pv_done, q_full, o_full;
    uint32_t tmem;
    int abort;
    int row0, nrow, kvh, table, part;  // this CTA's rows, kv head, chunk-table row, part number
    int lo, hi_max, hi_min, rs_max;    // positions [lo, hi) of the rows
    int a0, n1, t2, begin, end;        // tile list: a0 .. a0+n1-1, then t2 ..; this CTA's share of it
    int hi[TM_TOK], sk[TM_TOK], rs[TM_TOK];
    float ex[2][2][TM_ROWS];           // row maxima (then sums) exchanged between the two column halves
};

__device__ __forceinline__ void tw(uint64_t *bar, uint32_t parity, TileShared &s, unsigned code) {
    if (*(volatile int *)&s.abort) return;
    if (!mbar_wait(bar, parity, code)) *(volatile int *)&s.abort = 1;
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
// 128-byte swizzle; 64-dim blocks 8 KB apart (LBO), 8-position groups 1 KB apart (SBO)
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
    uint64_t d = smem_desc_sw128(saddr);
    return (d & ~((uint64_t)0x3FFFu << 16)) | ((uint64_t)(8192u >> 4) << 16);
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

// Row tile `tile` -> its run and first row, by one converged warp; false behind the last tile.
__device__ __forceinline__ bool find_tile(const AttnTileArgs &p, int tile, int &run, int &row0) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int u = 0; u < p.n_run; u += 32) {
        const int a = u + lane < p.n_run ? p.off[u + lane] : 0, b = u + lane < p.n_run ? p.off[u + lane + 1] : 0;
        const int n = b > a ? (b - a + TM_TOK - 1) / TM_TOK : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + sum > tile);
        if (hit) {
            const int w = __ffs(hit) - 1;
            run = u + w;
            row0 = __shfl_sync(0xffffffffu, a + (tile - (before + sum - n)) * TM_TOK, w);
            return true;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

// What this CTA does, by warp 0; begin = end = 0 and nrow = 0 when there is no such unit.
__device__ __forceinline__ void find_work(const AttnTileArgs &p, const TilePlan &pl, TileShared &s) {
    const int lane = threadIdx.x & 31;
    int id = blockIdx.x, run = -1, row0 = 0, nrow = 0, ns = pl.ns, split;
    const int n_first = pl.tiles * AKV * pl.ns;
    const bool tail = id >= n_first;
    if (!tail) {
        split = id % ns;
        s.kvh = (id / ns) % AKV;
        int tile = id / (AKV * ns);
        if (!p.shared_len) tile = pl.tiles - 1 - tile;  // the last tokens of a run have the most to do: first
        if (find_tile(p, tile, run, row0)) nrow = min(TM_TOK, p.off[run + 1] - row0);
    } else {
        id -= n_first;
        ns = pl.ns_own;
        split = id % ns;
        s.kvh = (id / ns) % AKV;
        row0 = id / (AKV * ns);
        run = run_of_row(p, row0);
        nrow = run >= 0 ? 1 : 0;
    }
    if (row0 < 0 || row0 + nrow > p.n_row) nrow = 0;
    // lane = token of the tile
    const bool real = lane < nrow;
    int hi = 0, sk = 0, rs = 0, lo = 0;
    if (real) {
        const int r = row0 + lane;
        int L = p.shared_len ? p.len[r] : p.len[run] - (p.off[run + 1] - p.off[run]) + (r - p.off[run]) + 1;
        L = max(0, min(L, p.max_chunks * ACHUNK));
        int total;
        attended_range(L, p.window, p.sink, total, sk, rs);
        hi = L;
        if (p.shared_len) {
            const int sh = max(0, p.shared_len[run]);
            if (tail) lo = sh;
            else hi = min(L, sh);
        }
    }
    if (lane < TM_TOK) {
        s.hi[lane] = hi;
        s.sk[lane] = sk;
        s.rs[lane] = rs;
    }
    lo = warp_max_i(lo);
    const int hi_max = warp_max_i(hi), hi_min = warp_min_i(real ? hi : 0x7fffffff);
    const int rs_min = warp_min_i(real && hi > 0 ? rs : 0x7fffffff), rs_max = warp_max_i(rs);
    const int sk_end = min(warp_max_i(sk), hi_max);
    const int end = (hi_max + TK - 1) / TK, a0 = lo / TK;
    const int a1 = sk_end > lo ? (sk_end + TK - 1) / TK : a0;
    int t2 = max(lo, min(rs_min, hi_max)) / TK, n1 = a1 - a0;
    if (a1 >= t2) {  // one stretch (always so without a window: rs_min is 0)
        n1 = 0;
        t2 = min(t2, a0);
    }
    const int total = hi_max > lo ? n1 + max(0, end - t2) : 0;
    if (lane == 0) {
        s.row0 = row0;
        s.nrow = nrow;
        s.table = p.shared_len ? (tail ? row0 : (run >= 0 ? p.off[run] : 0)) : max(run, 0);
        s.part = tail ? pl.ns + split : split;
        s.lo = lo; s.hi_max = hi_max; s.hi_min = hi_min; s.rs_max = rs_max;
        s.a0 = a0; s.n1 = n1; s.t2 = t2;
        s.begin = (int)((long long)total * split / ns);
        s.end = (int)((long long)total * (split + 1) / ns);
    }
}

__device__ __forceinline__ int tile_at(const TileShared &s, int i) { return i < s.n1 ? s.a0 + i : s.t2 + (i - s.n1); }

// 8 values of a q8_0 row (block c / 4, quarter c % 4) as f16, rounded (lo null) or as exact hi + lo halves
template <bool HL>
__device__ __forceinline__ void q8_piece(const uint8_t *row, int c, uint4 &hi, uint4 &lo) {
    const uint8_t *blk = row + 34 * (c >> 2);
    const float d = __half2float(*reinterpret_cast<const __half *>(blk));
    const unsigned short *qd = reinterpret_cast<const unsigned short *>(blk + 2 + 8 * (c & 3));
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t two = qd[i];
        const float a = d * (float)(int8_t)(two & 0xffu), b = d * (float)(int8_t)(two >> 8);
        if constexpr (HL) split2(a, b, h[i], l[i]);
        else h[i] = pack2(a, b);
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (HL) lo = make_uint4(l[0], l[1], l[2], l[3]);
}

__device__ __forceinline__ void sts16(uint32_t dst, const uint4 &v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// ---- producers ------------------------------------------------------------------
template <bool HL, bool Q8>
struct Loader {
    using G = TileGeo<HL>;
    const AttnTileArgs &p;
    TileShared &s;
    uint32_t ring;
    int tid, issued = 0, told = 0;

    __device__ __forceinline__ void signal() {  // the oldest unsignalled stage is written (by this thread)
        fence_async_smem();
        __syncwarp();
        if ((tid & 31) == 0) mbar_arrive(&s.full[told % G::NST]);
        ++told;
    }
    __device__ __forceinline__ uint32_t acquire() {
        const int slot = issued % G::NST;
        if (issued >= G::NST) tw(&s.empty[slot], (uint32_t)(issued / G::NST - 1) & 1u, s, 1u);
        ++issued;
        return ring + slot * STAGE;
    }
    // half 0 / 1 of K (dims) or V (positions) of position tile t
    template <bool V>
    __device__ __forceinline__ void half_tile(int t, int half) {
        const uint64_t base = p.chunk_ptrs[(size_t)s.table * p.max_chunks + t / (ACHUNK / TK)];
        const uint64_t plane = base + (V ? p.v_off : p.k_off);
        // rows outside [lo, hi) (and of a chunk that is missing) come in as zeros
        const int lo = s.lo, hi = base ? s.hi_max : 0;
        const int pos0 = t * TK + (V ? half * 64 : 0);
        const size_t row0 = (size_t)s.kvh * ACHUNK + pos0 % ACHUNK;
        constexpr int PC = V ? 32 : 16;       // 16-byte pieces of f16 a row of the stage has
        constexpr int RP = LOAD_WARPS * 32 / PC, N = (V ? 64 : 128) / RP;
        const int c = tid % PC, r0 = tid / PC;
        const uint32_t blk = (uint32_t)(c >> 3) * (V ? 8192u : 16384u);
        if constexpr (Q8) {
            const uint32_t d0 = acquire(), d1 = HL ? acquire() : 0u;
#pragma unroll 4
            for (int i = 0; i < N; ++i) {
                const int r = r0 + i * RP, pos = pos0 + r;
                uint4 vh = make_uint4(0, 0, 0, 0), vl = vh;
                if (pos >= lo && pos < hi)
                    q8_piece<HL>(reinterpret_cast<const uint8_t *>(plane) + (row0 + r) * kKvQ8Row, c + (V ? 0 : half * 16), vh, vl);
                const uint32_t at = blk + sw128_off(r, c & 7);
                sts16(d0 + at, vh);
                if constexpr (HL) sts16(d1 + at, vl);
            }
            signal();
            if constexpr (HL) signal();
        } else {
            const uint32_t d0 = acquire();
            const uint8_t *src = reinterpret_cast<const uint8_t *>(plane) + (row0 + r0) * (AHD * 2) + (V ? 0 : half * 256) + c * 16;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = r0 + i * RP, pos = pos0 + r;
                const bool ok = pos >= lo && pos < hi;
                cpa16(d0 + blk + sw128_off(r, c & 7), ok ? static_cast<const void *>(src + (size_t)i * RP * AHD * 2) : p.q, ok);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (issued > G::LAG) {
                asm volatile("cp.async.wait_group %0;" ::"n"(G::LAG) : "memory");
                signal();
            }
        }
    }
    template <bool V>
    __device__ __forceinline__ void tile(int t) {
        half_tile<V>(t, 0);
        half_tile<V>(t, 1);
    }
    // K(0), then K(j + 1) before V(j): the order in which the products consume them
    __device__ __forceinline__ void run() {
        const int n = s.end - s.begin;
        if (n > 0) tile<false>(tile_at(s, s.begin));
        for (int j = 0; j < n; ++j) {
            if (j + 1 < n) tile<false>(tile_at(s, s.begin + j + 1));
            tile<true>(tile_at(s, s.begin + j));
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        while (told < issued) signal();
    }
};

// ---- products (one thread) --------------------------------------------------------
template <bool HL, bool Q8>
struct Products {
    using G = TileGeo<HL>;
    TileShared &s;
    uint32_t q, ring, tmem;
    int used = 0;

    static constexpr int PARTS = HL && Q8 ? 2 : 1;  // stages of a K or V half: values, or hi then lo
    __device__ __forceinline__ uint32_t next() {
        const int slot = used % G::NST;
        tw(&s.full[slot], (uint32_t)(used / G::NST) & 1u, s, 2u);
        return ring + slot * STAGE;
    }
    __device__ __forceinline__ void done() {
        tc_commit(&s.empty[used % G::NST]);
        ++used;
    }
    __device__ __forceinline__ void scores(int j) {
        const uint32_t d = tmem + 256 + (j & 1) * 128;
        constexpr uint32_t idesc = idesc_f16_f32(TM_ROWS, TK);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint32_t k = next();
                tc_fence_after();
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint32_t a = q + (half * 2 + b) * 16384 + ks * 32;
                        const uint64_t bd = smem_desc_sw128(k + b * 16384 + ks * 32);
                        tc_mma_f16(d, smem_desc_sw128(a), bd, idesc, !(half == 0 && part == 0 && b == 0 && ks == 0));
                        if (HL && part == 0) tc_mma_f16(d, smem_desc_sw128(a + QBYTES), bd, idesc, 1);
                    }
                done();
            }
        tc_commit(&s.s_full[j & 1]);
    }
    __device__ __forceinline__ void values(int j) {
        const uint32_t pa = tmem + 256 + (j & 1) * 128;
        constexpr uint32_t idesc = idesc_f16_f32(TM_ROWS, AHD) | (1u << 16);  // B MN-major
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint32_t v = next();
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    const uint64_t bd = desc_v(v + ks * 2048);
                    const uint32_t a = pa + half * 32 + ks * 8;
                    tc_mma_f16_ts(tmem, a, bd, idesc, !(j == 0 && half == 0 && part == 0 && ks == 0));
                    if (HL && part == 0) tc_mma_f16_ts(tmem, a + 64, bd, idesc, 1);
                }
                done();
            }
        tc_commit(&s.pv_done);
    }
    __device__ __forceinline__ void run() {
        const int n = s.end - s.begin;
        if (n <= 0) return;
        tw(&s.q_full, 0, s, 4u);
        scores(0);
        for (int j = 0; j < n; ++j) {
            if (j + 1 < n) scores(j + 1);  // into the buffer whose P the product before last has consumed, in order
            tw(&s.p_full[j & 1], (uint32_t)(j >> 1) & 1u, s, 8u);
            tc_fence_after();
            values(j);
        }
        tc_commit(&s.o_full);
        // after a timeout nobody else may be waiting: let the products end before TMEM is freed
        if (*(volatile int *)&s.abort) mbar_wait(&s.o_full, 0, 16u);
    }
};

// ---- the kernel ---------------------------------------------------------------------
template <bool HL, bool Q8>
__global__ void __launch_bounds__(TILE_THREADS, 1) attn_tile_kernel(AttnTileArgs p, TilePlan pl) {
    using G = TileGeo<HL>;
    using T = typename std::conditional<HL, float, __half>::type;
    extern __shared__ __align__(1024) uint8_t smem[];
    TileShared &s = *reinterpret_cast<TileShared *>(smem + G::SMEM);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sbase = smem_u32(smem);
    constexpr int MMA_WARP = SOFT_WARPS + LOAD_WARPS;
    if (sbase & 1023u) {  // the swizzled layouts need 1024-byte aligned stages
        if (tid == 0) atomicOr(&g_dev_error, 256u);
        return;
    }

    if (warp == 0) find_work(p, pl, s);
    if (warp == MMA_WARP) tmem_alloc(&s.tmem, 512);
    if (tid == 32) {
        for (int i = 0; i < G::NST; ++i) {
            mbar_init(&s.full[i], LOAD_WARPS);
            mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], SOFT_WARPS);
        }
        mbar_init(&s.pv_done, 1);
        mbar_init(&s.q_full, SOFT_WARPS);
        mbar_init(&s.o_full, 1);
        s.abort = 0;
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;

    if (s.nrow > 0 && warp >= SOFT_WARPS && warp < MMA_WARP) {
        Loader<HL, Q8> ld{p, s, sbase + G::QB, tid - SOFT_WARPS * 32};
        ld.run();
    } else if (s.nrow > 0 && warp == MMA_WARP) {
        if (lane == 0) {
            Products<HL, Q8> mm{s, sbase, sbase + G::QB, tmem};
            mm.run();
        }
        __syncwarp();
    } else if (s.nrow > 0) {
        // softmax warps: row = TMEM lane, columns (positions, then dims) of one half
        const int quarter = warp & 3, half = warp >> 2;
        const int row = quarter * 32 + lane, tok = row / AGRP;
        const bool real = tok < s.nrow;
        const bool busy = quarter * 32 / AGRP < s.nrow;  // some row of this warp is real
        const size_t grow = ((size_t)(s.row0 + (real ? tok : 0)) * AH + s.kvh * AGRP + row % AGRP);
        const int n = s.end - s.begin;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;

        // stage Q: 16-byte pieces, 32 a row; a warp takes a row per pass
        if (n > 0) {
            const T *qg = static_cast<const T *>(p.q);
            for (int r = warp; r < s.nrow * AGRP; r += SOFT_WARPS) {
                const size_t at = ((size_t)(s.row0 + r / AGRP) * AH + s.kvh * AGRP + r % AGRP) * AHD + lane * 8;
                const uint32_t dst = sbase + (lane >> 3) * 16384 + sw128_off(r, lane & 7);
                if constexpr (HL) {
                    const float4 a = *reinterpret_cast<const float4 *>(qg + at), b = *reinterpret_cast<const float4 *>(qg + at + 4);
                    uint4 hi, lo;
                    split2(a.x, a.y, hi.x, lo.x);
                    split2(a.z, a.w, hi.y, lo.y);
                    split2(b.x, b.y, hi.z, lo.z);
                    split2(b.z, b.w, hi.w, lo.w);
                    sts16(dst, hi);
                    sts16(dst + QBYTES, lo);
                } else {
                    sts16(dst, *reinterpret_cast<const uint4 *>(qg + at));
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.q_full);
        }

        const float c = p.scale * kLog2e;
        const int hi = real ? s.hi[tok] : 0x7fffffff, sk = real ? s.sk[tok] : 0, rs = real ? s.rs[tok] : 0;
        float m = -INFINITY, l = 0.0f;  // maximum in use; sum of this half's columns
        for (int j = 0; j < n; ++j) {
            const uint32_t sb = tmem + lanes + 256 + (j & 1) * 128;
            tw(&s.s_full[j & 1], (uint32_t)(j >> 1) & 1u, s, 32u);
            tc_fence_after();
            if (busy) {
                uint32_t u[64];
                tmem_ld32_async(sb + half * 64, u);
                tmem_ld32_async(sb + half * 64 + 32, u + 32);
                tmem_ld_wait();
                float f[64];
#pragma unroll
                for (int i = 0; i < 64; ++i) f[i] = __uint_as_float(u[i]);
                const int t = tile_at(s, s.begin + j), pos0 = t * TK;
                if (pos0 < s.lo || pos0 + TK > s.hi_min || pos0 < s.rs_max) {  // some row does not see all of the tile
                    const int lo = s.lo;
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        const int pos = pos0 + half * 64 + i;
                        if (pos >= hi || pos < lo || (pos >= sk && pos < rs)) f[i] = -INFINITY;
                    }
                }
                float mx = f[0];
#pragma unroll
                for (int i = 1; i < 64; ++i) mx = fmaxf(mx, f[i]);
                s.ex[j & 1][half][row] = mx;
                named_sync(1 + quarter, 64);  // also: both halves have read S, P may overwrite it
                mx = fmaxf(mx, s.ex[j & 1][half ^ 1][row]);
                const bool grow_m = mx > m && (m == -INFINITY || (mx - m) * c > kSlack);
                if (__any_sync(0xffffffffu, grow_m)) {
                    const float nm = grow_m ? mx : m;
                    const float alpha = m == -INFINITY ? 0.0f : ex2((m - nm) * c);
                    if (j > 0) {
                        tw(&s.pv_done, (uint32_t)(j - 1) & 1u, s, 64u);
                        tc_fence_after();
#pragma unroll
                        for (int b = 0; b < 8; ++b) {
                            uint32_t o[16];
                            const uint32_t ob = tmem + lanes + half * 128 + b * 16;
                            tmem_ld16_async(ob, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st16(ob, o);
                        }
                    }
                    l *= alpha;
                    m = nm;
                }
                const float off = m == -INFINITY ? 0.0f : fmaf(m, c, -kShift);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    uint32_t h[16], w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float e0 = ex2(fmaf(f[32 * b + 2 * i], c, -off)), e1 = ex2(fmaf(f[32 * b + 2 * i + 1], c, -off));
                        l += e0 + e1;
                        if constexpr (HL) split2(e0, e1, h[i], w[i]);
                        else h[i] = pack2(e0, e1);
                    }
                    tmem_st16(sb + half * 32 + b * 16, h);
                    if constexpr (HL) tmem_st16(sb + 64 + half * 32 + b * 16, w);
                }
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[j & 1]);
        }
        if (n > 0) {
            tw(&s.o_full, 0, s, 128u);
            tc_fence_after();
        }
        if (busy) {
            s.ex[n & 1][half][row] = l;
            named_sync(1 + quarter, 64);
            l += s.ex[n & 1][half ^ 1][row];
            const bool join = pl.ns + pl.ns_own > 1;
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            const int parts = pl.ns + pl.ns_own;
            const size_t slot = grow * parts + s.part;
            float2 *ml = static_cast<float2 *>(p.ws);
            float *acc = reinterpret_cast<float *>(ml + (size_t)p.n_row * AH * parts) + slot * AHD + half * 128;
            T *out = static_cast<T *>(p.out) + grow * AHD + half * 128;
            const T *gate = p.gate ? static_cast<const T *>(p.gate) + grow * AHD + half * 128 : nullptr;
            if (join && real && half == 0) ml[slot] = make_float2(m == -INFINITY ? m : fmaf(m, c, -kShift), l);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld32_async(tmem + lanes + half * 128 + b * 32, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;
                }
                if (!real) continue;
                if (join) {
                    if (n > 0) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4 *>(acc + b * 32 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[i + e]) * inv;
                    if constexpr (HL) {
                        if (gate) {
                            const float4 ga = *reinterpret_cast<const float4 *>(gate + b * 32 + i), gb = *reinterpret_cast<const float4 *>(gate + b * 32 + i + 4);
                            const float g[8] = {ga.x, ga.y, ga.z, ga.w, gb.x, gb.y, gb.z, gb.w};
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[e] *= sigmoid_f(g[e]);
                        }
                        *reinterpret_cast<float4 *>(out + b * 32 + i) = make_float4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<float4 *>(out + b * 32 + i + 4) = make_float4(y[4], y[5], y[6], y[7]);
                    } else {
                        if (gate) {
                            const uint4 gw = *reinterpret_cast<const uint4 *>(gate + b * 32 + i);
                            const __half2 *gh = reinterpret_cast<const __half2 *>(&gw);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 g = __half22float2(gh[e]);
                                y[2 * e] *= sigmoid_f(g.x);
                                y[2 * e + 1] *= sigmoid_f(g.y);
                            }
                        }
                        *reinterpret_cast<uint4 *>(out + b * 32 + i) =
                            make_uint4(pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7]));
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Merges the parts of each (row, head): a warp per head, 8 dims a lane.
template <typename T>
__global__ void __launch_bounds__(AH * 32) attn_join_kernel(AttnTileArgs p, int parts) {
    const int row = blockIdx.x, lane = threadIdx.x & 31, h = threadIdx.x >> 5;
    if (run_of_row(p, row) < 0) return;
    const size_t g = (size_t)row * AH + h;
    const float2 *ml = static_cast<const float2 *>(p.ws) + g * parts;
    const float *acc = reinterpret_cast<const float *>(static_cast<const float2 *>(p.ws) + (size_t)p.n_row * AH * parts) +
                       g * parts * AHD + lane * 8;
    float mx = -INFINITY;
    for (int i = lane; i < parts; i += 32) mx = fmaxf(mx, ml[i].x);
    mx = warp_max(mx);
    float l = 0.0f, o[8] = {};
    for (int i0 = 0; i0 < parts; i0 += 32) {
        float w = 0.0f;
        if (i0 + lane < parts) {
            const float2 t = ml[i0 + lane];
            w = t.x == -INFINITY ? 0.0f : ex2(t.x - mx);
            l = fmaf(w, t.y, l);
        }
        const int n = min(32, parts - i0);
        for (int i = 0; i < n; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            if (wi == 0.0f) continue;
            const float4 a = *reinterpret_cast<const float4 *>(acc + (size_t)(i0 + i) * AHD);
            const float4 b = *reinterpret_cast<const float4 *>(acc + (size_t)(i0 + i) * AHD + 4);
            o[0] = fmaf(wi, a.x, o[0]); o[1] = fmaf(wi, a.y, o[1]); o[2] = fmaf(wi, a.z, o[2]); o[3] = fmaf(wi, a.w, o[3]);
            o[4] = fmaf(wi, b.x, o[4]); o[5] = fmaf(wi, b.y, o[5]); o[6] = fmaf(wi, b.z, o[6]); o[7] = fmaf(wi, b.w, o[7]);
        }
    }
    l = warp_sum(l);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    T *out = static_cast<T *>(p.out) + g * AHD + lane * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        o[i] *= inv;
        if (p.gate) o[i] *= sigmoid_f(to_f32(static_cast<const T *>(p.gate)[g * AHD + lane * 8 + i]));
    }
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(out) = make_float4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<float4 *>(out + 4) = make_float4(o[4], o[5], o[6], o[7]);
    } else {
        *reinterpret_cast<uint4 *>(out) = make_uint4(pack2(o[0], o[1]), pack2(o[2], o[3]), pack2(o[4], o[5]), pack2(o[6], o[7]));
    }
}

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// The same plan for the workspace query and the launch.
TilePlan plan_for(int n_row, int n_run, int max_run, int max_len, int max_own, bool shared) {
    TilePlan pl{};
    pl.tiles = n_row / TM_TOK + (n_run < n_row ? n_run : n_row);
    if (!shared) {
        const long long most = (long long)n_run * ceil_div(max_run, TM_TOK);
        if (most < pl.tiles) pl.tiles = (int)most;
        const int units = pl.tiles * AKV, kv = ceil_div(max_len, TK);
        pl.ns = units >= kPlanSMs ? 1 : kPlanSMs / units;
        if (pl.ns > kv) pl.ns = kv;
        return pl;
    }
    // shared prefixes: parts of equal length, one wave of CTAs at most for the prefixes
    const int kv = ceil_div(max_len, TK), kv_own = ceil_div(max_own, TK) + 1;
    const long long work = (long long)AKV * ((long long)pl.tiles * kv + (long long)n_row * kv_own);
    int each = ceil_div(work, kPlanSMs);
    pl.ns = kv > 0 ? ceil_div(kv, each) : 1;
    pl.own_tiles = n_row;
    pl.ns_own = ceil_div(kv_own, each);
    return pl;
}

size_t parts_bytes(int n_row, const TilePlan &pl) {
    const int parts = pl.ns + pl.ns_own;
    return parts > 1 ? (size_t)n_row * AH * parts * (sizeof(float2) + AHD * sizeof(float)) : 256;
}

template <bool HL, bool Q8>
cudaError_t launch_tile(const AttnTileArgs &a, const TilePlan &pl, cudaStream_t st) {
    auto kern = attn_tile_kernel<HL, Q8>;
    constexpr int smem = (int)(TileGeo<HL>::SMEM + sizeof(TileShared));
    static_assert(smem <= 227 * 1024, "stages and Q fit one SM");
    cudaError_t e = qw35h::smem_optin((const void *)kern, smem);
    if (e != cudaSuccess) return e;
    const long long grid = (long long)pl.tiles * AKV * pl.ns + (long long)pl.own_tiles * AKV * pl.ns_own;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
    kern<<<(unsigned)grid, TILE_THREADS, smem, st>>>(a, pl);
    return cudaGetLastError();
}

}  // namespace

size_t attn_tile_workspace_bytes(int n_row, int n_run, int max_run, int max_len, int max_own) {
    return parts_bytes(n_row, plan_for(n_row, n_run, max_run, max_len, max_own, max_run == 0));
}

cudaError_t attn_tile_run(const AttnTileArgs &a, cudaStream_t st) {
    if (a.n_row <= 0) return cudaSuccess;
    const TilePlan pl = plan_for(a.n_row, a.n_run, a.max_run, a.max_len, a.max_own, a.shared_len != nullptr);
    if (a.ws_bytes < parts_bytes(a.n_row, pl)) return cudaErrorInvalidValue;
    cudaError_t e = a.half ? (a.kv_q8 ? launch_tile<false, true>(a, pl, st) : launch_tile<false, false>(a, pl, st))
                           : (a.kv_q8 ? launch_tile<true, true>(a, pl, st) : launch_tile<true, false>(a, pl, st));
    if (e != cudaSuccess) return e;
    const int parts = pl.ns + pl.ns_own;
    if (parts > 1) {
        (a.half ? attn_join_kernel<__half> : attn_join_kernel<float>)<<<a.n_row, AH * 32, 0, st>>>(a, parts);
        e = cudaGetLastError();
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
