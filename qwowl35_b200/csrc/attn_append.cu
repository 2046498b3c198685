// attn_append.cu -- token runs enter the paged KV cache.
//
// For each token and head x of q and k:  y = x / sqrt(mean(x^2) + eps) * w,
// then the pairs (y_i, y_{i+32}), i < 32, turn by the angle p_a(i) * f_i:
//   y_i c - y_{i+32} s,  y_i s + y_{i+32} c      (NeoX order, as attn_pre_kernel)
// where a(i) is the axis of pair i: text has one axis, pictures and video three
// (time, height, width), each pair taking its position from one of them.  K and
// V go to the cache row of the token's own (table row, position), which has
// nothing to do with the rotary positions; q and the output gate go out in f32
// or f16.
//
// Angles: positions reach 2^18 and the first frequency is 1, so a product
// rounded to f32 is off by up to 2^-7 rad.  The product and its reduction to a
// part of a turn are in f64 (one pair per lane of one warp, shared by the
// token's 20 heads); sine and cosine of that part are f32.
//
// Bound by HBM: 40,960 bytes in and 20,480 (f16) or 36,864 (f32) out a token.
// Few tokens: a CTA each, all loads out before anything is waited for.  Many:
// a CTA per SM walks the tokens behind a ring of 5 whole rows (200 KB), one bulk
// copy a row, so that loads never pause for the norm, the turn and the stores.
#include "common.cuh"
#include "kvcache.cuh"
#include "ops.h"
#include "pipe.cuh"

namespace qw35 {

constexpr int APP_WARPS = AH + AKV + 1;  // a warp per head row, and one for the angles (and the ring's copies)

__device__ __forceinline__ void load8(const float *p, float *v) {
    if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
}
__device__ __forceinline__ void store8(float *p, const float *v) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__half *p, const float *v) {
    __align__(16) __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}

// Cosine and sine of pair `lane` of a token
__device__ __forceinline__ float2 turn_of(int pos, float freq) {
    const double turns = (double)pos * (double)freq * 0.15915494309189533577;  // 1 / (2 pi)
    float sn, cs;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    return make_float2(cs, sn);
}
__device__ __forceinline__ int axis_of(const AttnAppendArgs &p, int pair) { return (int)(p.axis_map >> (2 * pair)) & 3; }

// Chunk that token `tok` goes to; 0 when it lies outside the table (padding: a negative row)
__device__ __forceinline__ uint64_t chunk_of(const AttnAppendArgs &p, int row, int pos) {
    const bool in = row >= 0 && row < p.n_seq && pos >= 0 && pos < p.max_chunks * ACHUNK;
    return in ? p.chunk_ptrs[(size_t)row * p.max_chunks + pos / ACHUNK] : 0;
}

__device__ __forceinline__ void norm_row(const AttnAppendArgs &p, float *v, const float *w) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
    ss = warp_sum(ss);
    const float inv = rsqrtf(ss / (float)AHD + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
}

// Turns a normed head row (8 dims a lane) and writes it with its gate (q head) or V row (kv head) g; nothing is
// written without a chunk
template <typename T, bool Q8>
__device__ __forceinline__ void write_row(const AttnAppendArgs &p, int tok, int head, int pos, uint64_t base, float *v,
                                          const float *g, const float2 *turn) {
    const int lane = threadIdx.x & 31, d0 = lane * 8;
    // lanes 0..3 hold dims 0..31, lanes 4..7 their partners 32..63
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float partner = __shfl_xor_sync(0xffffffffu, v[i], 4);
        if (lane < 8) {
            const float2 t = turn[(d0 + i) & 31];
            v[i] = lane < 4 ? v[i] * t.x - partner * t.y : partner * t.y + v[i] * t.x;
        }
    }
    if (base == 0) return;
    if (head < AH) {
        const size_t at = ((size_t)tok * AH + head) * AHD + d0;
        store8(static_cast<T *>(p.q_out) + at, v);
        store8(static_cast<T *>(p.gate_out) + at, g);
        return;
    }
    const size_t at = (size_t)(head - AH) * ACHUNK + (pos % ACHUNK);
    if constexpr (Q8) {  // lanes 4b..4b+3 hold block b
        uint8_t *blk = reinterpret_cast<uint8_t *>(base) + at * kKvQ8Row + 34 * (lane >> 2);
        q8_block_store<true>(v, blk + p.k_off, lane);  // (a NaN stays one, as in f16 planes)
        q8_block_store<true>(g, blk + p.v_off, lane);
    } else {
        store8(reinterpret_cast<__half *>(base + p.k_off) + at * AHD + d0, v);
        store8(reinterpret_cast<__half *>(base + p.v_off) + at * AHD + d0, g);
    }
}

// offset of a head's q or k in a token's row, and from it to its gate or v
__device__ __forceinline__ int row_at(int head) { return head < AH ? head * 2 * AHD : QFULL + (head - AH) * AHD; }
__device__ __forceinline__ int pair_at(int head) { return head < AH ? AHD : AKV * AHD; }

template <typename T, bool Q8>
__global__ void __launch_bounds__(APP_WARPS * 32) attn_append_kernel(AttnAppendArgs p) {
    const int tok = blockIdx.x;
    const int lane = threadIdx.x & 31, head = threadIdx.x >> 5;
    __shared__ float2 turn[32];
    const int row = p.tok_seq[tok], pos = p.tok_pos[tok];
    if (head == AH + AKV) {
        turn[lane] = turn_of(p.rope_pos[(size_t)axis_of(p, lane) * p.n_tok + tok], p.rope_freq[lane]);
        __syncthreads();
        return;
    }
    float v[8], w[8], g[8];
    const float *x = p.qkv + (size_t)tok * p.qkv_stride + row_at(head) + lane * 8;
    load8(x, v);
    load8(x + pair_at(head), g);
    load8((head < AH ? p.q_norm_w : p.k_norm_w) + lane * 8, w);
    const uint64_t base = chunk_of(p, row, pos);
    norm_row(p, v, w);
    __syncthreads();
    write_row<T, Q8>(p, tok, head, pos, base, v, g, turn);
}

constexpr int RING = 5;
constexpr uint32_t ROW_BYTES = (QFULL + 2 * AKV * AHD) * 4;
struct __align__(16) AppendRing {
    uint64_t full[RING], empty[RING];
    uint64_t base[RING];
    int pos[RING];
    int abort;
    float2 turn[RING][32];
};

// rows of 16-byte aligned tokens
template <typename T, bool Q8>
__global__ void __launch_bounds__(APP_WARPS * 32) attn_append_ring_kernel(AttnAppendArgs p) {
    extern __shared__ __align__(128) uint8_t smem[];
    AppendRing &s = *reinterpret_cast<AppendRing *>(smem + RING * ROW_BYTES);
    const int lane = threadIdx.x & 31, head = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < RING; ++i) {
            mbar_init(&s.full[i], 2);  // the copy's bytes, and the token's words
            mbar_init(&s.empty[i], AH + AKV);
        }
        s.abort = 0;
        fence_barrier_init();
    }
    __syncthreads();
    auto wait = [&](uint64_t *bar, uint32_t parity) {  // after one wait has run out, none waits any more
        if (!*(volatile int *)&s.abort && !mbar_wait(bar, parity, 1024u)) *(volatile int *)&s.abort = 1;
    };
    const int n = (p.n_tok - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;  // this CTA's tokens
    int slot = 0;
    uint32_t phase = 0;
    if (head == AH + AKV) {
        const int axis = axis_of(p, lane);
        const float freq = p.rope_freq[lane];
        const uint64_t policy = policy_evict_first();
        int pos = 0;
        uint64_t base = 0;
        int rot = p.rope_pos[(size_t)axis * p.n_tok + blockIdx.x];
        for (int k = 0; k < n; ++k) {
            const int tok = (int)blockIdx.x + k * (int)gridDim.x;
            if (k >= RING) wait(&s.empty[slot], phase ^ 1u);
            const bool copied = !*(volatile int *)&s.abort;
            if (lane == 0 && copied) {
                mbar_arrive_expect_tx(&s.full[slot], ROW_BYTES);
                bulk_g2s(smem + slot * ROW_BYTES, p.qkv + (size_t)tok * p.qkv_stride, ROW_BYTES, &s.full[slot], policy);
            }
            if ((k & 31) == 0) {  // where the next 32 tokens go, one a lane
                const int t = tok + lane * (int)gridDim.x;
                pos = t < p.n_tok ? p.tok_pos[t] : 0;
                base = t < p.n_tok ? chunk_of(p, p.tok_seq[t], pos) : 0;
            }
            s.turn[slot][lane] = turn_of(rot, freq);
            const int tok_pos = __shfl_sync(0xffffffffu, pos, k & 31);
            const uint64_t tok_base = __shfl_sync(0xffffffffu, base, k & 31);
            if (k + 1 < n) rot = p.rope_pos[(size_t)axis * p.n_tok + tok + gridDim.x];
            if (lane == 0) {
                s.base[slot] = tok_base;
                s.pos[slot] = tok_pos;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.full[slot]);
            if (++slot == RING) {
                slot = 0;
                phase ^= 1u;
            }
            if (*(volatile int *)&s.abort) {  // no more copies; those under way land before this CTA ends
                for (int i = 0; i < RING && i <= k; ++i) {
                    slot = slot == 0 ? RING - 1 : slot - 1;
                    if (slot == RING - 1) phase ^= 1u;
                    if (lane == 0 && (i > 0 || copied)) mbar_wait(&s.full[slot], phase, 1024u);
                }
                return;
            }
        }
        return;
    }
    float w[8];
    load8((head < AH ? p.q_norm_w : p.k_norm_w) + lane * 8, w);
    for (int k = 0; k < n; ++k) {
        wait(&s.full[slot], phase);
        if (*(volatile int *)&s.abort) return;
        const float *x = reinterpret_cast<const float *>(smem + slot * ROW_BYTES) + row_at(head) + lane * 8;
        float v[8], g[8];
        load8(x, v);
        load8(x + pair_at(head), g);
        norm_row(p, v, w);
        write_row<T, Q8>(p, (int)blockIdx.x + k * (int)gridDim.x, head, s.pos[slot], s.base[slot], v, g, s.turn[slot]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.empty[slot]);
        if (++slot == RING) {
            slot = 0;
            phase ^= 1u;
        }
    }
}

template <typename T, bool Q8>
static cudaError_t append(const AttnAppendArgs &a, cudaStream_t st) {
    // The ring pays from about six tokens an SM on, for rows that bulk copies can fetch.  f16 on 148 SMs, a CTA a
    // token against the ring: 600 tokens 9.5 us both, 1200 15.8 against 15.0, 1837 24.5 against 20.2 (5.6 TB/s),
    // 8192 97.7 against 83.6 (6.0 TB/s); f32 8192 126.7 against 113.3.
    constexpr int kRingTokens = 6;
    const int sms = qw35h::sm_count();
    const bool aligned = (reinterpret_cast<uintptr_t>(a.qkv) & 15u) == 0 && a.qkv_stride % 4 == 0;
    if (aligned && a.n_tok >= kRingTokens * sms) {
        constexpr int smem = (int)(RING * ROW_BYTES + sizeof(AppendRing));
        static_assert(smem <= 227 * 1024, "the ring fits one SM");
        auto kern = attn_append_ring_kernel<T, Q8>;
        const cudaError_t e = qw35h::smem_optin((const void *)kern, smem);
        if (e != cudaSuccess) return e;
        kern<<<sms, APP_WARPS * 32, smem, st>>>(a);
    } else {
        attn_append_kernel<T, Q8><<<a.n_tok, APP_WARPS * 32, 0, st>>>(a);
    }
    return cudaGetLastError();
}

cudaError_t attn_append_run(const AttnAppendArgs &a, cudaStream_t st) {
    if (a.n_tok <= 0) return cudaSuccess;
    return a.half ? (a.kv_q8 ? append<__half, true>(a, st) : append<__half, false>(a, st))
                  : (a.kv_q8 ? append<float, true>(a, st) : append<float, false>(a, st));
}

unsigned int attn_append_error_read_and_clear() {
    unsigned int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_dev_error, sizeof(v));
    if (v) cudaMemcpyToSymbol(g_dev_error, &z, sizeof(z));
    return v;
}

}  // namespace qw35
