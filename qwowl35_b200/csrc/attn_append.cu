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
// rounded to f32 is off by up to 2^-7 rad.  Product and reduction modulo 2 pi
// are in f64 (one pair per lane of one warp, shared by the token's 20 heads);
// the sine and cosine of the reduced angle are f32.
#include "common.cuh"
#include "kvcache.cuh"
#include "ops.h"

namespace qw35 {

constexpr int APP_WARPS = AH + AKV + 1;  // a warp per head row, and one for the angles

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

template <typename T, bool Q8>
__global__ void __launch_bounds__(APP_WARPS * 32) attn_append_kernel(AttnAppendArgs p) {
    const int tok = blockIdx.x;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    __shared__ float2 turn[32];
    // a token outside the table (padding: a negative row) leaves everything as it was
    const int row = p.tok_seq[tok], pos = p.tok_pos[tok];
    if (row < 0 || row >= p.n_seq || pos < 0 || pos >= p.max_chunks * ACHUNK) return;
    const uint64_t base = p.chunk_ptrs[(size_t)row * p.max_chunks + pos / ACHUNK];
    if (base == 0) return;

    const float *src = p.qkv + (size_t)tok * p.qkv_stride;
    const int d0 = lane * 8;
    if (wid == AH + AKV) {
        const int axis = (int)(p.axis_map >> (2 * lane)) & 3;
        const double th = (double)p.rope_pos[(size_t)axis * p.n_tok + tok] * (double)p.rope_freq[lane];
        constexpr double kTwoPi = 6.283185307179586476925;
        const float r = (float)(th - rint(th * (1.0 / kTwoPi)) * kTwoPi);
        float sn, cs;
        sincosf(r, &sn, &cs);
        turn[lane] = make_float2(cs, sn);
        __syncthreads();
        return;
    }
    const bool isq = wid < AH;
    const int h = isq ? wid : wid - AH;
    const float *x = isq ? src + h * 2 * AHD : src + QFULL + h * AHD;
    float v[8], w[8], g[8];
    load8(x + d0, v);
    load8((isq ? x : x + AKV * AHD) + (isq ? AHD : 0) + d0, g);  // the gate of a q head, the V row of a kv head
    load8((isq ? p.q_norm_w : p.k_norm_w) + d0, w);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
    ss = warp_sum(ss);
    const float inv = rsqrtf(ss / (float)AHD + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * w[i];
    __syncthreads();
    // lanes 0..3 hold dims 0..31, lanes 4..7 their partners 32..63
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float partner = __shfl_xor_sync(0xffffffffu, v[i], 4);
        if (lane < 8) {
            const float2 t = turn[(d0 + i) & 31];
            v[i] = lane < 4 ? v[i] * t.x - partner * t.y : partner * t.y + v[i] * t.x;
        }
    }
    if (isq) {
        const size_t at = ((size_t)tok * AH + h) * AHD + d0;
        store8(static_cast<T *>(p.q_out) + at, v);
        store8(static_cast<T *>(p.gate_out) + at, g);
        return;
    }
    const size_t at = (size_t)h * ACHUNK + (pos % ACHUNK);
    if constexpr (Q8) {  // lanes 4b..4b+3 hold block b
        uint8_t *blk = reinterpret_cast<uint8_t *>(base) + at * kKvQ8Row + 34 * (lane >> 2);
        q8_block_store(v, blk + p.k_off, lane);
        q8_block_store(g, blk + p.v_off, lane);
    } else {
        store8(reinterpret_cast<__half *>(base + p.k_off) + at * AHD + d0, v);
        store8(reinterpret_cast<__half *>(base + p.v_off) + at * AHD + d0, g);
    }
}

cudaError_t attn_append_run(const AttnAppendArgs &a, cudaStream_t st) {
    if (a.n_tok <= 0) return cudaSuccess;
    auto kern = a.half ? (a.kv_q8 ? attn_append_kernel<__half, true> : attn_append_kernel<__half, false>)
                       : (a.kv_q8 ? attn_append_kernel<float, true> : attn_append_kernel<float, false>);
    kern<<<a.n_tok, APP_WARPS * 32, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace qw35
