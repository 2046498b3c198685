// attn_tile.cu -- attention of many query rows over one stretch of the paged
// KV cache: token runs that attend causally, and sequences that share a prefix.
//
// A query row of context length L attends o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(q . k_j / 16 - m) over what attended_range(L) keeps, then
// o *= sigmoid(gate).
#include "common.cuh"
#include "kvcache.cuh"
#include "ops.h"

namespace qw35 {

// run (or group) that row r belongs to; -1 behind the last one
__device__ __forceinline__ int run_of_row(const AttnTileArgs &p, int r) {
    for (int u = 0; u < p.n_run; ++u)
        if (r >= p.off[u] && r < p.off[u + 1]) return u;
    return -1;
}

// One warp per (row, head): 8 dims a lane, one position at a time, running
// maximum and sum in f32.
template <typename T, bool Q8>
__global__ void __launch_bounds__(128) attn_rows_kernel(AttnTileArgs p) {
    const int r = blockIdx.x, lane = threadIdx.x & 31, h = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int u = run_of_row(p, r);
    if (u < 0) return;
    const int kvh = h / AGRP, d0 = lane * 8;
    int L = p.shared_len ? p.len[r] : p.len[u] - (p.off[u + 1] - p.off[u]) + (r - p.off[u]) + 1;
    L = min(L, p.max_chunks * ACHUNK);
    int total = 0, sk = 0, rstart = 0;
    if (L > 0) attended_range(L, p.window, p.sink, total, sk, rstart);
    const uint64_t *ctab = p.chunk_ptrs + (size_t)(p.shared_len ? r : u) * p.max_chunks;
    const size_t at = ((size_t)r * AH + h) * AHD + d0;
    float q[8], o[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = to_f32(static_cast<const T *>(p.q)[at + i]) * p.scale;
    float m = -INFINITY, l = 0.0f;
    for (int idx = 0; idx < total; ++idx) {
        const int pos = idx < sk ? idx : rstart + (idx - sk);
        const uint64_t base = ctab[pos / ACHUNK];
        const size_t row = (size_t)kvh * ACHUNK + pos % ACHUNK;
        float k[8], v[8];
        if constexpr (Q8) {
            const uint8_t *kb = reinterpret_cast<const uint8_t *>(base + p.k_off) + row * kKvQ8Row + 34 * (lane >> 2);
            const uint8_t *vb = reinterpret_cast<const uint8_t *>(base + p.v_off) + row * kKvQ8Row + 34 * (lane >> 2);
            const float dk = __half2float(*reinterpret_cast<const __half *>(kb));
            const float dv = __half2float(*reinterpret_cast<const __half *>(vb));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                k[i] = dk * (float)(int8_t)kb[2 + 8 * (lane & 3) + i];
                v[i] = dv * (float)(int8_t)vb[2 + 8 * (lane & 3) + i];
            }
        } else {
            const __half *kp = reinterpret_cast<const __half *>(base + p.k_off) + row * AHD + d0;
            const __half *vp = reinterpret_cast<const __half *>(base + p.v_off) + row * AHD + d0;
#pragma unroll
            for (int i = 0; i < 8; ++i) { k[i] = __half2float(kp[i]); v[i] = __half2float(vp[i]); }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(q[i], k[i], s);
        s = warp_sum(s);
        const float nm = fmaxf(m, s);
        const float a = m == -INFINITY ? 0.0f : expf(m - nm), e = nm == -INFINITY ? 0.0f : expf(s - nm);
        l = l * a + e;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = o[i] * a + e * v[i];
        m = nm;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float y = l > 0.0f ? o[i] / l : 0.0f;
        if (p.gate) y *= sigmoid_f(to_f32(static_cast<const T *>(p.gate)[at + i]));
        static_cast<T *>(p.out)[at + i] = (T)y;
    }
}

size_t attn_tile_workspace_bytes(int n_row, int n_run, int max_run, int max_len, int max_own) { return 256; }

cudaError_t attn_tile_run(const AttnTileArgs &a, cudaStream_t st) {
    if (a.n_row <= 0) return cudaSuccess;
    auto kern = a.half ? (a.kv_q8 ? attn_rows_kernel<__half, true> : attn_rows_kernel<__half, false>)
                       : (a.kv_q8 ? attn_rows_kernel<float, true> : attn_rows_kernel<float, false>);
    kern<<<dim3(a.n_row, AH / 4), 128, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace qw35
