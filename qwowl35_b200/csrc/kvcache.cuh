// kvcache.cuh -- the head layout, the chunk-table KV cache and its q8_0 rows, as
// the kernels that write and read them share them.
#pragma once
#include "common.cuh"

namespace qw35 {

constexpr int AH = 16;      // query heads
constexpr int AKV = 4;      // kv heads
constexpr int AHD = 256;    // head dim
constexpr int AGRP = AH / AKV;
constexpr int ACHUNK = 256; // positions per chunk
constexpr int QFULL = AH * AHD * 2;  // q | gate per head

// One q8_0 block of 32 values held 8 per lane by 4 consecutive lanes (lane % 4
// = the lane's quarter): qw35_q8_0_quantize_block (qw35_attention.metal:429-440).
// d = amax / 127 in fp32, codes round(x * (1 / d)) (half away from zero)
// clamped to +-127 with the fp32 d, the block stores half(d).  `blk` points at
// the block's 34 bytes {f16 d; int8 qs[32]}; every lane of the warp calls this.
// fmaxf passes over NaNs, as the reference's maximum does: they become codes of 0
// in a block of the others.  NANS: a block that has one gets a NaN d instead.
template <bool NANS = false>
__device__ __forceinline__ void q8_block_store(const float *x, uint8_t *blk, int lane) {
    auto larger = [](float a, float b) {
        if constexpr (!NANS) return fmaxf(a, b);
        float y;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
        return y;
    };
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = larger(amax, fabsf(x[i]));
    amax = larger(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = larger(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float d = amax / 127.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    uint32_t packed[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = __fmul_rn(x[i], id);  // a plain product, as the reference (no contraction)
        int q = (int)roundf(y);
        q = q < -127 ? -127 : (q > 127 ? 127 : q);
        packed[i >> 2] |= ((uint32_t)q & 0xffu) << (8 * (i & 3));
    }
    // the block starts 2 bytes before the codes; codes of quarter j at 2 + 8 j:
    // even addresses, so 16-bit stores
    unsigned short *qd = reinterpret_cast<unsigned short *>(blk + 2 + 8 * (lane & 3));
    qd[0] = (unsigned short)(packed[0] & 0xffffu);
    qd[1] = (unsigned short)(packed[0] >> 16);
    qd[2] = (unsigned short)(packed[1] & 0xffffu);
    qd[3] = (unsigned short)(packed[1] >> 16);
    if ((lane & 3) == 0) *reinterpret_cast<unsigned short *>(blk) = __half_as_ushort(__float2half_rn(d));
}

// What a query of context length L attends: all of it, or the first sk
// positions and those from rstart on (total of them).
__device__ __forceinline__ void attended_range(int L, int window, int sink, int &total, int &sk, int &rstart) {
    sk = max(0, min(sink, L));
    if (window <= 0 || sk + window >= L) {
        sk = 0; rstart = 0; total = L;
    } else {
        rstart = L - window; total = sk + window;
    }
}

}  // namespace qw35
