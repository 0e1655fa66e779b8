// What the attention kernels over the quantized cache share: how queries, weights
// and values are scaled into fp16's range, and the matrix instructions' wrappers.
#pragma once

#include "mix_common.h"

namespace mx {

// The weights of the second product are p * vs * 2^9 / nu: at most 2^15 while
// the tile's value scales are at most 8 nu and p at most 8 (a row's scores are
// taken relative to a reference that they may pass by kSlack in log2).
constexpr float kPScale = 512.0f, kSlack = 3.0f;

typedef __attribute__((address_space(3))) s4* lds_s4;

__device__ inline h4 read_tr(const _Float16* p) {
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p)));
}
__device__ inline f16 mfma32(h8 a, h8 b, f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline h8 join(h4 a, h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// The power of two that a row's value scales in a tile are taken relative to: kept
// while the largest is within (nu / 16, 8 nu], `least` at least.  `peak` is the
// largest one yet, times what is left of its keys' weights.  The sums in units of
// nu / 2^9 are at most keys * 8 * 8 * 448 * 2^9 * peak / nu, below 2^54 peak / nu for
// 2^30 keys, so with nu at 2^-60 peak or more they stay within fp32; what a smaller
// one would keep of the present tile is below 2^-80 of the sums.  No step divides
// by more than 2^100, which fp32 holds.
__device__ inline float next_nu(float nu, float vmax, float peak, float least) {
    if (!(vmax > 0.0f) || vmax > 3e38f || (vmax <= nu * 8.0f && vmax > nu * 0x1p-4f)) return nu;
    const float want = fmaxf(fmaxf(vmax, peak * 0x1p-60f), fmaxf(nu * 0x1p-100f, least));
    return bits_f(f_bits(want) & 0x7F800000u);
}
// 2^9 / nu is finite: with value scales of fp32's smallest normal number a weight is 2 then.
constexpr float kLeastNu = 0x1p-118f;

__device__ inline uint32_t lane_max_u32(uint32_t x, int step) { return max(x, (uint32_t)__shfl_xor((int)x, step)); }

// The power of two that brings a row whose largest magnitude has these bits to [2^13, 2^14).
__device__ inline float row_scale(uint32_t top) {
    if (top >= 0x7F800000u) return __builtin_nanf("");
    const int e = 13 - ((int)(top >> 23) - 127);
    return top == 0 ? 1.0f : bits_f((uint32_t)(min(max(e, -126), 100) + 127) << 23);
}

// What a score is worth in log2, for a row scaled by `up`: positive and finite, since
// times infinity (a key that is not seen) or 0 (the largest score's own difference) it
// must not be NaN.  A row with a NaN or infinity has one too: its scores are NaN, where
// it sees a key at all.
__device__ inline float score_worth(float scale, float up) { return fminf(fmaxf(scale / up, 0x1p-149f), 0x1p127f); }

// Splits w into fp16 terms: hi, and what hi leaves.
__device__ inline void split8(const float* w, h8& hi, h8& lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const h2 a = to_h2(w[j], w[j + 1]);
        const h2 b = to_h2(w[j] - (float)a[0], w[j + 1] - (float)a[1]);
        hi[j] = a[0];
        hi[j + 1] = a[1];
        lo[j] = b[0];
        lo[j + 1] = b[1];
    }
}
__device__ inline h8 round8(const float* w) {
    h8 r;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const h2 a = to_h2(w[j], w[j + 1]);
        r[j] = a[0];
        r[j + 1] = a[1];
    }
    return r;
}

}  // namespace mx
