// Shared pieces of the token mixers (the quantized paged cache, attention over
// it, gated linear attention): element types, vector types and the conversions
// between them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

// Sets the calling thread's i4_last_error() text (qmm.hip).
void bq_set_error(const char* fmt, ...) __attribute__((format(printf, 1, 2), visibility("hidden")));

namespace mx {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));

// Element types of activations, and what a cache page holds.
enum { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum { kInt8 = 0, kFp8 = 1 };

constexpr float kLog2e = 1.4426950408889634f;

inline bool launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return true;
    bq_set_error("%s: %s", what, hipGetErrorString(e));
    return false;
}

__device__ inline float bits_f(uint32_t b) { return __builtin_bit_cast(float, b); }
__device__ inline uint32_t f_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

__device__ inline float bf_lo(uint32_t w) { return bits_f(w << 16); }
__device__ inline float bf_hi(uint32_t w) { return bits_f(w & 0xFFFF0000u); }

// Round to nearest even; NaN stays NaN.
__device__ inline uint32_t to_bf16(float f) {
    const uint32_t b = f_bits(f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return (b >> 16) | 0x40u;
    return (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
}

__device__ inline h2 to_h2(float a, float b) { return __builtin_convertvector((f2){a, b}, h2); }

// Four elements at element index i of a tensor of type dt, as fp32.  Rows are
// 16-byte (fp32) or 8-byte aligned at multiples of four elements.
__device__ inline f4 load4(const void* p, int dt, int64_t i) {
    if (dt == kF32) return *reinterpret_cast<const f4*>(static_cast<const float*>(p) + i);
    const u2 w = *reinterpret_cast<const u2*>(static_cast<const uint16_t*>(p) + i);
    if (dt == kBF16) return (f4){bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y)};
    const h4 h = __builtin_bit_cast(h4, w);
    return __builtin_convertvector(h, f4);
}

__device__ inline void store4(void* p, int dt, int64_t i, f4 v) {
    if (dt == kF32) {
        *reinterpret_cast<f4*>(static_cast<float*>(p) + i) = v;
    } else if (dt == kBF16) {
        u2 w;
        w.x = to_bf16(v.x) | to_bf16(v.y) << 16;
        w.y = to_bf16(v.z) | to_bf16(v.w) << 16;
        *reinterpret_cast<u2*>(static_cast<uint16_t*>(p) + i) = w;
    } else {
        *reinterpret_cast<h4*>(static_cast<uint16_t*>(p) + i) = __builtin_convertvector(v, h4);
    }
}

// Two values to bf16, by the instruction.
__device__ inline uint32_t pack_bf16(float a, float b) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, b2));
}

// store4 of a type known at compile time.
template <int DT>
__device__ inline void put4(void* p, int64_t i, f4 v) {
    if constexpr (DT == kBF16) {
        *reinterpret_cast<u2*>(static_cast<uint16_t*>(p) + i) = (u2){pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)};
    } else {
        store4(p, DT, i, v);
    }
}

// Two of the four 8-bit values of w as fp16, exactly.  INT8: the byte plus 128
// becomes the low mantissa of 1024 (one byte permute for two values), and
// 1152 comes off again.
template <int KIND, bool HI>
__device__ inline h2 unpack2(uint32_t w) {
    if constexpr (KIND == kInt8) {
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t x = __builtin_amdgcn_perm(0x64646464u, u, HI ? 0x04030402u : 0x04010400u);
        return __builtin_bit_cast(h2, x) - (h2){(_Float16)1152.0f, (_Float16)1152.0f};
    } else {
        return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
    }
}

template <int KIND>
__device__ inline h8 unpack8(uint32_t a, uint32_t b) {
    const h2 x = unpack2<KIND, false>(a), y = unpack2<KIND, true>(a);
    const h2 z = unpack2<KIND, false>(b), w = unpack2<KIND, true>(b);
    return (h8){x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}

// The max over lanes l and l ^ 32, in both.
__device__ inline float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(f_bits(x), f_bits(x), false, false);
    return fmaxf(bits_f(r[0]), bits_f(r[1]));
}
__device__ inline float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(f_bits(x), f_bits(x), false, false);
    return bits_f(r[0]) + bits_f(r[1]);
}
// The max over lanes l and l ^ 16, in both.
__device__ inline float max_rows16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(f_bits(x), f_bits(x), false, false);
    return fmaxf(bits_f(r[0]), bits_f(r[1]));
}
__device__ inline float sum_rows16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(f_bits(x), f_bits(x), false, false);
    return bits_f(r[0]) + bits_f(r[1]);
}

// The max over 16 neighbouring lanes, in all of them.
__device__ inline float max_16(float x) {
    const auto turned = [](float v, auto n) {
        return bits_f((uint32_t)__builtin_amdgcn_mov_dpp((int)f_bits(v), 0x120 + decltype(n)::value, 0xF, 0xF, true));
    };
    x = fmaxf(x, turned(x, std::integral_constant<int, 1>()));  // row_ror:1, 2, 4, 8 within 16 lanes
    x = fmaxf(x, turned(x, std::integral_constant<int, 2>()));
    x = fmaxf(x, turned(x, std::integral_constant<int, 4>()));
    return fmaxf(x, turned(x, std::integral_constant<int, 8>()));
}
// The max over a wave, in all lanes.
__device__ inline float max_wave(float x) { return max_halves(max_rows16(max_16(x))); }

// The last of n (1 or more) whole numbers from 0 on that `is` holds for, given that it holds
// for 0 and for all before one that it holds for: 64 at a time, one a lane, so that a search
// of up to 4096 waits for memory twice.
template <typename F>
__device__ inline int last_of(int n, F is) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (;;) {
        const int step = (n + 63) >> 6;
        const uint64_t yes = __ballot(lane * step < n && is(base + lane * step));
        const int last = yes ? 63 - __builtin_clzll(yes) : 0;
        base += last * step;
        if (step == 1) return base;
        n = min(step, n - last * step);
    }
}

__device__ inline float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes a lane from `src` to LDS at `lds` + 16 * lane.  The compiler does not
// see the load: its reader waits for it by hand.
__device__ inline void load_lds(const uint8_t* src, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(lds) : "memory");
}
__device__ inline uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)(p);
}
template <int N>
__device__ inline void wait_loads() {  // vmcnt(N)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace mx
