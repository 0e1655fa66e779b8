// Keys and values quantized into the pages of a cache, and read back.
//
// A row is one token's D values of one key-value head.  INT8: the scale is
// s = max|x| / 127 (one fp32 division) and a value the whole number nearest to
// x / s, ties to even.  e4m3: the scale is the smallest power of two that
// brings the row within 448, so x / s is exact and only the conversion rounds.
// A row that holds an infinity or NaN gets the scale NaN and reads back as
// NaN; a row of zeros gets the scale 0.
//
// Both kernels are bound by HBM: D values in, D bytes and a scale out (or the
// other way round).  A row takes D/4 lanes, four values each, so every load is
// 16 bytes a lane of fp32 and a row's maximum is a few lane exchanges.  A
// workgroup takes consecutive rows of the input, all heads of a token together
// (rows of one head, 4 KB apart: 25 us for the write below).  8192 tokens of 4
// heads of 256, fp32, INT8: write 20.0 us (84 MB, 4.2 TB/s), read 14.4 us (5.8
// TB/s, part of it from the caches); one token 3.2 and 2.5 us, the launch.
#include "mix_common.h"

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

struct KvArgs {
    const void* k;
    const void* v;
    int64_t k_token, k_head, v_token, v_head;  // element strides of k and v
    void* ko;                                  // kv_read: outputs [T, H, D]
    void* vo;
    uint8_t* kp;
    uint8_t* vp;
    float* ks;
    float* vs;
    const int32_t* slots;
    int64_t n_slots;  // slots of the cache
    int T, H, pshift, dt;
};

constexpr int kUnroll = 4;  // rows a lane holds at once

template <int L>
__device__ inline uint32_t max_lanes(uint32_t x) {
#pragma unroll
    for (int s = 1; s < L; s *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, s));
    return x;
}

// The whole number nearest to x / s (ties to even).  q is within one of it;
// x - q s is exact in fp32 (both are multiples of the smaller one's last bit
// and the difference is below s), so comparing it with s / 2 settles it.
__device__ inline float nearest(float x, float s, float inv) {
    const float q = __builtin_rintf(x * inv);
    const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s, a = __builtin_fabsf(r);
    const bool odd = ((int)q & 1) != 0;
    return a > h || (a == h && odd) ? q + __builtin_copysignf(1.0f, r) : q;
}

template <int KIND>
__device__ inline uint32_t quantize4(f4 x, uint32_t top, float& scale) {
    if (top >= 0x7F800000u) {
        scale = __builtin_nanf("");
        return 0;
    }
    if constexpr (KIND == kInt8) {
        // max|x| / 127: the product with the rounded reciprocal, corrected once, is the
        // quotient correctly rounded (the correction's remainder is exact) while nothing
        // is subnormal.
        constexpr float r127 = 1.0f / 127.0f;
        const float q = bits_f(top) * r127;
        scale = __builtin_fmaf(__builtin_fmaf(-q, 127.0f, bits_f(top)), r127, q);
        float up = 1.0f;
        if (top < 0x21800000u) {  // below 2^-60: s / 2 would lose a bit, the reciprocal overflow
            scale = bits_f(top) / 127.0f;
            if (scale == 0.0f) return 0;
            up = 0x1p64f;
        }
        const float s = scale * up, inv = __builtin_amdgcn_rcpf(s);  // nearest() puts right what it is off
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float q = fminf(fmaxf(nearest(x[i] * up, s, inv), -127.0f), 127.0f);
            w |= ((uint32_t)(int)q & 255u) << (8 * i);
        }
        return w;
    } else {
        if (top == 0) {
            scale = 0.0f;
            return 0;
        }
        // top <= 1.75 * 2^(e - 127): e - 8 brings it within 448, else e - 7.
        int e = (int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u);
        e = max(e, 1);  // the smallest normal scale
        scale = bits_f((uint32_t)e << 23);
        const float inv = bits_f((uint32_t)(254 - e) << 23);
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, w, true);
        return (uint32_t)w;
    }
}

template <int D, int KIND, int DT>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a) {
    constexpr int L = D / 4, R = 256 / L;  // lanes a row, rows a pass
    const int lane = threadIdx.x % L;
    const bool val = blockIdx.y;
    const void* src = val ? a.v : a.k;
    const int64_t ts = val ? a.v_token : a.k_token, hs = val ? a.v_head : a.k_head;
    uint8_t* pages = val ? a.vp : a.kp;
    float* scales = val ? a.vs : a.ks;
    const int64_t r0 = (int64_t)blockIdx.x * (R * kUnroll) + threadIdx.x / L, rows = (int64_t)a.T * a.H;
    f4 x[kUnroll];
    int64_t slot[kUnroll];
    int head[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t r = min(r0 + u * R, rows - 1);
        const int t = (int)((uint32_t)r / (uint32_t)a.H);
        head[u] = (int)r - t * a.H;
        slot[u] = a.slots[t];
        x[u] = load4(src, DT, t * ts + head[u] * hs + lane * 4);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, f_bits(x[u][i]) & 0x7FFFFFFFu);
        top = max_lanes<L>(top);
        if (r0 + u * R >= rows || slot[u] < 0 || slot[u] >= a.n_slots) continue;
        float scale;
        const uint32_t w = quantize4<KIND>(x[u], top, scale);
        const int64_t row = (((slot[u] >> a.pshift) * a.H + head[u]) << a.pshift) + (slot[u] & ((1 << a.pshift) - 1));
        *reinterpret_cast<uint32_t*>(pages + row * D + lane * 4) = w;
        if (lane == 0) scales[row] = scale;
    }
}

template <int D, int KIND, int DT>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a) {
    constexpr int L = D / 4, R = 256 / L;
    const int lane = threadIdx.x % L;
    const bool val = blockIdx.y;
    void* dst = val ? a.vo : a.ko;
    const uint8_t* pages = val ? a.vp : a.kp;
    const float* scales = val ? a.vs : a.ks;
    const int64_t r0 = (int64_t)blockIdx.x * (R * kUnroll) + threadIdx.x / L, rows = (int64_t)a.T * a.H;
    uint32_t w[kUnroll];
    float s[kUnroll];
    bool is[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t r = min(r0 + u * R, rows - 1);
        const int t = (int)((uint32_t)r / (uint32_t)a.H), h = (int)r - t * a.H;
        int64_t slot = a.slots[t];
        is[u] = slot >= 0 && slot < a.n_slots;
        slot = is[u] ? slot : 0;  // read, not used
        const int64_t row = (((slot >> a.pshift) * a.H + h) << a.pshift) + (slot & ((1 << a.pshift) - 1));
        w[u] = *reinterpret_cast<const uint32_t*>(pages + row * D + lane * 4);
        s[u] = scales[row];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        if (r0 + u * R >= rows) continue;
        const h2 lo = unpack2<KIND, false>(w[u]), hi = unpack2<KIND, true>(w[u]);
        f4 y = {(float)lo[0] * s[u], (float)lo[1] * s[u], (float)hi[0] * s[u], (float)hi[1] * s[u]};
        if (!is[u]) y = (f4){0, 0, 0, 0};
        store4(dst, DT, (r0 + u * R) * D + lane * 4, y);
    }
}

template <int D, int KIND, int DT>
void launch3(const KvArgs& a, bool write, hipStream_t st) {
    constexpr int per = 256 / (D / 4) * kUnroll;
    const dim3 grid((unsigned)(((int64_t)a.T * a.H + per - 1) / per), 2);
    if (write) kv_write_kernel<D, KIND, DT><<<grid, 256, 0, st>>>(a);
    else kv_read_kernel<D, KIND, DT><<<grid, 256, 0, st>>>(a);
}

template <int D, int KIND>
void launch2(const KvArgs& a, bool write, hipStream_t st) {
    if (a.dt == kF32) launch3<D, KIND, kF32>(a, write, st);
    else if (a.dt == kBF16) launch3<D, KIND, kBF16>(a, write, st);
    else launch3<D, KIND, kF16>(a, write, st);
}

template <int D>
void launch(const KvArgs& a, int kind, bool write, hipStream_t st) {
    if (kind == kInt8) launch2<D, kInt8>(a, write, st);
    else launch2<D, kFp8>(a, write, st);
}

int kv_call(const i4_kv_cache* c, KvArgs a, int T, int dtype, bool write, void* stream, const char* what) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
        bq_set_error("%s: null cache pointer", what);
        return -2;
    }
    if (c->kind != kInt8 && c->kind != kFp8) {
        bq_set_error("%s: cache kind must be 0 (INT8) or 1 (e4m3), got %d", what, c->kind);
        return -2;
    }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        bq_set_error("%s: head_dim must be 64, 128 or 256, got %d", what, c->head_dim);
        return -2;
    }
    int pshift = 4;
    while (pshift < 10 && (1 << pshift) != c->page_size) ++pshift;
    if ((1 << pshift) != c->page_size || c->num_pages < 1 || c->kv_heads < 1 || c->kv_heads > 4096 ||
        c->num_pages > (INT32_MAX >> pshift)) {
        bq_set_error("%s: needs a page size of 16 to 1024 that is a power of two, at least one page, 1 to 4096 heads "
                     "and fewer than 2^31 slots (got page size %d, %d pages, %d heads)",
                     what, c->page_size, c->num_pages, c->kv_heads);
        return -2;
    }
    if (dtype < kF32 || dtype > kF16 || T < 0) {
        bq_set_error("%s: needs a type of 0 to 2 and T >= 0 (got %d, %d)", what, dtype, T);
        return -2;
    }
    if ((int64_t)T * c->kv_heads > (1 << 27)) {  // a launch has fewer than 2^24 workgroups
        bq_set_error("%s: %d tokens of %d heads are too many for one call", what, T, c->kv_heads);
        return -2;
    }
    if (T == 0) return 0;
    if (!a.slots || (write ? !a.k || !a.v : !a.ko || !a.vo)) {
        bq_set_error("%s: null device pointer", what);
        return -2;
    }
    a.kp = static_cast<uint8_t*>(c->k);
    a.vp = static_cast<uint8_t*>(c->v);
    a.ks = c->k_scale;
    a.vs = c->v_scale;
    a.n_slots = (int64_t)c->num_pages << pshift;
    a.T = T;
    a.H = c->kv_heads;
    a.pshift = pshift;
    a.dt = dtype;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (c->head_dim == 64) launch<64>(a, c->kind, write, st);
    else if (c->head_dim == 128) launch<128>(a, c->kind, write, st);
    else launch<256>(a, c->kind, write, st);
    return launched(what) ? 0 : -5;
}

}  // namespace

extern "C" {

int i4_kv_write_dev(const i4_kv_cache* cache, const void* dK, const void* dV, int64_t k_token, int64_t k_head,
                    int64_t v_token, int64_t v_head, int T, int dtype, const int32_t* dSlots, void* stream) {
    KvArgs a{};
    a.k = dK;
    a.v = dV;
    a.k_token = k_token;
    a.k_head = k_head;
    a.v_token = v_token;
    a.v_head = v_head;
    a.slots = dSlots;
    return kv_call(cache, a, T, dtype, true, stream, "kv_write");
}

int i4_kv_read_dev(const i4_kv_cache* cache, void* dK, void* dV, int T, int dtype, const int32_t* dSlots,
                   void* stream) {
    KvArgs a{};
    a.ko = dK;
    a.vo = dV;
    a.slots = dSlots;
    return kv_call(cache, a, T, dtype, false, stream, "kv_read");
}

}  // extern "C"
