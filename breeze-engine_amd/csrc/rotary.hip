// Rotary positions: pairs of a head's values turned by an angle that grows with
// the token's position.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = position * f_i,
//
// for the pairs i of the first `rot` values of each head: (x_i, x_{i + rot/2})
// or (x_{2i}, x_{2i+1}).  The other values are copied, or left where the output is
// the input.
//
// A position of 10^6 times a frequency of 1 has its angle's last fp32 bit at
// 0.06: angles are taken in 64 bits, as quarter turns, whose whole part is
// dropped before the rest is rounded to fp32 (an error of 5e-8 in the angle,
// whatever the position).
//
// Bound by HBM: every value in and out once.  A token's angles serve all of its
// heads: a workgroup works them out once, in LDS, for its tokens.  8192 tokens of 40 heads
// of 128, bf16: 168 MB in 37 us (4.5 TB/s), 32 over the same inputs call after call, part of
// which the caches keep; few tokens: the host's part of the call, 12 us.
#include "mix_common.h"

#include <algorithm>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

struct RotArgs {
    const void* in[2];  // q, k
    void* out[2];
    int64_t in_token[2], in_head[2], out_token[2], out_head[2];  // element strides
    int q_heads, heads;  // q's heads, q's and k's together
    const int32_t* positions;
    const double* freqs;  // quarter turns a position, [half]
    int T, half, tokens;  // half = rot / 2; tokens a workgroup
    int rot_units, units;  // a row's units that are turned, and those with the ones that are copied
    float amplitude;
};

// V elements of a row, as fp32: 4 at a time, or one.
template <int DT, int V>
__device__ inline void load_row(const void* p, int64_t i, float* x) {
    if constexpr (V == 1) {
        if constexpr (DT == kF32) {
            x[0] = static_cast<const float*>(p)[i];
        } else {
            const uint16_t w = static_cast<const uint16_t*>(p)[i];
            x[0] = DT == kBF16 ? bf_lo(w) : (float)__builtin_bit_cast(_Float16, w);
        }
    } else {
        const f4 v = load4(p, DT, i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    }
}
template <int DT, int V>
__device__ inline void store_row(void* p, int64_t i, const float* x) {
    if constexpr (V == 1) {
        if constexpr (DT == kF32) static_cast<float*>(p)[i] = x[0];
        else if constexpr (DT == kBF16) static_cast<uint16_t*>(p)[i] = (uint16_t)to_bf16(x[0]);
        else static_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, (_Float16)x[0]);
    } else {
        store4(p, DT, i, (f4){x[0], x[1], x[2], x[3]});
    }
}

constexpr int kAngles = 2048;  // of a workgroup's tokens

// A unit is 2 V values of a row: V pairs, or what is copied.
template <int DT, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
    __shared__ float sc[kAngles], ss[kAngles];
    const int t0 = blockIdx.x * a.tokens, n = min(a.tokens, a.T - t0);
    for (int i = threadIdx.x; i < n * a.half; i += 256) {
        const int t = i / a.half;
        const double x = (double)a.positions[t0 + t] * a.freqs[i - t * a.half], whole = __builtin_rint(x);
        const float rest = (float)(x - whole);  // within half a quarter turn
        float s, c;
        sincospif(0.5f * rest, &s, &c);
        // Quarter turns past 2^31: the last two bits are what counts.
        const int quarter = (int)(whole - 4.0 * __builtin_floor(whole * 0.25));
        const float cq = quarter & 1 ? s : c, sq = quarter & 1 ? c : s;
        sc[i] = (quarter == 1 || quarter == 2 ? -cq : cq) * a.amplitude;
        ss[i] = (quarter == 2 || quarter == 3 ? -sq : sq) * a.amplitude;
    }
    __syncthreads();
    const uint32_t total = (uint32_t)n * a.heads * a.units;
    for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < total; i += gridDim.y * 256) {
        const uint32_t row = i / (uint32_t)a.units, u = i - row * a.units;
        const uint32_t t = row / (uint32_t)a.heads, r = row - t * a.heads;
        const bool key = r >= (uint32_t)a.q_heads;
        const int64_t tok = t0 + t, h = key ? r - a.q_heads : r;
        const void* const in = key ? a.in[1] : a.in[0];
        void* const out = key ? a.out[1] : a.out[0];
        const int64_t from = tok * (key ? a.in_token[1] : a.in_token[0]) + h * (key ? a.in_head[1] : a.in_head[0]);
        const int64_t to = tok * (key ? a.out_token[1] : a.out_token[0]) + h * (key ? a.out_head[1] : a.out_head[0]);
        const bool turned = (int)u < a.rot_units;
        const int first = INTER || !turned ? 2 * V * u : V * u, second = INTER || !turned ? first + V : first + a.half;
        float x[V], y[V];
        load_row<DT, V>(in, from + first, x);
        load_row<DT, V>(in, from + second, y);
        if (turned) {
            const float *c = sc + t * a.half + V * u, *s = ss + t * a.half + V * u;
            float p[V], q[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                // INTER with V > 1: pair j is values 2 j and 2 j + 1 of the unit's 2 V.
                const float re = !INTER || V == 1 ? x[j] : 2 * j < V ? x[2 * j % V] : y[2 * j % V];
                const float im = !INTER || V == 1 ? y[j] : 2 * j < V ? x[(2 * j + 1) % V] : y[(2 * j + 1) % V];
                p[j] = re * c[j] - im * s[j];
                q[j] = im * c[j] + re * s[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (!INTER || V == 1) {
                    x[j] = p[j];
                    y[j] = q[j];
                } else {
                    x[j] = j % 2 ? q[j / 2] : p[j / 2];
                    y[j] = j % 2 ? q[(V + j) / 2] : p[(V + j) / 2];
                }
            }
        }
        store_row<DT, V>(out, to + first, x);
        store_row<DT, V>(out, to + second, y);
    }
}

template <int DT, int V>
void launch2(const RotArgs& a, bool inter, dim3 grid, hipStream_t st) {
    if (inter) rotary_kernel<DT, V, true><<<grid, 256, 0, st>>>(a);
    else rotary_kernel<DT, V, false><<<grid, 256, 0, st>>>(a);
}

template <int DT>
void launch1(const RotArgs& a, int v, bool inter, dim3 grid, hipStream_t st) {
    if (v == 4) launch2<DT, 4>(a, inter, grid, st);
    else launch2<DT, 1>(a, inter, grid, st);
}

}  // namespace

extern "C" int i4_rotary_dev(const void* dQ, int64_t q_token, int64_t q_head, int q_heads, const void* dK,
                             int64_t k_token, int64_t k_head, int k_heads, int T, int head_dim, int rot, int interleaved,
                             int dtype, const int32_t* dPositions, const double* dFreqs, float amplitude, void* dQo,
                             int64_t qo_token, int64_t qo_head, void* dKo, int64_t ko_token, int64_t ko_head,
                             void* stream) {
    // A launch has fewer than 2^24 workgroups in a dimension.
    if (dtype < kF32 || dtype > kF16 || T < 0 || T > (1 << 23) || head_dim < 2 || head_dim > 4096 || head_dim % 2 || rot < 2 ||
        rot > head_dim || rot % 2 || q_heads < 0 || k_heads < 0 || q_heads > 65536 || k_heads > 65536) {
        bq_set_error("rotary: needs a type of 0 to 2, even head_dim up to 4096, even rotary dim up to that, up to "
                     "65536 heads and 2^23 tokens (got %d, %d, %d, %d and %d heads, %d tokens)",
                     dtype, head_dim, rot, q_heads, k_heads, T);
        return -2;
    }
    if (T == 0 || q_heads + k_heads == 0) return 0;
    if (!dPositions || !dFreqs || (q_heads > 0 && (!dQ || !dQo)) || (k_heads > 0 && (!dK || !dKo))) {
        bq_set_error("rotary: null device pointer");
        return -2;
    }
    RotArgs a{};
    a.in[0] = dQ;
    a.in[1] = dK;
    a.out[0] = dQo;
    a.out[1] = dKo;
    a.q_heads = q_heads;
    a.heads = q_heads + k_heads;
    const int heads[2] = {q_heads, k_heads};
    const int64_t strides[8] = {q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head};
    for (int i = 0; i < 2; ++i) {
        a.in_token[i] = strides[2 * i];
        a.in_head[i] = strides[2 * i + 1];
        a.out_token[i] = strides[4 + 2 * i];
        a.out_head[i] = strides[5 + 2 * i];
    }
    // Four values a load where every row and pair allows it: 8192 tokens of 40 heads of 128, bf16, 32 us; one
    // value 57; 16 bytes (eight) 33.  fp32: 73, 72 with one.
    const int size = dtype == kF32 ? 4 : 2;
    const auto fits = [&](int n) {
        if (head_dim % (2 * n) || rot % (2 * n)) return false;
        for (int i = 0; i < 2; ++i) {
            if (heads[i] == 0) continue;
            for (const void* p : {a.in[i], static_cast<const void*>(a.out[i])})
                if (reinterpret_cast<uintptr_t>(p) % (n * size)) return false;
            if ((T > 1 && (a.in_token[i] % n || a.out_token[i] % n)) ||
                (heads[i] > 1 && (a.in_head[i] % n || a.out_head[i] % n)))
                return false;
        }
        return true;
    };
    const int v = fits(4) ? 4 : 1;
    a.positions = dPositions;
    a.freqs = dFreqs;
    a.T = T;
    a.half = rot / 2;
    a.rot_units = rot / (2 * v);
    const auto in_place = [&](int i) {
        return heads[i] == 0 ||
               (a.in[i] == a.out[i] && a.in_token[i] == a.out_token[i] && a.in_head[i] == a.out_head[i]);
    };
    a.units = in_place(0) && in_place(1) ? a.rot_units : head_dim / (2 * v);
    a.amplitude = amplitude;
    // Workgroups of about 2048 units, of as many tokens as their angles have room for; a token's units
    // over several where it has more, or where there are few tokens (one of 28 heads of 256: 2.5 us
    // on the GPU, 3.2 by one workgroup).
    const int64_t per_token = (int64_t)a.heads * a.units;
    a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>({2048 / per_token, kAngles / a.half, T / 512}));
    const int64_t units = a.tokens * per_token;
    const int64_t y = T < 512 ? (units + 255) / 256 : (units + 2047) / 2048;
    const dim3 grid((unsigned)((T + a.tokens - 1) / a.tokens),
                    (unsigned)std::min<int64_t>(y, 64));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (dtype == kF32) launch1<kF32>(a, v, interleaved != 0, grid, st);
    else if (dtype == kBF16) launch1<kBF16>(a, v, interleaved != 0, grid, st);
    else launch1<kF16>(a, v, interleaved != 0, grid, st);
    return launched("rotary") ? 0 : -5;
}
