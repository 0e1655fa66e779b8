// Gated linear attention, with the delta rule where beta is given.
//
//   S_t = e^{g_t} S_{t-1} + k_t u_t^T,   o_t = scale S_t^T q_t,
//   u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t)   (delta rule), or v_t
//
// for each value head, with its key head's q and k; S is [Dk, Dv] in fp32.
//
// Sequences of up to kShort tokens run the recurrence as it stands
// (gla_step_kernel), bound by reading and writing S.  Longer ones go in chunks
// of C = 64 tokens.  With G_i the sum of a chunk's g up to token i and S_0 the
// state before it,
//
//   (I + A) U = diag(beta) (V - diag(e^G) K S_0),
//   A_ij = beta_i e^{G_i - G_j} (k_i . k_j)  for j < i,
//   O = scale (diag(e^G) Q S_0 + M U),  M_ij = e^{G_i - G_j} (q_i . k_j)  for j <= i,
//   S_C = e^{G_C} S_0 + sum_j e^{G_C - G_j} k_j u_j^T.
//
// gla_intra_kernel computes T = (I + A)^{-1} and M for all chunks at once;
// gla_inter_kernel walks a sequence's chunks with S in registers, 16 of its
// columns a wave.
//
// Numerics.  Products run on the fp16 matrix instructions with each operand
// as two fp16 terms (hi, and what hi leaves; 22 bits and more) and three
// products, fp32 sums; q, k and v given as bf16 or fp16 are one term.  A power
// of two for each tile, row or column puts the largest value where fp16 has
// room; it changes no digit.  T is computed in fp32.  Sums of g are taken in
// 64 bits: e^{G_i - G_j} would lose what G_i and G_j have in common.
#include "mix_common.h"

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

constexpr int kChunk = 64;
constexpr int kShort = 16;

struct GlaArgs {
    const void* q;
    const void* k;
    const void* v;
    void* o;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
    const float* g;
    const float* beta;  // null: no delta rule
    int64_t g_token, beta_token;
    const float* s_in;  // [B, Hv, Dk, Dv]; null: zeros
    float* s_out;
    const int32_t* cu;  // null: one token a sequence
    _Float16* kf;       // [slots][Hk][hi, lo][64][Dk]
    _Float16* qf;
    _Float16* tf;  // [slots][Hv][hi, lo][64][64]
    _Float16* mf;
    float* unit;  // [slots][Hk][2]: what one unit of kf and of qf is worth
    float* fac;   // [slots][Hv][4][64]: e^G, beta, e^{G_C - G}, worth of a unit of T's row
    int T, B, Hk, Hv, rep, Dv, dt, nslots;
    int nshort;  // sequences of up to this many tokens are gla_step_kernel's
    float scale;
};

struct Span {
    int q0, n;
};
__device__ inline Span span_of(const GlaArgs& a, int b) {
    if (!a.cu) return {b, 1};
    const int q0 = min(max(a.cu[b], 0), a.T), q1 = min(max(a.cu[b + 1], q0), a.T);
    return {q0, q1 - q0};
}

__device__ inline float load1(const void* p, int dt, int64_t i) {
    if (dt == kF32) return static_cast<const float*>(p)[i];
    const uint16_t w = static_cast<const uint16_t*>(p)[i];
    return dt == kBF16 ? bits_f((uint32_t)w << 16) : (float)__builtin_bit_cast(_Float16, w);
}
__device__ inline void store1(void* p, int dt, int64_t i, float x) {
    if (dt == kF32) static_cast<float*>(p)[i] = x;
    else if (dt == kBF16) static_cast<uint16_t*>(p)[i] = (uint16_t)to_bf16(x);
    else static_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, (_Float16)x);
}

// A decay's logarithm; -infinity (a state that is dropped) as a number whose
// exponential is zero and whose sums stay exact.
__device__ inline float clean_g(float g) { return g < -1e4f ? -1e4f : g; }

// ------------------------------------------------------------------ short sequences

// A wave for 16 columns of one sequence's and head's state: lane (row r mod 16,
// four columns).  Before the update both S^T k and S^T q are summed over the
// rows, since S_t^T q = e^g S_{t-1}^T q + (k . q) u: one exchange a token.
template <int DK>
__global__ __launch_bounds__(256) void gla_step_kernel(GlaArgs a) {
    constexpr int R = DK / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = a.Dv / 16;
    const int64_t id = (int64_t)blockIdx.x * 4 + wave;
    if (id >= (int64_t)a.B * a.Hv * blocks) return;
    const int cb = (int)(id % blocks), hv = (int)(id / blocks % a.Hv), b = (int)(id / blocks / a.Hv);
    const Span sp = span_of(a, b);
    if (sp.n > a.nshort) return;
    const int hk = hv / a.rep, col = 16 * cb + 4 * (lane & 3), r0 = lane >> 2;
    const int64_t at = ((int64_t)b * a.Hv + hv) * DK * a.Dv;
    f4 S[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        S[i] = a.s_in ? *reinterpret_cast<const f4*>(a.s_in + at + (int64_t)(r0 + 16 * i) * a.Dv + col) : (f4){0, 0, 0, 0};
    for (int t = sp.q0; t < sp.q0 + sp.n; ++t) {
        float kv[R], qv[R], kq = 0.0f;
        f4 sk = {0, 0, 0, 0}, sq = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < R; ++i) {
            kv[i] = load1(a.k, a.dt, t * a.k_token + hk * a.k_head + r0 + 16 * i);
            qv[i] = load1(a.q, a.dt, t * a.q_token + hk * a.q_head + r0 + 16 * i);
        }
        const f4 v = load4(a.v, a.dt, t * a.v_token + hv * a.v_head + col);
        const float decay = expf(clean_g(a.g[t * a.g_token + hv]));
#pragma unroll
        for (int i = 0; i < R; ++i) {
            kq = __builtin_fmaf(kv[i], qv[i], kq);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                S[i][j] *= decay;
                sk[j] = __builtin_fmaf(S[i][j], kv[i], sk[j]);
                sq[j] = __builtin_fmaf(S[i][j], qv[i], sq[j]);
            }
        }
#pragma unroll
        for (int st = 4; st < 16; st *= 2) {
            kq += __shfl_xor(kq, st);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk[j] += __shfl_xor(sk[j], st);
                sq[j] += __shfl_xor(sq[j], st);
            }
        }
        kq = sum_halves(sum_rows16(kq));
        f4 u, o;
        const float beta = a.beta ? a.beta[t * a.beta_token + hv] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sk[j] = sum_halves(sum_rows16(sk[j]));
            sq[j] = sum_halves(sum_rows16(sq[j]));
            u[j] = a.beta ? beta * (v[j] - sk[j]) : v[j];
            o[j] = a.scale * __builtin_fmaf(kq, u[j], sq[j]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = __builtin_fmaf(kv[i], u[j], S[i][j]);
        if (r0 == 0) store4(a.o, a.dt, t * a.o_token + hv * a.o_head + col, o);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<f4*>(a.s_out + at + (int64_t)(r0 + 16 * i) * a.Dv + col) = S[i];
}

// ------------------------------------------------------------------ inside the chunks

// The power of two that brings a magnitude with these bits to [2^TOP, 2^(TOP + 1)).
template <int TOP>
__device__ inline float to_top(uint32_t bits) {
    const int e = TOP + 127 - (int)(bits >> 23);
    return bits == 0 ? 1.0f : bits_f((uint32_t)(min(max(e, -126), 126) + 127) << 23);
}
__device__ inline float inverse_pow2(float p) { return bits_f((254u << 23) - f_bits(p)); }

__device__ inline uint32_t abs_bits(float x) { return f_bits(x) & 0x7FFFFFFFu; }

__device__ inline f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// The chunk of a slot: sequence b's chunks take the slots from cu[b] / 64 + b on.
__device__ inline bool chunk_of(const GlaArgs& a, int slot, int& tok, int& n) {
    int b = 0, hi = a.B;
    while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (min(max(a.cu[mid], 0), a.T) / kChunk + mid <= slot) b = mid;
        else hi = mid;
    }
    const Span sp = span_of(a, b);
    const int c = slot - (sp.q0 / kChunk + b);
    tok = sp.q0 + c * kChunk;
    n = min(kChunk, sp.n - c * kChunk);
    return sp.n > a.nshort && c >= 0 && n > 0;
}

// One workgroup for a chunk and a key head: the products k_i . k_j and
// q_i . k_j once, then T and M for each of its value heads.
template <int DK, bool LO, bool DELTA>
__global__ __launch_bounds__(256) void gla_intra_kernel(GlaArgs a) {
    constexpr int KS = DK + 8, AS = kChunk + 4, L = DK / 4, NP = kChunk * L / 256;
    constexpr int NT = LO ? 2 : 1;
    __shared__ __align__(16) _Float16 sk[NT][kChunk * KS], sq[NT][kChunk * KS];
    __shared__ __align__(16) float sa[kChunk * AS], st[kChunk * AS], sm[kChunk * AS];
    __shared__ double sg[kChunk];
    __shared__ float sbeta[kChunk];
    __shared__ uint32_t stop[2][4];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % a.Hk, slot = blockIdx.x / a.Hk;
    int tok, n;
    if (!chunk_of(a, slot, tok, n)) return;

    // q and k, scaled to [2^3, 2^4) so that their products fit fp16 too.
    f4 kx[NP], qx[NP];
    uint32_t kt = 0, qt = 0;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int row = (tid + 256 * i) / L, d = 4 * (tid % L);
        kx[i] = qx[i] = (f4){0, 0, 0, 0};
        if (row < n) {
            kx[i] = load4(a.k, a.dt, (int64_t)(tok + row) * a.k_token + hk * a.k_head + d);
            qx[i] = load4(a.q, a.dt, (int64_t)(tok + row) * a.q_token + hk * a.q_head + d);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t x = abs_bits(kx[i][j]), y = abs_bits(qx[i][j]);
            kt = max(kt, x < 0x7F800000u ? x : 0u);
            qt = max(qt, y < 0x7F800000u ? y : 0u);
        }
    }
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        kt = max(kt, (uint32_t)__shfl_xor((int)kt, s));
        qt = max(qt, (uint32_t)__shfl_xor((int)qt, s));
    }
    if (lane == 0) {
        stop[0][wave] = kt;
        stop[1][wave] = qt;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        kt = max(kt, stop[0][w]);
        qt = max(qt, stop[1][w]);
    }
    const float kup = to_top<3>(kt), qup = to_top<3>(qt), kunit = inverse_pow2(kup), qunit = inverse_pow2(qup);
    const int64_t ck = (int64_t)slot * a.Hk + hk;
    if (tid == 0) {
        a.unit[2 * ck] = kunit;
        a.unit[2 * ck + 1] = qunit;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int row = (tid + 256 * i) / L, d = 4 * (tid % L);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            f4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = w ? qx[i][j] * qup : kx[i][j] * kup;
            const h4 hi = __builtin_convertvector(x, h4);
            _Float16* s = w ? sq[0] : sk[0];
            _Float16* out = (w ? a.qf : a.kf) + ck * (NT * kChunk * DK) + row * DK + d;
            *reinterpret_cast<h4*>(s + row * KS + d) = hi;
            *reinterpret_cast<h4*>(out) = hi;
            if constexpr (LO) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] -= (float)hi[j];
                const h4 lo = __builtin_convertvector(x, h4);
                *reinterpret_cast<h4*>((w ? sq[NT - 1] : sk[NT - 1]) + row * KS + d) = lo;
                *reinterpret_cast<h4*>(out + kChunk * DK) = lo;
            }
        }
    }
    __syncthreads();

    // Wave w: rows 16 w ..; columns up to them.
    const int r16 = lane & 15, c = lane >> 4;
    f4 kk[4], qk[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) kk[t] = qk[t] = (f4){0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < DK / 32; ++s) {
        const int ar = (16 * wave + r16) * KS + 32 * s + 8 * c;
        const h8 ak = *reinterpret_cast<const h8*>(sk[0] + ar), aq = *reinterpret_cast<const h8*>(sq[0] + ar);
        const h8 akl = *reinterpret_cast<const h8*>(sk[NT - 1] + ar), aql = *reinterpret_cast<const h8*>(sq[NT - 1] + ar);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t > wave) continue;
            const int br = (16 * t + r16) * KS + 32 * s + 8 * c;
            const h8 b = *reinterpret_cast<const h8*>(sk[0] + br);
            if constexpr (DELTA) kk[t] = mfma16(ak, b, kk[t]);
            qk[t] = mfma16(aq, b, qk[t]);
            if constexpr (LO) {
                const h8 bl = *reinterpret_cast<const h8*>(sk[NT - 1] + br);
                if constexpr (DELTA) kk[t] = mfma16(akl, b, mfma16(ak, bl, kk[t]));
                qk[t] = mfma16(aql, b, mfma16(aq, bl, qk[t]));
            }
        }
    }

    for (int r = 0; r < a.rep; ++r) {
        const int hv = hk * a.rep + r;
        const int64_t cv = (int64_t)slot * a.Hv + hv;
        float* fac = a.fac + cv * (4 * kChunk);
        if (wave == 0) {
            const bool is = lane < n;
            double G = is ? (double)clean_g(a.g[(int64_t)(tok + lane) * a.g_token + hv]) : 0.0;
            float be = 0.0f;
            if constexpr (DELTA) be = is ? a.beta[(int64_t)(tok + lane) * a.beta_token + hv] : 0.0f;
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const double up = __shfl_up(G, s);
                if (lane >= s) G += up;
            }
            sg[lane] = G;
            sbeta[lane] = be;
            fac[lane] = expf((float)G);
            fac[kChunk + lane] = be;
            fac[2 * kChunk + lane] = expf((float)(__shfl(G, 63) - G));
        }
        __syncthreads();
        // A and M, the blocks past the diagonal as zeros.
        {
            double gi[4];
            float bi[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                gi[e] = sg[16 * wave + 4 * c + e];
                bi[e] = sbeta[16 * wave + 4 * c + e] * kunit * kunit;
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int j = 16 * t + r16;
                const double gj = sg[j];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 16 * wave + 4 * c + e;
                    float av = 0.0f, mv = 0.0f;
                    if (j <= i) {
                        const float x = expf((float)(gi[e] - gj));
                        mv = x * qk[t][e];
                        av = j < i ? bi[e] * x * kk[t][e] : 0.0f;
                    }
                    sm[i * AS + j] = mv;
                    if constexpr (DELTA) sa[i * AS + j] = av;
                }
            }
        }
        __syncthreads();
        if constexpr (DELTA) {
            // The four blocks on the diagonal: a lane solves one column of one.
            if (wave == 0) {
                float x[16];
                const float* ab = sa + (16 * c) * AS + 16 * c;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float s = i == r16 ? 1.0f : 0.0f;
#pragma unroll
                    for (int j = 0; j < i; ++j) s = __builtin_fmaf(-ab[i * AS + j], x[j], s);
                    x[i] = s;
                    st[(16 * c + i) * AS + 16 * c + r16] = s;
                }
            }
            __syncthreads();
            // Column block c of T, from the diagonal down: T_rc = -T_rr sum_m A_rm T_mc.
            // The contraction takes row 4 c + m at step m, so a result is the next operand.
            if (wave < 3) {
                f4 col[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) col[0][e] = st[(16 * wave + 4 * c + e) * AS + 16 * wave + r16];
#pragma unroll
                for (int d = 1; d < 4; ++d) {  // block row wave + d
                    if (wave + d > 3) break;
                    const int rr = 16 * (wave + d);
                    f4 acc = {0, 0, 0, 0};
#pragma unroll
                    for (int m = 0; m < d; ++m) {
                        const f4 ar = *reinterpret_cast<const f4*>(sa + (rr + r16) * AS + 16 * (wave + m) + 4 * c);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc = mfma4(ar[e], col[m][e], acc);
                    }
                    const f4 tr = *reinterpret_cast<const f4*>(st + (rr + r16) * AS + rr + 4 * c);
                    f4 out = {0, 0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 4; ++e) out = mfma4(-tr[e], acc[e], out);
                    col[d] = out;
#pragma unroll
                    for (int e = 0; e < 4; ++e) st[(rr + 4 * c + e) * AS + 16 * wave + r16] = out[e];
                }
            }
            __syncthreads();
        }
        // Out as two fp16 terms: four lanes a row, sixteen values each.
        const int row = tid >> 2, q4 = 16 * (tid & 3);
        const bool past = q4 > (row & ~15);
#pragma unroll
        for (int w = 0; w < (DELTA ? 2 : 1); ++w) {
            const float* src = (w ? st : sm) + row * AS + q4;
            float x[16];
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                x[j] = past ? 0.0f : src[j];
                top = max(top, abs_bits(x[j]));
            }
            if (w) {
                top = max(top, (uint32_t)__shfl_xor((int)top, 1));
                top = max(top, (uint32_t)__shfl_xor((int)top, 2));
                const float up = to_top<12>(top);
                if (q4 == 0) fac[3 * kChunk + row] = inverse_pow2(up);
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] *= up;
            }
            _Float16* out = (w ? a.tf : a.mf) + cv * (2 * kChunk * kChunk) + row * kChunk + q4;
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
                h8 hi, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    hi[e] = (_Float16)x[j + e];
                    lo[e] = (_Float16)(x[j + e] - (float)hi[e]);
                }
                *reinterpret_cast<h8*>(out + j) = hi;
                *reinterpret_cast<h8*>(out + kChunk * kChunk + j) = lo;
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ from chunk to chunk

// Values in a result's layout (rows 16 t + 4 c + e, one column a lane) as the
// operand of a contraction over those rows, two fp16 terms scaled for the
// column; returns what a unit is worth.  Slab s holds tiles 2 s and 2 s + 1.
template <int NT>
__device__ inline float to_operand(const f4* x, h8* hi, h8* lo) {
    uint32_t top = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, abs_bits(x[t][e]));
    top = f_bits(max_halves(max_rows16(bits_f(top))));  // magnitudes order as their bits do
    const float up = to_top<12>(top);
#pragma unroll
    for (int s = 0; s < NT / 2; ++s)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const f4 v = x[2 * s + (j >> 2)];
            const float p = v[j & 3] * up, q = v[(j & 3) + 1] * up;
            const h2 a = to_h2(p, q);
            const h2 b = to_h2(p - (float)a[0], q - (float)a[1]);
            hi[s][j] = a[0];
            hi[s][j + 1] = a[1];
            lo[s][j] = b[0];
            lo[s][j + 1] = b[1];
        }
    return inverse_pow2(up);
}

typedef __attribute__((address_space(3))) s4* lds_s4;
__device__ inline h4 read_tr(const _Float16* p) {
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p)));
}
__device__ inline h8 join(h4 a, h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// The operand whose contraction index runs in a result's order: 4 c + 0..3, 16 + 4 c + 0..3.
__device__ inline h8 read_rows(const _Float16* p) {
    return join(*reinterpret_cast<const h4*>(p), *reinterpret_cast<const h4*>(p + 16));
}

template <int DK, bool LO, bool DELTA>
__global__ __launch_bounds__(256, 1) void gla_inter_kernel(GlaArgs a) {
    constexpr int KS = DK + 8, TS = kChunk + 8, NT = LO ? 2 : 1;
    constexpr int NK = NT * kChunk * DK / 8 / 256, NM = 2 * kChunk * kChunk / 8 / 256;
    constexpr int ST = DK / 16, SS = DK / 32;  // tiles and slabs of the state's rows
    __shared__ __align__(16) _Float16 sk[NT][kChunk * KS], sq[NT][kChunk * KS];
    __shared__ __align__(16) _Float16 sm[2][kChunk * TS], stt[2][DELTA ? kChunk * TS : 8];
    __shared__ __align__(16) float sf[4][kChunk];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, c = lane >> 4;
    const int blocks = (a.Dv + 63) / 64;
    const int cb = blockIdx.x % blocks, hv = blockIdx.x / blocks % a.Hv, b = blockIdx.x / blocks / a.Hv;
    const Span sp = span_of(a, b);
    if (sp.n <= a.nshort) return;
    const int hk = hv / a.rep, col0 = 64 * cb + 16 * wave, col = col0 + r16;
    const bool mine = col0 < a.Dv;  // 16 columns are there or not, for the whole wave
    const int nchunk = (sp.n + kChunk - 1) / kChunk, slot0 = sp.q0 / kChunk + b;
    const int64_t at = ((int64_t)b * a.Hv + hv) * DK * a.Dv + col;

    f4 S[ST];
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            S[t][e] = mine && a.s_in ? a.s_in[at + (int64_t)(16 * t + 4 * c + e) * a.Dv] : 0.0f;

    u4 kr[NK], qr[NK], mr[NM], tr[DELTA ? NM : 1];
    float fr, ku, qu;
    f4 v[4];
    const auto load = [&](int ch) {
        const int64_t ck = (int64_t)(slot0 + ch) * a.Hk + hk, cv = (int64_t)(slot0 + ch) * a.Hv + hv;
        const u4* kp = reinterpret_cast<const u4*>(a.kf + ck * (NT * kChunk * DK));
        const u4* qp = reinterpret_cast<const u4*>(a.qf + ck * (NT * kChunk * DK));
        const u4* mp = reinterpret_cast<const u4*>(a.mf + cv * (2 * kChunk * kChunk));
        const u4* tp = reinterpret_cast<const u4*>(a.tf + cv * (2 * kChunk * kChunk));
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            kr[i] = kp[tid + 256 * i];
            qr[i] = qp[tid + 256 * i];
        }
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            mr[i] = mp[tid + 256 * i];
            if constexpr (DELTA) tr[i] = tp[tid + 256 * i];
        }
        fr = a.fac[cv * (4 * kChunk) + tid];
        ku = a.unit[2 * ck];
        qu = a.unit[2 * ck + 1];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = kChunk * ch + 16 * t + 4 * c + e;
                v[t][e] = mine && i < sp.n ? load1(a.v, a.dt, (int64_t)(sp.q0 + i) * a.v_token + hv * a.v_head + col) : 0.0f;
            }
    };
    load(0);

    for (int ch = 0; ch < nchunk; ++ch) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            constexpr int per = DK / 8;
            const int x = tid + 256 * i, row = x / per, half = row / kChunk;
            *reinterpret_cast<u4*>(sk[half] + (row % kChunk) * KS + 8 * (x % per)) = kr[i];
            *reinterpret_cast<u4*>(sq[half] + (row % kChunk) * KS + 8 * (x % per)) = qr[i];
        }
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            const int x = tid + 256 * i, row = x / 8, half = row / kChunk;
            *reinterpret_cast<u4*>(sm[half] + (row % kChunk) * TS + 8 * (x % 8)) = mr[i];
            if constexpr (DELTA) *reinterpret_cast<u4*>(stt[half] + (row % kChunk) * TS + 8 * (x % 8)) = tr[i];
        }
        sf[tid >> 6][tid & 63] = fr;
        const float kunit = ku, qunit = qu;
        f4 x[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = v[t];
        __syncthreads();
        if (ch + 1 < nchunk) load(ch + 1);

        // K S and Q S.
        h8 sh[SS], sl[SS];
        const float sunit = to_operand<ST>(S, sh, sl);
        f4 ks[4], qs[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            ks[t] = qs[t] = (f4){0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < SS; ++s) {
                const int p = (16 * t + r16) * KS + 32 * s + 4 * c;
                const h8 qh = read_rows(sq[0] + p);
                qs[t] = mfma16(qh, sl[s], mfma16(qh, sh[s], qs[t]));
                if constexpr (LO) qs[t] = mfma16(read_rows(sq[NT - 1] + p), sh[s], qs[t]);
                if constexpr (DELTA) {
                    const h8 kh = read_rows(sk[0] + p);
                    ks[t] = mfma16(kh, sl[s], mfma16(kh, sh[s], ks[t]));
                    if constexpr (LO) ks[t] = mfma16(read_rows(sk[NT - 1] + p), sh[s], ks[t]);
                }
            }
        }
        h8 uh[2], ul[2];
        f4 u[4];
        if constexpr (DELTA) {
            const float w = kunit * sunit;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f4 eg = *reinterpret_cast<const f4*>(&sf[0][16 * t + 4 * c]);
                const f4 be = *reinterpret_cast<const f4*>(&sf[1][16 * t + 4 * c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[t][e] = be[e] * __builtin_fmaf(-eg[e] * w, ks[t][e], x[t][e]);
            }
            h8 xh[2], xl[2];
            const float xunit = to_operand<4>(x, xh, xl);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                f4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s <= t / 2; ++s) {
                    const int p = (16 * t + r16) * TS + 32 * s + 4 * c;
                    const h8 th = read_rows(stt[0] + p), tl = read_rows(stt[1] + p);
                    acc = mfma16(tl, xh[s], mfma16(th, xl[s], mfma16(th, xh[s], acc)));
                }
                const f4 tw = *reinterpret_cast<const f4*>(&sf[3][16 * t + 4 * c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) u[t][e] = acc[e] * (tw[e] * xunit);
            }
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) u[t] = x[t];
        }
        const float uunit = to_operand<4>(u, uh, ul);
        // O = scale (e^G Q S + M U).
        {
            const float w1 = qunit * sunit * a.scale, w2 = kunit * qunit * uunit * a.scale;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                f4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s <= t / 2; ++s) {
                    const int p = (16 * t + r16) * TS + 32 * s + 4 * c;
                    const h8 mh = read_rows(sm[0] + p), ml = read_rows(sm[1] + p);
                    acc = mfma16(ml, uh[s], mfma16(mh, ul[s], mfma16(mh, uh[s], acc)));
                }
                const f4 eg = *reinterpret_cast<const f4*>(&sf[0][16 * t + 4 * c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = kChunk * ch + 16 * t + 4 * c + e;
                    const float y = __builtin_fmaf(eg[e] * w1, qs[t][e], acc[e] * w2);
                    if (mine && i < sp.n) store1(a.o, a.dt, (int64_t)(sp.q0 + i) * a.o_token + hv * a.o_head + col, y);
                }
            }
        }
        // S = e^{G_C} S + K^T (e^{G_C - G} U).
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f4 de = *reinterpret_cast<const f4*>(&sf[2][16 * t + 4 * c]);
#pragma unroll
            for (int e = 0; e < 4; ++e) u[t][e] *= de[e];
        }
        const float dunit = to_operand<4>(u, uh, ul) * kunit, all = sf[0][kChunk - 1];
#pragma unroll
        for (int t = 0; t < ST; ++t) {
            f4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int p = (32 * s + 4 * c + (r16 >> 2)) * KS + 16 * t + 4 * (r16 & 3);
                const h8 kh = join(read_tr(sk[0] + p), read_tr(sk[0] + p + 16 * KS));
                acc = mfma16(kh, ul[s], mfma16(kh, uh[s], acc));
                if constexpr (LO) {
                    const h8 kl = join(read_tr(sk[NT - 1] + p), read_tr(sk[NT - 1] + p + 16 * KS));
                    acc = mfma16(kl, uh[s], acc);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) S[t][e] = __builtin_fmaf(all, S[t][e], acc[e] * dunit);
        }
    }
    if (!mine) return;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) a.s_out[at + (int64_t)(16 * t + 4 * c + e) * a.Dv] = S[t][e];
}

// ------------------------------------------------------------------ host

struct GlaPlan {
    bool chunks;
    int nslots;
    size_t kf, mf, unit, fac, bytes;
};

GlaPlan plan_gla(int T, int B, int Hk, int Hv, int Dk, int dtype, bool cu, bool delta) {
    GlaPlan p{};
    p.chunks = cu && T > kShort;
    if (!p.chunks) return p;
    p.nslots = T / kChunk + B;
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    p.kf = up((size_t)p.nslots * Hk * (dtype == kF32 ? 2 : 1) * kChunk * Dk * 2);
    p.mf = up((size_t)p.nslots * Hv * 2 * kChunk * kChunk * 2);
    p.unit = up((size_t)p.nslots * Hk * 8);
    p.fac = up((size_t)p.nslots * Hv * 4 * kChunk * 4);
    p.bytes = 2 * p.kf + (delta ? 2 : 1) * p.mf + p.unit + p.fac;
    return p;
}

template <int DK, bool LO, bool DELTA>
void launch3(const GlaArgs& a, const GlaPlan& p, hipStream_t st) {
    if (p.chunks) {
        gla_intra_kernel<DK, LO, DELTA><<<(unsigned)p.nslots * a.Hk, 256, 0, st>>>(a);
        gla_inter_kernel<DK, LO, DELTA><<<(unsigned)a.B * a.Hv * ((a.Dv + 63) / 64), 256, 0, st>>>(a);
    }
    const int64_t waves = (int64_t)a.B * a.Hv * (a.Dv / 16);
    if (a.nshort >= 0) gla_step_kernel<DK><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(a);
}

template <int DK>
void launch1(const GlaArgs& a, const GlaPlan& p, hipStream_t st) {
    const bool lo = a.dt == kF32;
    if (a.beta) lo ? launch3<DK, true, true>(a, p, st) : launch3<DK, false, true>(a, p, st);
    else lo ? launch3<DK, true, false>(a, p, st) : launch3<DK, false, false>(a, p, st);
}

bool check(int T, int B, int Hk, int Hv, int Dk, int Dv, int dtype, bool cu) {
    if (T < 0 || B < 0 || Hk < 1 || Hv < 1 || Hv > 65536 || Hv % Hk || (Dk != 64 && Dk != 128) || Dv < 16 || Dv > 1024 ||
        Dv % 16 || dtype < kF32 || dtype > kF16 || (!cu && T != B)) {
        bq_set_error("gated_linear_attention: needs value heads in multiples of the key heads, key dimension 64 or 128, "
                     "value dimension a multiple of 16 up to 1024, a type of 0 to 2, and one token a sequence where no "
                     "offsets are given (got %d tokens, %d sequences, %d and %d heads of %d and %d, type %d)",
                     T, B, Hk, Hv, Dk, Dv, dtype);
        return false;
    }
    // Workgroups are counted in 32 bits.
    if (((int64_t)T / kChunk + B) * Hk > INT32_MAX / 2 || (int64_t)B * Hv * (Dv / 16) > INT32_MAX / 2) {
        bq_set_error("gated_linear_attention: %d tokens in %d sequences are too many for one call", T, B);
        return false;
    }
    return true;
}

}  // namespace

extern "C" {

int64_t i4_gated_linear_attention_workspace(int T, int B, int k_heads, int v_heads, int k_dim, int v_dim, int dtype,
                                            int has_cu, int has_beta) {
    if (!check(T, B, k_heads, v_heads, k_dim, v_dim, dtype, has_cu != 0)) return -2;
    return (int64_t)plan_gla(T, B, k_heads, v_heads, k_dim, dtype, has_cu != 0, has_beta != 0).bytes;
}

int i4_gated_linear_attention_dev(const void* dQ, int64_t q_token, int64_t q_head, const void* dK, int64_t k_token,
                                  int64_t k_head, const void* dV, int64_t v_token, int64_t v_head, const float* dG,
                                  int64_t g_token, const float* dBeta, int64_t beta_token, int T, int k_heads,
                                  int v_heads, int k_dim, int v_dim, int dtype, const int32_t* dCu, int B, float scale,
                                  const float* dStateIn, float* dStateOut, void* dOut, int64_t o_token, int64_t o_head,
                                  void* dWork, int64_t work_bytes, void* stream) {
    if (!check(T, B, k_heads, v_heads, k_dim, v_dim, dtype, dCu != nullptr)) return -2;
    if (B == 0) return 0;
    if (!dStateOut || (T > 0 && (!dQ || !dK || !dV || !dG || !dOut))) {
        bq_set_error("gated_linear_attention: null device pointer");
        return -2;
    }
    GlaArgs a{};
    a.q = dQ;
    a.k = dK;
    a.v = dV;
    a.o = dOut;
    a.q_token = q_token;
    a.q_head = q_head;
    a.k_token = k_token;
    a.k_head = k_head;
    a.v_token = v_token;
    a.v_head = v_head;
    a.o_token = o_token;
    a.o_head = o_head;
    a.g = dG;
    a.g_token = g_token;
    a.beta = dBeta;
    a.beta_token = beta_token;
    a.s_in = dStateIn;
    a.s_out = dStateOut;
    a.cu = dCu;
    a.T = T;
    a.B = B;
    a.Hk = k_heads;
    a.Hv = v_heads;
    a.rep = v_heads / k_heads;
    a.Dv = v_dim;
    a.dt = dtype;
    a.scale = scale;
    const GlaPlan p = plan_gla(T, B, k_heads, v_heads, k_dim, dtype, dCu != nullptr, dBeta != nullptr);
    if (p.bytes > 0 && (!dWork || work_bytes < (int64_t)p.bytes)) {
        bq_set_error("gated_linear_attention: needs a workspace of %zu bytes, got %lld", p.bytes, (long long)work_bytes);
        return -4;
    }
    a.nslots = p.nslots;
    // One sequence alone is never worth a third launch that may find nothing to do.
    a.nshort = !p.chunks ? 1 << 30 : B == 1 ? -1 : kShort;
    uint8_t* w = static_cast<uint8_t*>(dWork);
    a.kf = reinterpret_cast<_Float16*>(w);
    a.qf = reinterpret_cast<_Float16*>(w + p.kf);
    a.mf = reinterpret_cast<_Float16*>(w + 2 * p.kf);
    a.tf = reinterpret_cast<_Float16*>(w + 2 * p.kf + p.mf);
    w += 2 * p.kf + (dBeta ? 2 : 1) * p.mf;
    a.unit = reinterpret_cast<float*>(w);
    a.fac = reinterpret_cast<float*>(w + p.unit);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (k_dim == 64) launch1<64>(a, p, st);
    else launch1<128>(a, p, st);
    return launched("gated_linear_attention") ? 0 : -5;
}

}  // extern "C"
