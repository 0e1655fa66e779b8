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
//   (I + A) U = diag(beta) (V - diag(e^G) K S_0) = diag(beta) X,
//   A_ij = beta_i e^{G_i - G_j} (k_i . k_j)  for j < i,
//   O = scale (diag(e^G) Q S_0 + M U),  M_ij = e^{G_i - G_j} (q_i . k_j)  for j <= i,
//   S_C = e^{G_C} S_0 + sum_j e^{G_C - G_j} k_j u_j^T.
//
// gla_intra_kernel computes T = (I + A)^{-1} diag(beta) and M for all chunks at once;
// gla_inter_kernel walks a sequence's chunks with S in registers, 16 of its
// columns a wave.
//
// Numerics.  Products run on the fp16 matrix instructions with each operand
// as two fp16 terms (hi, and what hi leaves; 22 bits and more) and three
// products, fp32 sums; q and k given as bf16 or fp16 are one term, and so are
// the state and U where they only make rows of O of bf16 (11 bits, three more than
// those keep; the state itself and U go on with two).  A power
// of two for each tile (of q and k: each chunk and head) or column puts the
// largest value where fp16 has room; what a second term cannot hold then is
// 2^-28 of a chunk's largest q or k, 2^-37 of a column's largest.  T is computed in fp32.  Sums of g are taken in
// 64 bits: e^{G_i - G_j} would lose what G_i and G_j have in common.
#include "mix_common.h"

#include <algorithm>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

constexpr int kChunk = 64;
constexpr int kShort = 16;
constexpr int kFac = 256;  // 2 * 64 + 4, and what one load to LDS brings

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
    uint8_t* kq;        // [slots][Hk]: operands of k (hi, lo), then of q
    uint8_t* tm;        // [slots][Hv]: operands of M (hi, lo), then of T
    // [slots][Hv][kFac]: e^G, e^{G_C - G}, what a unit of T's, k's and q's operands is worth,
    // and the first row whose k, g or beta is no finite number (64: none).
    float* fac;
    int slot0, slot1;   // the chunks' slots that the workspace holds now
    int T, B, Hk, Hv, rep, Dv, dt;
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

// One element as it is stored, and its value.
template <int DT>
__device__ inline uint32_t raw1(const void* p, int64_t i) {
    if constexpr (DT == kF32) return static_cast<const uint32_t*>(p)[i];
    else return static_cast<const uint16_t*>(p)[i];
}
template <int DT>
__device__ inline float value1(uint32_t w) {
    if constexpr (DT == kF32) return bits_f(w);
    else if constexpr (DT == kBF16) return bits_f(w << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
}
template <int DT>
__device__ inline void store1(void* p, int64_t i, float x) {
    if constexpr (DT == kF32) static_cast<float*>(p)[i] = x;
    else if constexpr (DT == kBF16) static_cast<uint16_t*>(p)[i] = (uint16_t)to_bf16(x);
    else static_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, (_Float16)x);
}

// A decay's logarithm; -infinity (a state that is dropped) as a number whose
// exponential is zero and whose sums stay exact.
__device__ inline float clean_g(float g) { return g < -1e4f ? -1e4f : g; }

// ------------------------------------------------------------------ short sequences

// Bound by HBM: 64 tokens of 48 heads, 128 x 128 states (403 MB): 84 to 88 us,
// 4.6 to 4.8 TB/s, the rate of a large copy.  One token: 4.8 us.
//
// A wave for 16 columns of one sequence's and head's state: lane (row r mod 16,
// four columns).  Before the update both S^T k and S^T q are summed over the
// rows, since S_t^T q = e^g S_{t-1}^T q + (k . q) u: one exchange a token.
template <int DK, int DT>
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
            kv[i] = value1<DT>(raw1<DT>(a.k, t * a.k_token + hk * a.k_head + r0 + 16 * i));
            qv[i] = value1<DT>(raw1<DT>(a.q, t * a.q_token + hk * a.q_head + r0 + 16 * i));
        }
        const f4 v = load4(a.v, DT, t * a.v_token + hv * a.v_head + col);
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
        if (r0 == 0) store4(a.o, DT, t * a.o_token + hv * a.o_head + col, o);
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
constexpr uint32_t kInfBits = 0x7F800000u;  // and above: NaN

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

typedef __attribute__((address_space(3))) s4* lds_s4;
__device__ inline h4 read_tr(const void* p) {
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p)));
}
__device__ inline h8 join(h4 a, h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// Columns 4 c + 0..3 and 16 + 4 c + 0..3 of a row, from its column 4 c.
__device__ inline h8 read_rows(const _Float16* p) {
    return join(*reinterpret_cast<const h4*>(p), *reinterpret_cast<const h4*>(p + 16));
}

// Operands between the kernels.  A 16 x 32 operand of the matrix instruction is
// 1 KB, 16 bytes a lane (row r, quarter c): columns 4 c + 0..3 and 16 + 4 c +
// 0..3, the order in which a result's rows come as the other operand.  Lane
// (r, c)'s 16 bytes lie at place 16 c + (r ^ 4 (c & 1)), which also lets the
// transposed reads of k for the state's update touch twice the banks.
__device__ inline int place(int r, int c) { return 16 * c + (r ^ ((c & 1) << 2)); }

// T and M are lower triangular: row tile t has column slabs 0 .. t / 2, six
// operands in all.
constexpr int kTri = 6;
constexpr int kTriBytes = kTri * 1024;
__host__ __device__ constexpr int tri(int t, int s) { return t + (t == 3) + s; }

constexpr int kq_bytes(int dk, bool lo) { return 2 * (lo ? 2 : 1) * 4 * (dk / 32) * 1024; }
constexpr int tm_bytes(bool delta) { return (delta ? 4 : 2) * kTriBytes; }

// One workgroup for a chunk and a key head: the products k_i . k_j and
// q_i . k_j once, then T and M for each of its value heads.  64 chunks of 16 key
// and 48 value heads, fp32: 60 us, of which 28 for the operands of k and q (134
// MB in and out) and 10 for each value head's T and M (25 KB a chunk and head
// out, and a chain of small triangular products).
template <int DK, int DT, bool DELTA>
__global__ __launch_bounds__(256, 2) void gla_intra_kernel(GlaArgs a) {
    constexpr bool LO = DT == kF32;  // two terms of q and k
    constexpr int KS = DK + 8, AS = kChunk + 4, L = DK / 4, NP = kChunk * L / 256, SS = DK / 32;
    constexpr int NT = LO ? 2 : 1;
    constexpr int kIn = 2 * NT * kChunk * KS * 2, kOut = (DELTA ? 3 : 1) * kChunk * AS * 4;
    __shared__ __align__(16) uint8_t lds[kIn > kOut ? kIn : kOut];
    __shared__ double sg[kChunk];
    __shared__ __align__(16) float sbeta[kChunk];
    __shared__ uint32_t stop[2][4];
    __shared__ int sbad[4];
    _Float16* const in = reinterpret_cast<_Float16*>(lds);  // k hi, k lo, q hi, q lo
    _Float16* const sk = in;
    _Float16* const sq = in + NT * kChunk * KS;
    constexpr int kLow = (NT - 1) * kChunk * KS;
    float* const sm = reinterpret_cast<float*>(lds);  // once the products are done
    float* const sa = sm + kChunk * AS;
    float* const st = sa + kChunk * AS;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % a.Hk, slot = blockIdx.x / a.Hk;  // counted from slot0 on
    int tok, n;
    if (!chunk_of(a, a.slot0 + slot, tok, n)) return;

    // q and k, scaled to [2^3, 2^4) so that their products fit fp16 too.
    f4 kx[NP], qx[NP];
    uint32_t kt = 0, qt = 0;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int row = (tid + 256 * i) / L, d = 4 * (tid % L);
        const int64_t at = tok + min(row, n - 1);
        kx[i] = load4(a.k, DT, at * a.k_token + hk * a.k_head + d);
        qx[i] = load4(a.q, DT, at * a.q_token + hk * a.q_head + d);
    }
    // A k that is no finite number enters no product, whose zeros it would spoil for the rows
    // before it: its row and those after it are made NaN at the end.  A q spoils its own row only.
    int bad = kChunk;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int row = (tid + 256 * i) / L;
        if (row >= n) kx[i] = qx[i] = (f4){0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t x = abs_bits(kx[i][j]), y = abs_bits(qx[i][j]);
            if (x >= kInfBits) {
                kx[i][j] = 0.0f;
                bad = min(bad, row);
            } else {
                kt = max(kt, x);
            }
            qt = max(qt, y < kInfBits ? y : 0u);
        }
    }
    if (__any(bad < kChunk))
#pragma unroll
        for (int s = 1; s < 64; s *= 2) bad = min(bad, __shfl_xor(bad, s));
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        kt = max(kt, (uint32_t)__shfl_xor((int)kt, s));
        qt = max(qt, (uint32_t)__shfl_xor((int)qt, s));
    }
    if (lane == 0) {
        stop[0][wave] = kt;
        stop[1][wave] = qt;
        sbad[wave] = bad;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        kt = max(kt, stop[0][w]);
        qt = max(qt, stop[1][w]);
        bad = min(bad, sbad[w]);
    }
    const float kup = to_top<3>(kt), qup = to_top<3>(qt), kunit = inverse_pow2(kup), qunit = inverse_pow2(qup);
    const int64_t ck = (int64_t)slot * a.Hk + hk;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int row = (tid + 256 * i) / L, d = 4 * (tid % L);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            f4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = w ? qx[i][j] * qup : kx[i][j] * kup;
            const h4 hi = __builtin_convertvector(x, h4);
            _Float16* s = (w ? sq : sk) + row * KS + d;
            *reinterpret_cast<h4*>(s) = hi;
            if constexpr (LO) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] -= (float)hi[j];
                *reinterpret_cast<h4*>(s + kLow) = __builtin_convertvector(x, h4);
            }
        }
    }
    __syncthreads();

    // The other kernel's operands of k and q.
    {
        h8* out = reinterpret_cast<h8*>(a.kq + ck * kq_bytes(DK, LO));
#pragma unroll
        for (int i = 0; i < 2 * NT * 4 * SS / 4; ++i) {
            const int f = 4 * i + wave, part = f / (4 * SS), t = f % (4 * SS) / SS, s = f % SS;
            const int c = lane >> 4, r = (lane & 15) ^ ((c & 1) << 2);
            out[f * 64 + lane] = read_rows(in + part * kChunk * KS + (16 * t + r) * KS + 32 * s + 4 * c);
        }
    }

    // Wave w: rows 16 w ..; columns up to them.
    const int r16 = lane & 15, c = lane >> 4;
    f4 kk[4], qk[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) kk[t] = qk[t] = (f4){0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < SS; ++s) {
        const int ar = (16 * wave + r16) * KS + 32 * s + 8 * c;
        const h8 ak = *reinterpret_cast<const h8*>(sk + ar), aq = *reinterpret_cast<const h8*>(sq + ar);
        const h8 akl = *reinterpret_cast<const h8*>(sk + kLow + ar), aql = *reinterpret_cast<const h8*>(sq + kLow + ar);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (t > wave) continue;
            const int br = (16 * t + r16) * KS + 32 * s + 8 * c;
            const h8 b = *reinterpret_cast<const h8*>(sk + br);
            if constexpr (DELTA) kk[t] = mfma16(ak, b, kk[t]);
            qk[t] = mfma16(aq, b, qk[t]);
            if constexpr (LO) {
                const h8 bl = *reinterpret_cast<const h8*>(sk + kLow + br);
                if constexpr (DELTA) kk[t] = mfma16(akl, b, mfma16(ak, bl, kk[t]));
                qk[t] = mfma16(aql, b, mfma16(aq, bl, qk[t]));
            }
        }
    }

    for (int r = 0; r < a.rep; ++r) {
        const int hv = hk * a.rep + r;
        const int64_t cv = (int64_t)slot * a.Hv + hv;
        float* fac = a.fac + cv * kFac;
        if (wave == 0) {
            const bool is = lane < n;
            float gv = is ? clean_g(a.g[(int64_t)(tok + lane) * a.g_token + hv]) : 0.0f, be = 0.0f;
            if constexpr (DELTA) be = is ? a.beta[(int64_t)(tok + lane) * a.beta_token + hv] : 0.0f;
            const uint64_t spoilt = __ballot(abs_bits(gv) >= kInfBits || abs_bits(be) >= kInfBits);
            if (abs_bits(gv) >= kInfBits) gv = 0.0f;
            if (abs_bits(be) >= kInfBits) be = 0.0f;
            if (lane == 0) fac[2 * kChunk + 3] = (float)min(bad, spoilt ? __builtin_ctzll(spoilt) : kChunk);
            double G = gv;
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const double up = __shfl_up(G, s);
                if (lane >= s) G += up;
            }
            sg[lane] = G;
            sbeta[lane] = be;
            fac[lane] = expf((float)G);
            fac[kChunk + lane] = expf((float)(__shfl(G, 63) - G));
        }
        __syncthreads();  // the first time, the products' operands are read too
        // A and M; the blocks past the diagonal that an operand reaches into are zeros.
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
                if (t > (wave | 1)) continue;
                const int j = 16 * t + r16;
                const double gj = sg[j];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 16 * wave + 4 * c + e;
                    float av = 0.0f, mv = 0.0f;
                    if (t <= wave) {
                        const float x = expf((float)(gi[e] - gj));
                        mv = j <= i ? x * qk[t][e] : 0.0f;
                        av = j < i ? bi[e] * x * kk[t][e] : 0.0f;
                    } else if (DELTA) {
                        st[i * AS + j] = 0.0f;
                    }
                    sm[i * AS + j] = mv;
                    if constexpr (DELTA) sa[i * AS + j] = av;
                }
            }
        }
        __syncthreads();
        float tup = 1.0f;
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
            // T diag(beta), its largest value to [2^12, 2^13).
            const int row = tid >> 2, q4 = 16 * (tid & 3);
            uint32_t top = 0;
            if (q4 <= row)
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const f4 x = *reinterpret_cast<const f4*>(st + row * AS + q4 + j);
                    const f4 be = *reinterpret_cast<const f4*>(sbeta + q4 + j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = max(top, abs_bits(x[e] * be[e]));
                }
#pragma unroll
            for (int s = 1; s < 64; s *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, s));
            if (lane == 0) stop[0][wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 4; ++w) top = max(top, stop[0][w]);
            tup = to_top<12>(top);
            if (tid == 0) fac[2 * kChunk] = inverse_pow2(tup);
        }
        if (tid == 0) {
            fac[2 * kChunk + 1] = kunit;
            fac[2 * kChunk + 2] = qunit;
        }
        // Out as operands of two terms.
        h8* out = reinterpret_cast<h8*>(a.tm + cv * tm_bytes(DELTA));
#pragma unroll
        for (int w = 0; w < (DELTA ? 2 : 1); ++w)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int f = 4 * i + wave;
                if (f >= kTri) continue;
                const int t = f < 2 ? f : f < 4 ? 2 : 3, s = f - tri(t, 0);
                const int cc = lane >> 4, rr = (lane & 15) ^ ((cc & 1) << 2);
                const float* p = (w ? st : sm) + (16 * t + rr) * AS + 32 * s + 4 * cc;
                f4 x = *reinterpret_cast<const f4*>(p), y = *reinterpret_cast<const f4*>(p + 16);
                if (w) {
                    x *= *reinterpret_cast<const f4*>(sbeta + 32 * s + 4 * cc) * tup;
                    y *= *reinterpret_cast<const f4*>(sbeta + 32 * s + 16 + 4 * cc) * tup;
                }
                const h4 xh = __builtin_convertvector(x, h4), yh = __builtin_convertvector(y, h4);
                const f4 xl = x - __builtin_convertvector(xh, f4), yl = y - __builtin_convertvector(yh, f4);
                out[(2 * kTri * w + f) * 64 + lane] = join(xh, yh);
                out[(2 * kTri * w + kTri + f) * 64 + lane] =
                    join(__builtin_convertvector(xl, h4), __builtin_convertvector(yl, h4));
            }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ from chunk to chunk

// The largest magnitude of a column that four lanes hold (rows 16 t + 4 c + e); of
// its numbers, or (ANY) NaN where it holds one.
template <int N, bool ANY = false>
__device__ inline float column_top(const f4* x) {
    const auto larger = [](float a, float b) { return ANY ? __builtin_elementwise_maximum(a, b) : fmaxf(a, b); };
    float top = 0.0f;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int e = 0; e < 4; e += 2) top = larger(larger(top, __builtin_fabsf(x[t][e])), __builtin_fabsf(x[t][e + 1]));
    const auto a = __builtin_amdgcn_permlane16_swap(f_bits(top), f_bits(top), false, false);
    top = larger(bits_f(a[0]), bits_f(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(f_bits(top), f_bits(top), false, false);
    return larger(bits_f(b[0]), bits_f(b[1]));
}

// x p and y q as two fp16 terms: each is one instruction, which multiplies,
// subtracts the first term in fp32 and rounds.
__device__ inline void two_terms(float x, float y, float p, float q, uint32_t& hi, uint32_t& lo) {
    uint32_t h, l;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(x), "v"(p));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(y), "v"(q));
    asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(l) : "v"(x), "v"(p), "v"(h));
    asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(l) : "v"(y), "v"(q), "v"(h));
    hi = h;
    lo = l;
}

// Values in a result's layout times `up` (times `rows`' factor for their row)
// as the operand of a contraction over those rows.  Slab s holds tiles 2 s and
// 2 s + 1.
template <int N>
__device__ inline void to_operand(const f4* x, float up, const float* rows, int c, h8* hi, h8* lo) {
#pragma unroll
    for (int s = 0; s < N / 2; ++s) {
        u4 h, l;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const f4 v = x[2 * s + j];
            f4 f = {up, up, up, up};
            if (rows) f *= *reinterpret_cast<const f4*>(rows + 16 * (2 * s + j) + 4 * c);
            uint32_t a, b;
            two_terms(v[0], v[1], f[0], f[1], a, b);
            h[2 * j] = a;
            l[2 * j] = b;
            two_terms(v[2], v[3], f[2], f[3], a, b);
            h[2 * j + 1] = a;
            l[2 * j + 1] = b;
        }
        hi[s] = __builtin_bit_cast(h8, h);
        lo[s] = __builtin_bit_cast(h8, l);
    }
}

// A lower triangular factor (T or M) of two terms times 16 columns of two, or
// (rows of O that are rounded to bf16) of one.
template <bool TWO>
__device__ inline void tri_product(const h8* hi, const h8* lo, const h8* xh, const h8* xl, f4* acc) {
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = mfma16(hi[tri(t, 0)], xh[0], (f4){0, 0, 0, 0});
    if constexpr (TWO)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = mfma16(hi[tri(t, 0)], xl[0], acc[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = mfma16(lo[tri(t, 0)], xh[0], acc[t]);
#pragma unroll
    for (int t = 2; t < 4; ++t) acc[t] = mfma16(hi[tri(t, 1)], xh[1], acc[t]);
    if constexpr (TWO)
#pragma unroll
        for (int t = 2; t < 4; ++t) acc[t] = mfma16(hi[tri(t, 1)], xl[1], acc[t]);
#pragma unroll
    for (int t = 2; t < 4; ++t) acc[t] = mfma16(lo[tri(t, 1)], xh[1], acc[t]);
}

// Four waves for 32 columns of a head's state: two carry 16 columns each from
// chunk to chunk (K S, T X, the state's update), and each hands its operands to
// one of the other two, which computes the rows of O and brings the next
// chunk's operands of k and q to LDS.  A wave of each kind a SIMD: what one
// waits for, its own next product, the other does not.
//
// Bound by the chain through the state: per chunk 114 matrix instructions
// (1,824 cycles of fp32 calls) and about as much in conversions, exchanges of
// column maxima and LDS reads between them; 3.2 us a chunk, of which the
// update's products take 0.6 and the hand-over 0.4 (64 chunks of 48 heads of
// 128 x 128, 192 workgroups: fp32 202 us, fp16 166, bf16 160).  All products in one
// wave and 64 columns a workgroup took 5.0 (the LDS reads of four waves, 480 KB,
// alone 1.6).  fp16's second terms for the rows of O leave one workgroup a unit: where
// there are many (6 sequences of 32 heads), 69 us against 54 with one term.
template <int DK, int DT, bool DELTA>
__global__ __launch_bounds__(256, DT == kF32 || (DT == kF16 && DK == 128) ? 1 : 2) void gla_inter_kernel(GlaArgs a) {
    constexpr bool LO = DT == kF32;      // two terms of q and k
    constexpr bool TWO = DT != kBF16;    // two of the state and U for the rows of O
    constexpr int NT = LO ? 2 : 1, NO = TWO ? 2 : 1, ST = DK / 16, SS = DK / 32;  // tiles and slabs of the state's rows
    constexpr int kPart = 4 * SS * 1024, kBuf = kq_bytes(DK, LO);
    __shared__ __align__(1024) uint8_t skq[2][kBuf];       // operands of k, then of q
    // What the state's waves hand over: the state's operands and U's, one term of each
    // for rows of O that are rounded to bf16 (80 KB of LDS in all: two workgroups a unit).
    __shared__ __align__(1024) uint8_t ss[2][NO * SS * 1024];
    __shared__ __align__(1024) uint8_t su[2][NO * 2 * 1024];
    __shared__ __align__(1024) float sf[2][kFac];
    __shared__ float sunits[2][2][16];  // what a unit of those is worth, for each column
    __shared__ int sbad[2][16];         // a column's first row whose k, v, g or beta is no finite number

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pair = wave & 1, r16 = lane & 15, c = lane >> 4;
    // A head's workgroups are B * Hv apart: on one XCD, whose L2 then holds what they share, wherever 8 divides that.
    const int heads = a.B * a.Hv, cb = blockIdx.x / heads, hv = blockIdx.x % heads % a.Hv, b = blockIdx.x % heads / a.Hv;
    const Span sp = span_of(a, b);
    if (sp.n <= a.nshort) return;
    const int hk = hv / a.rep, col0 = 32 * cb + 16 * pair;
    const bool mine = col0 < a.Dv;  // 16 columns are there or not, for the whole wave
    const int col = (mine ? col0 : 0) + r16;
    // Its chunks whose slots are here; one without any writes its state in the first segment.
    const int chunks = (sp.n + kChunk - 1) / kChunk, slot0 = sp.q0 / kChunk + b - a.slot0;
    const int begin = max(-slot0, 0), nchunk = min(chunks, a.slot1 - a.slot0 - slot0);
    if (begin >= nchunk && (chunks > 0 || a.slot0 > 0)) return;
    const int64_t at = ((int64_t)b * a.Hv + hv) * DK * a.Dv + col;
    const int rd = 16 * place(r16, c);  // where the lane's 16 bytes of an operand lie
    const auto op = [&](const uint8_t* base, int f) { return *reinterpret_cast<const h8*>(base + 1024 * f + rd); };
    const auto tm_of = [&](int ch) { return a.tm + ((int64_t)(slot0 + ch) * a.Hv + hv) * tm_bytes(DELTA); };

    if (wave >= 2) {  // ---------------------------------------------------- the rows of O
        // k's and q's operands and the factors of chunk ch, on their way.
        const auto fetch = [&](int ch, int part) {  // a quarter of them
            const uint8_t* src = a.kq + ((int64_t)(slot0 + ch) * a.Hk + hk) * kBuf + 1024 * pair + 16 * lane;
            const uint32_t dst = lds_address(skq[ch & 1]) + 1024 * pair;
#pragma unroll
            for (int i = 0; i < kBuf / 8192; ++i)
                load_lds(src + 2048 * (4 * i + part), dst + 2048 * (4 * i + part));
            if (pair == 0 && part == 0)
                load_lds(reinterpret_cast<const uint8_t*>(a.fac + ((int64_t)(slot0 + ch) * a.Hv + hv) * kFac) + 16 * lane,
                         lds_address(sf[ch & 1]));
        };
        f4 y[4];
        const auto store = [&](int ch, bool full) {
            const int first = kChunk * ch + 4 * c;
            const int64_t p = (int64_t)(sp.q0 + first) * a.o_token + hv * a.o_head + col;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (full || first + 16 * t + e < sp.n) store1<DT>(a.o, p + (16 * t + e) * a.o_token, y[t][e]);
        };
        if (begin < nchunk)
#pragma unroll
            for (int i = 0; i < 4; ++i) fetch(begin, i);
        wait_loads<0>();
        __syncthreads();
        for (int ch = begin; ch < nchunk; ++ch) {
            h8 mh[kTri], ml[kTri];
            const h8* mp = reinterpret_cast<const h8*>(tm_of(ch));
#pragma unroll
            for (int f = 0; f < kTri; ++f) {
                mh[f] = mp[64 * f + rd / 16];
                ml[f] = mp[64 * (kTri + f) + rd / 16];
            }
            // Q S: the operands of one slab are read while those of the one before it are multiplied.
            const uint8_t* const qb = skq[ch & 1] + NT * kPart;
            f4 qs[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) qs[t] = (f4){0, 0, 0, 0};
            h8 oh[2][4], ol[2][4], sh[2], sl[2];
            const auto get = [&](int s) {
                sh[s & 1] = *reinterpret_cast<const h8*>(ss[pair] + 1024 * s + 16 * lane);
                if constexpr (TWO) sl[s & 1] = *reinterpret_cast<const h8*>(ss[pair] + 1024 * (SS + s) + 16 * lane);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    oh[s & 1][t] = op(qb, t * SS + s);
                    if constexpr (LO) ol[s & 1][t] = op(qb + kPart, t * SS + s);
                }
            };
            get(0);
#pragma unroll
            for (int s = 0; s < SS; ++s) {
                if (s + 1 < SS) get(s + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < 4; ++t) qs[t] = mfma16(oh[s & 1][t], sh[s & 1], qs[t]);
                if constexpr (TWO)
#pragma unroll
                    for (int t = 0; t < 4; ++t) qs[t] = mfma16(oh[s & 1][t], sl[s & 1], qs[t]);
                if constexpr (LO)
#pragma unroll
                    for (int t = 0; t < 4; ++t) qs[t] = mfma16(ol[s & 1][t], sh[s & 1], qs[t]);
                if (ch + 1 < nchunk)
#pragma unroll
                    for (int i = 4 * s / SS; i < 4 * (s + 1) / SS; ++i) fetch(ch + 1, i);
                __builtin_amdgcn_sched_barrier(0);
            }
            const float* const fac = sf[ch & 1];
            const float w1 = fac[2 * kChunk + 2] * sunits[0][pair][r16] * a.scale;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f4 eg = *reinterpret_cast<const f4*>(fac + 16 * t + 4 * c);
#pragma unroll
                for (int e = 0; e < 4; ++e) qs[t][e] *= eg[e] * w1;
            }
            const float w2 = fac[2 * kChunk + 1] * fac[2 * kChunk + 2] * a.scale;
            __syncthreads();  // U is there
            h8 uh[2], ul[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uh[s] = *reinterpret_cast<const h8*>(su[pair] + 1024 * s + 16 * lane);
                if constexpr (TWO) ul[s] = *reinterpret_cast<const h8*>(su[pair] + 1024 * (2 + s) + 16 * lane);
            }
            const float w3 = w2 * sunits[1][pair][r16];
            f4 acc[4];
            tri_product<TWO>(mh, ml, uh, ul, acc);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[t][e] = __builtin_fmaf(acc[t][e], w3, qs[t][e]);
            const int bad = sbad[pair][r16];
            if (__any(bad < kChunk))
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * t + 4 * c + e >= bad) y[t][e] = __builtin_nanf("");
            // The stores come last and stay on their way; the loads before them are waited for.
            if (ch + 1 < nchunk) {
                if (mine) {
                    store(ch, true);
                    wait_loads<16>();
                } else {
                    wait_loads<0>();
                }
            } else if (mine) {
                store(ch, sp.n >= kChunk * nchunk);
            }
            __syncthreads();  // the next state is there, and the next chunk's operands
        }
        return;
    }

    // ------------------------------------------------------------------ the state
    f4 S[ST];  // the state is S times sworth
    float sworth = 1.0f;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[t][e] = 0.0f;
    const float* const from = begin > 0 ? a.s_out : a.s_in;  // the segment before left it there
    if (from)
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[t][e] = from[at + (int64_t)(16 * t + 4 * c + e) * a.Dv];

    uint32_t v[4][4];
    const auto load_v = [&](int ch) {
        const int first = kChunk * ch + 4 * c;
        if (kChunk * (ch + 1) <= sp.n) {
            const int64_t p = (int64_t)(sp.q0 + first) * a.v_token + hv * a.v_head + col;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[t][e] = raw1<DT>(a.v, p + (16 * t + e) * a.v_token);
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[t][e] = raw1<DT>(a.v, (int64_t)(sp.q0 + min(first + 16 * t + e, sp.n - 1)) * a.v_token +
                                                hv * a.v_head + col);
        }
    };
    h8 th[kTri], tl[kTri];
    const auto load_t = [&](int ch) {
        const h8* tp = reinterpret_cast<const h8*>(tm_of(ch) + 2 * kTriBytes);
#pragma unroll
        for (int f = 0; f < kTri; ++f) {
            th[f] = tp[64 * f + rd / 16];
            tl[f] = tp[64 * (kTri + f) + rd / 16];
        }
    };
    h8 sh[SS], sl[SS];
    float sunit;
    const auto hand_over = [&]() {
        const float up = to_top<12>(f_bits(column_top<ST>(S)));
        sunit = inverse_pow2(up) * sworth;
        to_operand<ST>(S, up, nullptr, c, sh, sl);
#pragma unroll
        for (int s = 0; s < SS; ++s) {
            *reinterpret_cast<h8*>(ss[pair] + 1024 * s + 16 * lane) = sh[s];
            if constexpr (TWO) *reinterpret_cast<h8*>(ss[pair] + 1024 * (SS + s) + 16 * lane) = sl[s];
        }
        if (c == 0) sunits[0][pair][r16] = sunit;
    };
    if (begin < nchunk) {
        load_v(begin);
        if constexpr (DELTA) load_t(begin);
    }
    hand_over();
    __syncthreads();

    // The transposed reads: key 4 c + r16 / 4 of a tile, values 4 (r16 & 3) + 0..3 of 16.
    const int rt = 16 * place(4 * c + (r16 >> 2), r16 & 3);
    for (int ch = begin; ch < nchunk; ++ch) {
        const uint8_t* const kb = skq[ch & 1];
        const float* const fac = sf[ch & 1];
        const float kunit = fac[2 * kChunk + 1];
        const int kgb_bad = (int)fac[2 * kChunk + 3];
        f4 u[4];  // U is u times uworth
        float uworth = 1.0f;
        f4 x[4];
        const int left = sp.n - kChunk * ch - 4 * c;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[t][e] = 16 * t + e < left ? value1<DT>(v[t][e]) : 0.0f;
        if constexpr (DELTA) {
            f4 ks[4], eg[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                ks[t] = (f4){0, 0, 0, 0};
                eg[t] = *reinterpret_cast<const f4*>(fac + 16 * t + 4 * c);
            }
            h8 oh[2][4], ol[2][4];
            const auto get = [&](int s) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    oh[s & 1][t] = op(kb, t * SS + s);
                    if constexpr (LO) ol[s & 1][t] = op(kb + kPart, t * SS + s);
                }
            };
            get(0);
#pragma unroll
            for (int s = 0; s < SS; ++s) {
                if (s + 1 < SS) get(s + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < 4; ++t) ks[t] = mfma16(oh[s & 1][t], sh[s], ks[t]);
#pragma unroll
                for (int t = 0; t < 4; ++t) ks[t] = mfma16(oh[s & 1][t], sl[s], ks[t]);
                if constexpr (LO)
#pragma unroll
                    for (int t = 0; t < 4; ++t) ks[t] = mfma16(ol[s & 1][t], sh[s], ks[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
            const float w = -kunit * sunit;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[t][e] = __builtin_fmaf(eg[t][e] * w, ks[t][e], x[t][e]);
        }
        // What is no finite number stays out of the products, whose zeros it would spoil for the
        // column's earlier rows: its row and those after it are made NaN at the end.
        float xtop = column_top<4, true>(x), utop;
        int bad = kChunk;
        if (__builtin_expect(__any(!(xtop < INFINITY)), 0)) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (abs_bits(x[t][e]) >= kInfBits) {
                        x[t][e] = 0.0f;
                        bad = min(bad, 16 * t + 4 * c + e);
                    }
            bad = min(bad, __shfl_xor(bad, 16));
            bad = min(bad, __shfl_xor(bad, 32));
            xtop = column_top<4>(x);
        }
        if constexpr (DELTA) {
            h8 xh[2], xl[2];
            const float xup = to_top<12>(f_bits(xtop));
            to_operand<4>(x, xup, nullptr, c, xh, xl);
            tri_product<true>(th, tl, xh, xl, u);
            uworth = fac[2 * kChunk] * inverse_pow2(xup);
            utop = column_top<4>(u);
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) u[t] = x[t];
            utop = xtop;
        }
        bad = min(bad, kgb_bad);
        const float uup = to_top<12>(f_bits(utop)), uunit = inverse_pow2(uup) * uworth;
        h8 uh[2], ul[2];
        to_operand<4>(u, uup, nullptr, c, uh, ul);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            *reinterpret_cast<h8*>(su[pair] + 1024 * s + 16 * lane) = uh[s];
            if constexpr (TWO) *reinterpret_cast<h8*>(su[pair] + 1024 * (2 + s) + 16 * lane) = ul[s];
        }
        if (c == 0) {
            sunits[1][pair][r16] = uunit;
            sbad[pair][r16] = bad;
        }
        __syncthreads();
        if (ch + 1 < nchunk) {
            load_v(ch + 1);
            if constexpr (DELTA) load_t(ch + 1);
        }
        // S = e^{G_C} S + K^T (e^{G_C - G} U), summed in the units of this product; a
        // product too small to show beside the state does not set them (S is at most 2^13
        // sunit, so 2^93 in units of 2^-80 of that).
        {
            constexpr int GT = 2;  // tiles of the state's rows a group
            h8 oh[2][GT][2], ol[2][GT][2];
            const auto get = [&](int g) {
#pragma unroll
                for (int i = 0; i < GT; ++i)
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int t = GT * g + i;
                        const uint8_t* p = kb + ((2 * s) * SS + (t >> 1)) * 1024 + rt + 8 * (t & 1);
                        oh[g & 1][i][s] = join(read_tr(p), read_tr(p + SS * 1024));
                        if constexpr (LO) ol[g & 1][i][s] = join(read_tr(p + kPart), read_tr(p + kPart + SS * 1024));
                    }
            };
            get(0);
            const float worth = fmaxf(fmaxf(uunit * kunit, sworth * 0x1p-60f), fmaxf(sunit * 0x1p-80f, 0x1p-100f));
            to_operand<4>(u, uworth * kunit * inverse_pow2(worth), fac + kChunk, c, uh, ul);
            const float keep = fac[kChunk - 1] * (sworth * inverse_pow2(worth));
            sworth = worth;
#pragma unroll
            for (int t = 0; t < ST; ++t) S[t] *= keep;
#pragma unroll
            for (int g = 0; g < ST / GT; ++g) {
                if (g + 1 < ST / GT) get(g + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < GT; ++i) S[GT * g + i] = mfma16(oh[g & 1][i][s], uh[s], S[GT * g + i]);
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < GT; ++i) S[GT * g + i] = mfma16(oh[g & 1][i][s], ul[s], S[GT * g + i]);
                if constexpr (LO)
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int i = 0; i < GT; ++i) S[GT * g + i] = mfma16(ol[g & 1][i][s], uh[s], S[GT * g + i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (__any(bad < kChunk))
#pragma unroll
            for (int t = 0; t < ST; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[t][e] = bad < kChunk ? __builtin_nanf("") : S[t][e];
        if (ch + 1 < nchunk) hand_over();
        __syncthreads();
    }
    if (!mine) return;
#pragma unroll
    for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) a.s_out[at + (int64_t)(16 * t + 4 * c + e) * a.Dv] = S[t][e] * sworth;
}

// ------------------------------------------------------------------ host

struct GlaPlan {
    bool chunks;
    int nslots, segment;  // slots of chunks, and how many of them the workspace holds at a time
    size_t kq, tm, fac, bytes;
};

// The chunks' operands take about as much as the call's own tensors, 36 KB a token of 16/48
// heads of 128 in fp32; past these bytes they go in segments, one after the other,
// with the states in between where the call leaves them at its end.
constexpr size_t kMostOperands = (size_t)1 << 30;

GlaPlan plan_gla(int T, int B, int Hk, int Hv, int Dk, int dtype, bool cu, bool delta) {
    GlaPlan p{};
    p.chunks = cu && T > kShort;
    if (!p.chunks) return p;
    p.nslots = T / kChunk + B;
    const size_t kq = (size_t)Hk * kq_bytes(Dk, dtype == kF32), tm = (size_t)Hv * tm_bytes(delta), fac = (size_t)Hv * kFac * 4;
    p.segment = (int)std::max<size_t>(1, std::min<size_t>(p.nslots, kMostOperands / (kq + tm + fac)));
    p.kq = p.segment * kq;  // multiples of 1024 bytes
    p.tm = p.segment * tm;
    p.fac = p.segment * fac;
    p.bytes = p.kq + p.tm + p.fac;
    return p;
}

template <int DK, int DT, bool DELTA>
void launch3(GlaArgs a, const GlaPlan& p, hipStream_t st) {
    for (int at = 0; at < p.nslots; at += p.segment) {
        a.slot0 = at;
        a.slot1 = std::min(at + p.segment, p.nslots);
        gla_intra_kernel<DK, DT, DELTA><<<(unsigned)(a.slot1 - at) * a.Hk, 256, 0, st>>>(a);
        gla_inter_kernel<DK, DT, DELTA><<<(unsigned)a.B * a.Hv * ((a.Dv + 31) / 32), 256, 0, st>>>(a);
    }
    const int64_t waves = (int64_t)a.B * a.Hv * (a.Dv / 16);
    if (a.nshort >= 0) gla_step_kernel<DK, DT><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(a);
}

template <int DK, int DT>
void launch2(const GlaArgs& a, const GlaPlan& p, hipStream_t st) {
    if (a.beta) launch3<DK, DT, true>(a, p, st);
    else launch3<DK, DT, false>(a, p, st);
}

template <int DK>
void launch1(const GlaArgs& a, const GlaPlan& p, hipStream_t st) {
    if (a.dt == kF32) launch2<DK, kF32>(a, p, st);
    else if (a.dt == kBF16) launch2<DK, kBF16>(a, p, st);
    else launch2<DK, kF16>(a, p, st);
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
    // A launch has fewer than 2^24 workgroups.
    if (((int64_t)T / kChunk + B) * Hk > (1 << 23) || (int64_t)B * Hv * (Dv / 16) > (1 << 23)) {
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
    // One sequence alone is never worth a third launch that may find nothing to do.
    a.nshort = !p.chunks ? 1 << 30 : B == 1 ? -1 : kShort;
    uint8_t* w = static_cast<uint8_t*>(dWork);
    a.kq = w;
    a.tm = w + p.kq;
    a.fac = reinterpret_cast<float*>(w + p.kq + p.tm);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (k_dim == 64) launch1<64>(a, p, st);
    else launch1<128>(a, p, st);
    return launched("gated_linear_attention") ? 0 : -5;
}

}  // extern "C"
