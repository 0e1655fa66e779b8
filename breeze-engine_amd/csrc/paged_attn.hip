// Attention of new tokens over the quantized paged cache.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,   j <= kv_len - q_len + i
//
// for the q_len new tokens i of each sequence, whose keys and values are in
// the cache already; k_j = ks_j * (what the page holds), v_j alike.
//
// Numerics.  A page's INT8 or e4m3 values are exact in fp16, so both products
// run on the fp16 matrix instructions with exact cache operands and fp32 sums.
// q is scaled by a power of two for each row (its largest magnitude lands in
// [2^13, 2^14)), which bf16 and fp16 queries survive exactly down to 2^-27 of that (an
// element errs by 2^-25 at most); fp32 queries are split into two fp16 terms (22
// bits), as are their probabilities.  bf16 calls round the probabilities once to
// fp16's 11 bits, three more than their output keeps: against 64 bits their outputs
// are as near as those of fp32 sums (1.7e-3, the output's own rounding), and a second
// term would take 2% of a batch of single tokens, 27% of a prompt.  For fp16 that is as
// many as the output keeps: few rows, and rows of few keys, take the second term, the
// others not (a 4096-token prompt 2.4e-4 off, where one rounding leaves 2.0e-4).
// The key scales multiply the scores and the value scales the probabilities; the
// latter are held relative to a power of two `nu` near the largest value scale
// that the row sees in the tile (a later token's values, however large, take no
// bits from an earlier one's row), so that the fp16 range covers them whatever the
// values' size.  Running maxima and sums are fp32.
//
// Both kernels compute S^T = K Q^T and O^T = V^T P^T: a lane then holds one
// query row's scores, and the first product's result is the second one's
// operand as it stands, with the keys in the order that the result layout
// gives them; V's operand is read from LDS in that order, transposed by the
// LDS unit.
#include "mix_common.h"

#include <algorithm>
#include <type_traits>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

struct AttnArgs {
    const void* q;
    void* out;
    int64_t q_token, q_head, o_token, o_head;  // element strides
    const uint8_t* kp;
    const uint8_t* vp;
    const float* ks;
    const float* vs;
    const int32_t* table;
    const int32_t* kv_lens;
    const int32_t* cu;  // null: one token a sequence
    uint8_t* unpacked;  // [copies][H][tiles]: the copies that long chunks read
    int tiles;          // of 64 keys, in the whole table
    int by_seq;         // a copy for each sequence; else for those of kBigRows rows or more
    // Sums of rows whose keys are split, one set for each kind of kernel, where that kind
    // has more than one split: [nkeys][krows][D] and [nrows][T * Hq][D], with maximum and
    // sum of each.  A first sum below zero: the row is not this kind's.
    float* kpart;
    float* rpart;
    f2* kml;
    f2* rml;
    int64_t krows;
    int kper;           // attn_keys_kernel's rows are [B][H][kper] (0: [T][Hq])
    int64_t table_row;
    int T, B, Hq, H, G, P, pshift, table_w, nslots, dt;
    int ntile16;               // workgroups for a sequence's rows in attn_keys_kernel
    int few, big;              // attn_rows_kernel's sequences have more than `few` and fewer than `big` rows
    int nkeys, nrows;          // splits of the keys: of the two kinds of kernels
    float scale;  // softmax scale * log2(e)
};

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

struct Seq {
    int q0, n, kv;  // first token, new tokens, keys
};

__device__ inline Seq sequence(const AttnArgs& a, int b) {
    Seq s;
    int q0 = b, q1 = b + 1;
    if (a.cu) {
        q0 = min(max(a.cu[b], 0), a.T);
        q1 = min(max(a.cu[b + 1], q0), a.T);
    }
    s.q0 = q0;
    s.n = q1 - q0;
    s.kv = (int)min((int64_t)max(a.kv_lens[b], 0), (int64_t)a.table_w << a.pshift);
    return s;
}

// Cache row (in rows of D) of the 16 keys from `key` on for head h; -1 where
// the sequence or its table has none.  kv > 0.
__device__ inline int64_t group_row(const AttnArgs& a, const int32_t* table, int h, int key, int kv) {
    const int page = table[min(key, kv - 1) >> a.pshift];
    const bool is = key < kv && page >= 0 && page < a.P;
    const int64_t row = (((int64_t)page * a.H + h) << a.pshift) + (key & ((1 << a.pshift) - 1));
    return is ? row : -1;
}

constexpr f2 kNotMine = {0.0f, -1.0f};  // no sum of exponentials is below zero

// attn_keys_kernel's row among its sums: token `tok`, query head `head`, which is row
// `row` of sequence b and key head h.
__device__ inline int64_t keys_row_of(const AttnArgs& a, int b, int h, int row, int tok, int head) {
    return a.kper ? ((int64_t)b * a.H + h) * a.kper + row : (int64_t)tok * a.Hq + head;
}

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

// ------------------------------------------------------------------ few rows: the keys shared out
//
// One workgroup for 16 of a sequence's up to few_rows() rows (new tokens times the
// query heads of one key-value head), one key-value head and one split of the
// keys; its four waves take tiles of 32 keys in turn.  Bound by HBM: the next tile's
// keys and values are on their way while this one is computed, 16 KB a wave
// (D = 256), and no wave waits for another before the end.  64 single tokens
// over 100 to 16000 keys of 8 heads of 128 (537 MB): 125 us, 4.3 TB/s, and the
// join 5.6; over 4 heads of 256 141 (bf16) and 163 (fp32), and 5.8.  One token over
// 4101 keys of 4 heads of 256, 129 tiles: of 64 splits 43 have three tiles each
// and the others none, 10.6 us and the join 7.2; of 32 26 have five, 13.2 and 5.2.
// Latency, of the table, the keys and one tile's chain of products.

// LDS row of a key's values: the transposed reads' four rows fall on unlike banks.
constexpr int keys_row(int D) { return D + 16; }
constexpr int keys_lds(int D) { return std::max(4 * 32 * keys_row(D) * 2, 4 * 16 * (D + 4) * 4); }

// lds: keys_lds(D) bytes; sql: the queries' second terms, the same for all waves.
template <int D, int KIND, int DT>
__device__ __forceinline__ void attend_keys(const AttnArgs& a, int block, uint8_t* lds, float (*sm)[16], float (*sl)[16],
                                            float (*snu)[16], h8* sql) {
    constexpr bool SPLIT = DT == kF32;    // two terms of the queries
    constexpr bool PSPLIT = DT != kBF16;  // and of the probabilities: the matrix rate is not what binds here
    constexpr int KC = D / 64;        // 16-byte chunks of a key a lane takes (a quarter of each 64 values)
    constexpr int VC = D / 32;        // 16-byte chunks of a tile's values a lane takes
    constexpr int VS = keys_row(D), OS = D + 4;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = block % a.H, tile16 = block / a.H % a.ntile16, bs = block / a.H / a.ntile16;
    const int split = bs % a.nkeys, b = bs / a.nkeys;
    const Seq sq = sequence(a, b);
    if ((int64_t)sq.n * a.G > a.few) return;
    const int row0 = 16 * tile16, rows = min(sq.n * a.G - row0, 16);  // this workgroup's
    if (rows <= 0) return;
    const int r16 = lane & 15, c = lane >> 4;
    const int32_t* table = a.table + b * a.table_row;

    // The query operand: row r16, values 64 i + 16 c + 8 half + 0..7 for slab 2 i + half.
    const bool has_row = r16 < rows;
    const int row = row0 + (has_row ? r16 : 0), tok = sq.q0 + row / a.G, head = h * a.G + row % a.G;
    const int last = has_row ? sq.kv - sq.n + row / a.G : -1;  // the last key that the row sees
    const int ntile = (sq.kv + 31) >> 5, per = (ntile + a.nkeys - 1) / a.nkeys;
    const int t1 = min((split + 1) * per, ntile);
    int t = split * per + wave;

    f4 o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = (f4){0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f, nu = kLeastNu, peak = 0.0f;

    u4 kraw[2][KC], vraw[VC];
    f4 ksc[2], vsc[2];
    _Float16* vt = reinterpret_cast<_Float16*>(lds) + wave * (32 * VS);

    int64_t at2[2];
    const auto rows_of = [&](int tile, int64_t* r) {
#pragma unroll
        for (int u = 0; u < 2; ++u) r[u] = group_row(a, table, h, 32 * tile + 16 * u, sq.kv);
    };
    const auto load = [&](const int64_t* r) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t at = r[u] < 0 ? 0 : r[u];  // a masked group reads the cache's first rows
            const uint8_t* kp = a.kp + (at + r16) * D + 16 * c;
#pragma unroll
            for (int i = 0; i < KC; ++i) kraw[u][i] = *reinterpret_cast<const u4*>(kp + 64 * i);
            ksc[u] = *reinterpret_cast<const f4*>(a.ks + at + 4 * c);
            vsc[u] = *reinterpret_cast<const f4*>(a.vs + at + 4 * c);
        }
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            constexpr int per_row = D / 16;
            const int chunk = lane + 64 * i, kr = chunk / per_row;  // kr / 16 does not depend on the lane
            const int64_t at = r[(64 * i / per_row) >> 4] < 0 ? 0 : r[(64 * i / per_row) >> 4];
            vraw[i] = *reinterpret_cast<const u4*>(a.vp + (at + (kr & 15)) * D + 16 * (chunk % per_row));
        }
    };
    int64_t next[2] = {-1, -1};
    if (t < t1) {
        rows_of(t, at2);
        load(at2);
        rows_of(t + 4, next);
    }
    h8 qh[D / 32];
    float rowf;
    {
        float x[D / 4];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                f4 v = {0, 0, 0, 0};
                if (has_row) v = load4(a.q, DT, tok * a.q_token + head * a.q_head + 64 * i + 16 * c + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[16 * i + j + e] = v[e];
                    top = max(top, f_bits(v[e]) & 0x7FFFFFFFu);
                }
            }
        top = lane_max_u32(lane_max_u32(top, 16), 32);
        const float up = row_scale(top);
        rowf = score_worth(a.scale, up);
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = x[8 * s + j] * up;
            if constexpr (SPLIT) {
                h8 lo;
                split8(w, qh[s], lo);
                if (wave == 0) sql[64 * s + lane] = lo;
            } else {
                qh[s] = round8(w);
            }
        }
    }

    if constexpr (SPLIT) __syncthreads();

    for (; t < t1; t += 4) {
        const int key0 = 32 * t;
        const bool tail = key0 + 32 > sq.kv || at2[0] < 0 || at2[1] < 0;
        // Values to LDS, [key][d] in fp16.
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            constexpr int per_row = D / 16;
            const int chunk = lane + 64 * i, kr = chunk / per_row;
            u4 w = vraw[i];
            if (KIND == kFp8 && tail && (key0 + kr >= sq.kv || at2[kr >> 4] < 0)) w = (u4){0, 0, 0, 0};
            h8* dst = reinterpret_cast<h8*>(vt + kr * VS + 16 * (chunk % per_row));
            dst[0] = unpack8<KIND>(w.x, w.y);
            dst[1] = unpack8<KIND>(w.z, w.w);
        }
        f4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f4 s1 = {0, 0, 0, 0};  // a chain of its own: one tile is all that a wave may have
            s[u] = s1;
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                const h8 k0 = unpack8<KIND>(kraw[u][i].x, kraw[u][i].y), k1 = unpack8<KIND>(kraw[u][i].z, kraw[u][i].w);
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[2 * i], s[u], 0, 0, 0);
                s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[2 * i + 1], s1, 0, 0, 0);
                if constexpr (SPLIT) {
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, sql[64 * (2 * i) + lane], s[u], 0, 0, 0);
                    s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, sql[64 * (2 * i + 1) + lane], s1, 0, 0, 0);
                }
            }
            s[u] += s1;
        }
        float x[8], vw[8];
        bool see[8];
        float top = -INFINITY, vmax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int u = j >> 2, key = key0 + 16 * u + 4 * c + (j & 3);
            see[j] = key <= last && at2[u] >= 0;
            x[j] = see[j] ? s[u][j & 3] * ksc[u][j & 3] : -INFINITY;
            vw[j] = see[j] ? vsc[u][j & 3] : 0.0f;
            top = fmaxf(top, x[j]);
            vmax = fmaxf(vmax, vw[j]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) at2[u] = next[u];
        if (t + 4 < t1) load(at2);
        rows_of(t + 8, next);

        top = max_halves(max_rows16(top));
        vmax = max_halves(max_rows16(vmax));  // of the keys that the row sees: what others hold is not its concern
        const float mn = fmaxf(m, top), safe = mn == -INFINITY ? 0.0f : mn;
        const float lalpha = fast_exp2((m - safe) * rowf);
        m = mn;
        peak *= lalpha;
        const float now = next_nu(nu, vmax, peak, kLeastNu), alpha = lalpha * (nu / now);
        nu = now;
        peak = fmaxf(peak, now);
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] *= alpha;
        }
        l *= lalpha;
        const float up = kPScale / nu;
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float p = fast_exp2((x[j] - safe) * rowf);
            l += p;
            w[j] = vw[j] == 0.0f ? 0.0f : p * (vw[j] * up);
        }
        h8 ph, pl;
        if constexpr (PSPLIT) split8(w, ph, pl);
        else ph = round8(w);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const _Float16* p = vt + (4 * c + (r16 >> 2)) * VS + 16 * i + 4 * (r16 & 3);
            const h8 v = join(read_tr(p), read_tr(p + 16 * VS));
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[i], 0, 0, 0);
            if constexpr (PSPLIT) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[i], 0, 0, 0);
        }
    }

    // The four waves' sums, joined in wave order.
    l = sum_halves(sum_rows16(l));
    __syncthreads();
    float* so = reinterpret_cast<float*>(lds);
    if (c == 0) {
        sm[wave][r16] = m * rowf;  // in units of log2
        sl[wave][r16] = l;
        snu[wave][r16] = nu * (1.0f / kPScale);
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<f4*>(so + (wave * 16 + r16) * OS + 16 * i + 4 * c) = o[i];
    __syncthreads();
    const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
    if (r >= rows) return;
    float top = -INFINITY, sum = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, sm[w][r]);
    const float safe = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = fast_exp2(sm[w][r] - safe);
        sum += f[w] * sl[w][r];
        f[w] *= snu[w][r];
    }
    const int ot = sq.q0 + (row0 + r) / a.G, oh = h * a.G + (row0 + r) % a.G;
    const int64_t prow = split * a.krows + keys_row_of(a, b, h, row0 + r, ot, oh);
    const float inv = a.nkeys > 1 ? 1.0f : sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    if (part == 0) {
        if (a.nkeys > 1) a.kml[prow] = (f2){top, sum};
        if (a.nrows > 1 && split == 0) a.rml[(int64_t)ot * a.Hq + oh] = kNotMine;
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const int d = 64 * i + 4 * part;
        f4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f4*>(so + (w * 16 + r) * OS + d) * f[w];
        v *= inv;
        if (a.nkeys > 1) *reinterpret_cast<f4*>(a.kpart + prow * D + d) = v;
        else store4(a.out, DT, ot * a.o_token + oh * a.o_head + d, v);
    }
}

// Workgroups a compute unit.  fp32 with heads of 256 spills 49 to 57 registers a lane at
// two, whose traffic weighs where a workgroup has few rows and waits for HBM: 32
// single tokens over up to 8000 keys of 4 heads 91 us at two, 51 at one, 64 over 100 to
// 16000 keys 224 and 162; 12 tokens over 6000 keys, 72 rows, 48 and 56.  Half types
// with heads of 128 spill nothing at three (INT8: 64 tokens over 100 to 16000 keys 130
// us, at two 133).
constexpr int keys_per_unit(int D, int DT, bool lone) {
    if (D == 256 && DT == kF32) return lone ? 1 : 2;
    return D == 256 || DT == kF32 ? 2 : 3;
}

template <int D, int KIND, int DT, bool LONE>
__global__ __launch_bounds__(256, keys_per_unit(D, DT, LONE)) void attn_keys_kernel(AttnArgs a) {
    __shared__ __align__(16) uint8_t lds[keys_lds(D)];
    __shared__ float sm[4][16], sl[4][16], snu[4][16];
    __shared__ __align__(16) h8 sql[DT == kF32 ? D / 32 * 64 : 1];
    attend_keys<D, KIND, DT>(a, blockIdx.x, lds, sm, sl, snu, sql);
}

// ------------------------------------------------------------------ many rows: the rows shared out
//
// One workgroup for 128 rows of a sequence, one key-value head and one split
// of the keys; each of its four waves holds 32 rows' queries and sums, and
// tiles of 64 keys pass through LDS, unpacked to fp16 on the way in.  The next
// tile's bytes are loaded while this one is computed.  Sequences of few rows
// are attn_keys_kernel's.

constexpr int kRowTile = 128, kKeyTile = 64;

// The 128 rows of a slot: their sequence (-1: none) and the first of them.  Sequence b's tiles take the slots from
// cu[b] * G / 128 + b on, which leaves room for all without a pass over the lengths.
__device__ inline int rows_of_slot(const AttnArgs& a, int slot, Seq& sq, int64_t& first) {
    const int per = (a.G + kRowTile - 1) / kRowTile;
    int b = 0;
    if (a.cu) {
        int hi = a.B;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            const int64_t start = (int64_t)min(max(a.cu[mid], 0), a.T) * a.G / kRowTile + mid;
            if (start <= slot) b = mid;
            else hi = mid;
        }
    } else {
        b = slot / per;
    }
    sq = sequence(a, b);
    const int64_t rows = (int64_t)sq.n * a.G;
    first = (slot - (a.cu ? (int64_t)sq.q0 * a.G / kRowTile + b : (int64_t)b * per)) * kRowTile;
    return first < 0 || first >= rows ? -1 : b;
}

// A row's maximum and sum, and where attn_keys_kernel's sums are by tokens too, that it is not among them.
__device__ inline void mark_row(const AttnArgs& a, int split, int64_t row, float top, float sum) {
    if (a.nrows > 1) a.rml[(int64_t)split * a.T * a.Hq + row] = (f2){top, sum};
    if (a.nkeys > 1 && !a.kper && split == 0) a.kml[row] = kNotMine;
}

// A row's queries as operands (values 16 s + 8 (lane / 32) + 0..7 for slab s,
// from element `at` on), scaled; returns what a score is worth in log2.
template <int D, int DT>
__device__ inline float load_queries(const AttnArgs& a, int64_t at, h8* hi, h8* lo) {
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const f4 v = load4(a.q, DT, at + 16 * s + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, f_bits(v[e]) & 0x7FFFFFFFu);
        }
    top = lane_max_u32(top, 32);
    const float up = row_scale(top);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const f4 v = load4(a.q, DT, at + 16 * s + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[j + e] = v[e] * up;
        }
        if constexpr (DT == kF32) split8(w, hi[s], lo[s]);
        else hi[s] = round8(w);
    }
    return score_worth(a.scale, up);
}

template <int D, int KIND, int DT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_rows_kernel(AttnArgs a) {
    constexpr bool SPLIT = DT == kF32, PSPLIT = DT != kBF16;  // two terms of the queries, and of the probabilities
    constexpr int KS = D + 8, VS = D + 16;  // LDS rows of a key: reads of one instruction fall on unlike banks
    constexpr int NC = D / 64;              // 16-byte chunks a thread loads of a tile's keys (and of its values)
    constexpr int per_row = D / 16;
    __shared__ __align__(16) _Float16 sk[kKeyTile * KS], sv[kKeyTile * VS];
    __shared__ __align__(16) float sks[kKeyTile], svs[kKeyTile];
    __shared__ float sbad[kKeyTile], smax;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, hf = lane >> 5;
    const int h = blockIdx.x % a.H, ss = blockIdx.x / a.H, split = ss % a.nrows;
    const int slot = a.nslots - 1 - ss / a.nrows;  // a prompt's last rows see the most keys: first
    Seq sq;
    int64_t first;
    const int b = rows_of_slot(a, slot, sq, first);
    const int64_t rows = (int64_t)sq.n * a.G;
    if (b < 0 || rows <= a.few || rows >= a.big) return;
    const int64_t row = first + 32 * wave + r32;
    const bool has_row = row < rows;
    const int tok_in = has_row ? (int)(row / a.G) : 0;
    const int tok = sq.q0 + tok_in, head = h * a.G + (has_row ? (int)(row % a.G) : 0);
    const int last = has_row ? sq.kv - sq.n + tok_in : -1;
    // Keys that the workgroup's, and this wave's, last row sees; keys that all of the wave's rows see.
    const auto seen_by = [&](int64_t r) { return max(sq.kv - sq.n + (int)(min(r, rows - 1) / a.G) + 1, 0); };
    const int wg_end = seen_by(first + kRowTile - 1);
    const bool wave_rows = first + 32 * wave < rows;
    const int wave_end = wave_rows ? seen_by(first + 32 * wave + 31) : 0;
    const int wave_all = seen_by(first + 32 * wave);

    h8 qh[D / 16], ql[SPLIT ? D / 16 : 1];
    const float rowf = load_queries<D, DT>(a, tok * a.q_token + head * a.q_head + 8 * hf, qh, ql);

    const int ntile = (min(wg_end, sq.kv) + kKeyTile - 1) / kKeyTile, per = (ntile + a.nrows - 1) / a.nrows;
    const int t1 = min((split + 1) * per, ntile);
    int t = split * per;
    const int32_t* table = a.table + b * a.table_row;

    f16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f, nu = kLeastNu, peak = 0.0f;

    u4 kraw[NC], vraw[NC];
    int64_t grow[NC];    // cache rows of the groups of 16 keys that this wave's chunks belong to
    float ksc = 0.0f, vsc = 0.0f;  // wave 0: a key's two scales
    bool sc_bad = true;
    const auto load = [&](int tile) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int kr = (wave * 64 + 256 * i) / per_row;  // the wave's first row of this pass
            grow[i] = group_row(a, table, h, kKeyTile * tile + (kr & ~15), sq.kv);
            const int64_t at = (grow[i] < 0 ? 0 : grow[i]) + ((tid + 256 * i) / per_row & 15);
            kraw[i] = *reinterpret_cast<const u4*>(a.kp + at * D + 16 * (tid % per_row));
            vraw[i] = *reinterpret_cast<const u4*>(a.vp + at * D + 16 * (tid % per_row));
        }
        if (wave == 0) {
            const int64_t at = group_row(a, table, h, kKeyTile * tile + (lane & ~15), sq.kv);
            sc_bad = at < 0 || kKeyTile * tile + lane >= sq.kv;
            ksc = sc_bad ? 0.0f : a.ks[at + (lane & 15)];
            vsc = sc_bad ? 0.0f : a.vs[at + (lane & 15)];
        }
    };
    if (t < t1) load(t);

    for (; t < t1; ++t) {
        const int key0 = kKeyTile * t;
        __syncthreads();  // the last tile's reads are over
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int kr = (tid + 256 * i) / per_row, col = 16 * (tid % per_row);
            u4 kw = kraw[i], vw = vraw[i];
            if (KIND == kFp8 && (grow[i] < 0 || key0 + kr >= sq.kv)) kw = vw = (u4){0, 0, 0, 0};
            h8* kd = reinterpret_cast<h8*>(sk + kr * KS + col);
            h8* vd = reinterpret_cast<h8*>(sv + kr * VS + col);
            kd[0] = unpack8<KIND>(kw.x, kw.y);
            kd[1] = unpack8<KIND>(kw.z, kw.w);
            vd[0] = unpack8<KIND>(vw.x, vw.y);
            vd[1] = unpack8<KIND>(vw.z, vw.w);
        }
        if (wave == 0) {
            // A value scale of NaN goes with the key's, whose score a row that does
            // not see the key leaves out; times a probability of zero it would not.
            const bool nan = vsc != vsc;
            sks[lane] = nan ? vsc : ksc;
            sbad[lane] = sc_bad ? 1.0f : 0.0f;
            float vmax = nan ? 0.0f : vsc;
#pragma unroll
            for (int st = 1; st < 64; st *= 2) vmax = fmaxf(vmax, __shfl_xor(vmax, st));
            svs[lane] = nan ? 0.0f : vsc;
            if (lane == 0) smax = vmax;
        }
        __syncthreads();
        if (t + 1 < t1) load(t + 1);
        if (key0 >= wave_end) continue;

        f16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int j = 0; j < 16; ++j) s[u][j] = 0.0f;
            const _Float16* p = sk + (32 * u + r32) * KS + 8 * hf;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const h8 k = *reinterpret_cast<const h8*>(p + 16 * i);
                s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[i], s[u], 0, 0, 0);
                if constexpr (SPLIT) s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[i], s[u], 0, 0, 0);
            }
        }
        // Scores times the key scales; result register j holds key 8 (j / 4) + 4 hf + j % 4.
        float top = -INFINITY, vmax = smax;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const f4 sc = *reinterpret_cast<const f4*>(sks + 32 * u + 2 * j + 4 * hf);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[u][j + e] *= sc[e];
            }
        // Past the wave's first row, past the sequence's end or in a page that is not
        // there: neither a score, nor among the values that set the row's units.
        if (key0 + kKeyTile > wave_all || key0 + kKeyTile > sq.kv || __any(sbad[lane] != 0.0f)) {
            vmax = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int k = 32 * u + 8 * (j / 4) + 4 * hf + j % 4;
                    const bool out = key0 + k > last || sbad[k] != 0.0f;
                    s[u][j] = out ? -INFINITY : s[u][j];
                    vmax = fmaxf(vmax, out ? 0.0f : svs[k]);
                }
            vmax = max_halves(vmax);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, s[u][j]);
        top = max_halves(top);
        const float mn = fmaxf(m, top), safe = mn == -INFINITY ? 0.0f : mn;
        const float lalpha = fast_exp2((m - safe) * rowf);
        m = mn;
        peak *= lalpha;
        const float now = next_nu(nu, vmax, peak, kLeastNu), alpha = lalpha * (nu / now), up = kPScale / now;
        nu = now;
        peak = fmaxf(peak, now);
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
        }
        l *= lalpha;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int g = 0; g < 2; ++g) {  // 16 keys
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = fast_exp2((s[u][8 * g + j] - safe) * rowf);
                    l += w[j];
                }
                const f4 s0 = *reinterpret_cast<const f4*>(svs + 32 * u + 16 * g + 4 * hf);
                const f4 s1 = *reinterpret_cast<const f4*>(svs + 32 * u + 16 * g + 8 + 4 * hf);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] *= s0[j] * up;
                    w[4 + j] *= s1[j] * up;
                }
                h8 ph, pl;
                if constexpr (PSPLIT) split8(w, ph, pl);
                else ph = round8(w);
                const int i16 = lane & 15;
                const _Float16* p = sv + (32 * u + 16 * g + 4 * hf + (i16 >> 2)) * VS + 16 * (r32 >> 4) + 4 * (i16 & 3);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const h8 v = join(read_tr(p + 32 * i), read_tr(p + 32 * i + 8 * VS));
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, o[i], 0, 0, 0);
                    if constexpr (PSPLIT) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[i], 0, 0, 0);
                }
            }
    }

    if (!has_row) return;
    l = sum_halves(l);
    const int64_t orow = (int64_t)tok * a.Hq + head, prow = (int64_t)split * a.T * a.Hq + orow;
    float f = nu * (1.0f / kPScale);
    if (hf == 0) mark_row(a, split, orow, m * rowf, l);
    if (a.nrows == 1) f *= l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const int d = 32 * i + 2 * j + 4 * hf;
            const f4 v = {o[i][j] * f, o[i][j + 1] * f, o[i][j + 2] * f, o[i][j + 3] * f};
            if (a.nrows > 1) *reinterpret_cast<f4*>(a.rpart + prow * D + d) = v;
            else store4(a.out, DT, tok * a.o_token + head * a.o_head + d, v);
        }
}

// ------------------------------------------------------------------ many rows over one unpacked copy
//
// A long chunk reads every key once for each 128 of its rows, and unpacking a
// tile costs the kernel above about half as much vector work as its softmax.
// So keys and values of long chunks are first unpacked once, to fp16 (exactly),
// in the order of the matrix instructions' operands (1 KB each, 16 bytes a
// lane), V transposed, with the scales beside them.  Tiles then come straight
// to LDS.  32768 keys of 4 heads of 256: 42 us for the copy, beside 1.6 ms.

// Rows from which on a sequence has a copy where not all have one.  Two such
// sequences' first rows are that far apart, so first row / kBigRows tells them apart.
constexpr int kBigRows = 256;
// fp16 rows of fewer keys than this take two terms of the probabilities: one term's rounding is as large as
// the output's own, and where a few keys hold most of a row it does not average out
// (a 4096-token prompt of 32/8 heads of 128: 188.2 us with one term throughout, 189.2 so).
constexpr int kTwoTerms = 512;
__device__ inline int copy_of(const AttnArgs& a, const Seq& sq, int b) {
    return a.by_seq ? b : (int)((int64_t)sq.q0 * a.G / kBigRows);
}

constexpr int kHead = 1024;  // a tile's scales: ks[64], vs[64], 1 where a key is not there [64], largest vs, any not there
template <int D>
constexpr int tile_bytes() { return kKeyTile * D * 4 + kHead; }

constexpr int unpack_lds(int D) { return 2 * kKeyTile * (D + 16) * 2; }

// lds: unpack_lds(D) bytes.
template <int D, int KIND>
__device__ __forceinline__ void unpack_tiles(const AttnArgs& a, unsigned block, unsigned blocks, uint8_t* lds) {
    constexpr int VS = D + 16, NC = D / 64, per_row = D / 16, KF = D / 8;  // KF operands of K, as many of V
    _Float16 *const sv = reinterpret_cast<_Float16*>(lds), *const sk = sv + kKeyTile * VS;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t items = (int64_t)a.B * a.H * a.tiles;
    for (int64_t it = block; it < items; it += blocks) {
        const int tile = (int)(it % a.tiles), h = (int)(it / a.tiles % a.H), b = (int)(it / a.tiles / a.H);
        const Seq sq = sequence(a, b);
        if ((int64_t)sq.n * a.G < a.big) {
            // None of this sequence's: on to the next one's first.
            const int64_t next = (int64_t)(b + 1) * a.H * a.tiles;
            it += (next - 1 - it) / blocks * blocks;
            continue;
        }
        if (tile * kKeyTile >= sq.kv) continue;
        const int32_t* table = a.table + b * a.table_row;
        uint8_t* out = a.unpacked + (((int64_t)copy_of(a, sq, b) * a.H + h) * a.tiles + tile) * tile_bytes<D>();
        if (wave == 0) {
            const int64_t at = group_row(a, table, h, kKeyTile * tile + (lane & ~15), sq.kv);
            const bool bad = at < 0 || kKeyTile * tile + lane >= sq.kv;
            const int64_t from = (at < 0 ? 0 : at) + (lane & 15);
            const float ks = a.ks[from], vs = a.vs[from];
            // A value scale of NaN goes with the key's, whose score a row that does
            // not see the key leaves out; times a probability of zero it would not.
            const bool nan = vs != vs;
            const float vv = bad || nan ? 0.0f : vs, vmax = max_wave(vv);
            float* head = reinterpret_cast<float*>(out + kKeyTile * D * 4);
            head[lane] = bad ? 0.0f : nan ? vs : ks;
            head[64 + lane] = vv;
            head[128 + lane] = bad ? 1.0f : 0.0f;
            head[192 + lane] = lane == 0 ? vmax : __any(bad) ? 1.0f : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int kr = (tid + 256 * i) / per_row, col = 16 * (tid % per_row);
            const int64_t row = group_row(a, table, h, kKeyTile * tile + (kr & ~15), sq.kv);
            const bool is = row >= 0 && kKeyTile * tile + kr < sq.kv;
            const int64_t at = ((row < 0 ? 0 : row) + (kr & 15)) * D + col;
            u4 kw = *reinterpret_cast<const u4*>(a.kp + at), vw = *reinterpret_cast<const u4*>(a.vp + at);
            if (!is) kw = vw = (u4){0, 0, 0, 0};
            h8* kd = reinterpret_cast<h8*>(sk + kr * VS + col);
            h8* vd = reinterpret_cast<h8*>(sv + kr * VS + col);
            kd[0] = unpack8<KIND>(kw.x, kw.y);
            kd[1] = unpack8<KIND>(kw.z, kw.w);
            vd[0] = unpack8<KIND>(vw.x, vw.y);
            vd[1] = unpack8<KIND>(vw.z, vw.w);
        }
        __syncthreads();
        h8* ko = reinterpret_cast<h8*>(out);
#pragma unroll
        for (int i = 0; i < KF / 4; ++i) {
            const int f = 4 * i + wave;
            // K: keys 32 u + lane % 32, values 16 s + 8 (lane / 32) + 0..7.
            const int u = f / (D / 16), sl = f % (D / 16), r32 = lane & 31, hf = lane >> 5, i16 = lane & 15;
            ko[64 * f + lane] = *reinterpret_cast<const h8*>(sk + (32 * u + r32) * VS + 16 * sl + 8 * hf);
            // V: value 32 t + lane % 32, keys 16 g + 4 (lane / 32) + 0..3 and 8 more.
            const int g = f / (D / 32), t = f % (D / 32);
            const _Float16* p = sv + (16 * g + 4 * hf + (i16 >> 2)) * VS + 32 * t + 16 * (r32 >> 4) + 4 * (i16 & 3);
            ko[64 * (KF + f) + lane] = join(read_tr(p), read_tr(p + 8 * VS));
        }
        __syncthreads();
    }
}

template <int D, int KIND>
__global__ __launch_bounds__(256) void attn_unpack_kernel(AttnArgs a) {
    __shared__ __align__(16) uint8_t lds[unpack_lds(D)];
    unpack_tiles<D, KIND>(a, blockIdx.x, gridDim.x, lds);
}

// Both, where a call has few rows of some sequences and many of others: the first
// `keys` workgroups are attn_keys_kernel's.  Each waits on memory most of its time:
// 27 us together, 20 and 13 one after the other (8 sequences of 1 to 700 tokens behind
// up to 5000, 32/8 heads of 128, bf16, INT8).
template <int D, int KIND, int DT>
__global__ __launch_bounds__(256, keys_per_unit(D, DT, false)) void attn_keys_unpack_kernel(AttnArgs a, unsigned keys) {
    __shared__ __align__(16) uint8_t lds[std::max(keys_lds(D), unpack_lds(D))];
    __shared__ float sm[4][16], sl[4][16], snu[4][16];
    __shared__ __align__(16) h8 sql[DT == kF32 ? D / 32 * 64 : 1];
    if (blockIdx.x < keys) attend_keys<D, KIND, DT>(a, blockIdx.x, lds, sm, sl, snu, sql);
    else unpack_tiles<D, KIND>(a, blockIdx.x - keys, gridDim.x - keys, lds);
}

// As attn_rows_kernel, over the copy.  The scores of tile t + 1 are computed
// beside the softmax of tile t, which they do not wait for, then the weighted
// values of tile t; K of tile t + 2 and V of tile t + 1 are on their way.
//
// Bound by the issue of matrix and vector instructions together: on a 4096-token
// prompt of 32/8 heads of 128 (fp16, 137 GFLOP, 175 to 220 us) they were busy 41%
// and 54% of the cycles, one beside the other hardly ever, whatever the waves'
// priorities and the order of the code.  1024 tokens behind 31744, 24/4 heads
// of 256, fp32 (812 GFLOP, twice that in two-term products): 1.66 ms, 980
// TFLOP/s of matrix instructions against 1160 of a large library product.
template <int D, int DT>
__global__ __launch_bounds__(256, D == 256 || (D == 128 && DT == kF32) ? 1 : 2) void attn_tiles_kernel(AttnArgs a) {
    constexpr bool SPLIT = DT == kF32;
    constexpr int KB = kKeyTile * D * 2;
    __shared__ __align__(1024) uint8_t sk[2][KB], sv[2][KB];
    __shared__ __align__(1024) float sh[2][kHead / 4];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, hf = lane >> 5;
    const int h = blockIdx.x % a.H, ss = blockIdx.x / a.H, split = ss % a.nrows;
    const int slot = a.nslots - 1 - ss / a.nrows;  // a prompt's last rows see the most keys: first
    Seq sq;
    int64_t first;
    const int b = rows_of_slot(a, slot, sq, first);
    const int64_t rows = (int64_t)sq.n * a.G, row = first + 32 * wave + r32;
    if (b < 0 || rows < a.big) return;
    const bool has_row = row < rows;
    const int tok_in = has_row ? (int)(row / a.G) : 0;
    const int tok = sq.q0 + tok_in, head = h * a.G + (has_row ? (int)(row % a.G) : 0);
    const int last = has_row ? sq.kv - sq.n + tok_in : -1;
    // Keys that the workgroup's last row sees, and keys that all of the wave's rows see.
    const auto seen_by = [&](int64_t r) { return max(sq.kv - sq.n + (int)(min(r, rows - 1) / a.G) + 1, 0); };
    const int wg_end = min(seen_by(first + kRowTile - 1), sq.kv);
    const int wave_all = first + 32 * wave + 31 < rows ? min(seen_by(first + 32 * wave), sq.kv) : 0;

    h8 qh[D / 16], ql[SPLIT ? D / 16 : 1];
    const float rowf = load_queries<D, DT>(a, tok * a.q_token + head * a.q_head + 8 * hf, qh, ql);

    const int ntile = (wg_end + kKeyTile - 1) / kKeyTile, per = (ntile + a.nrows - 1) / a.nrows;
    const int t0 = split * per, t1 = min(t0 + per, ntile);
    const uint8_t* const tiles = a.unpacked + ((int64_t)copy_of(a, sq, b) * a.H + h) * a.tiles * tile_bytes<D>();

    f16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    // A tile's weights are computed in units in which a probability of 1 is 2^9 / nu, at
    // most 2^119 of those eight, so that a lane's 32 add up to less than fp32 holds.
    // Past nu = 2^96 (values of 1e31) the smallest of them fall out of its range.
    constexpr float least = 0x1p-110f;
    float m = -INFINITY, l = 0.0f, nu = least, peak = 0.0f, unit = __builtin_log2f(kPScale / least);

    // Past the last tile the loads repeat it.
    const auto fetch = [&](int t, int from, uint8_t* to) {
        const uint8_t* src = tiles + (int64_t)min(t, t1 - 1) * tile_bytes<D>() + from + 1024 * wave + 16 * lane;
#pragma unroll
        for (int i = 0; i < KB / 4096; ++i) load_lds(src + 4096 * i, lds_address(to) + 1024 * wave + 4096 * i);
    };
    const auto fetch_head = [&](int t) {
        if (wave == 0)
            load_lds(tiles + (int64_t)min(t, t1 - 1) * tile_bytes<D>() + 2 * KB + 16 * lane, lds_address(sh[t & 1]));
    };
    f16 s[2];
    const auto scores = [&](const uint8_t* kb) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[u][j] = 0.0f;
        const h8* p = reinterpret_cast<const h8*>(kb) + lane;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const h8 k0 = p[64 * i], k1 = p[64 * (D / 16 + i)];
            s[0] = mfma32(k0, qh[i], s[0]);
            s[1] = mfma32(k1, qh[i], s[1]);
            if constexpr (SPLIT) {
                s[0] = mfma32(k0, ql[i], s[0]);
                s[1] = mfma32(k1, ql[i], s[1]);
            }
        }
    };
    if (t0 < t1) {
        fetch(t0, 0, sk[t0 & 1]);
        fetch_head(t0);
        fetch(t0 + 1, 0, sk[(t0 + 1) & 1]);
        fetch(t0, KB, sv[t0 & 1]);
        wait_loads<0>();
        __syncthreads();
        scores(sk[t0 & 1]);
    }
    const auto run = [&](auto terms) {
        constexpr bool two = decltype(terms)::value;
        for (int t = t0; t < t1; ++t) {
            const int key0 = kKeyTile * t, par = t & 1;
            wait_loads<0>();
            __syncthreads();  // K of t + 1 and V of t are there; K of t and V of t - 1 are read
            fetch(t + 2, 0, sk[par]);
            fetch(t + 1, KB, sv[par ^ 1]);
            fetch_head(t + 1);
            const float* const hd = sh[par];
            float vmax = hd[192];
            f16 x[2];
            // Scores times the key scales; result register j holds key 8 (j / 4) + 4 hf + j % 4.
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const f4 sc = *reinterpret_cast<const f4*>(hd + 32 * u + 2 * j + 4 * hf);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[u][j + e] = s[u][j + e] * sc[e];
                }
            // Past the wave's first row, past the sequence's end or in a page that is not
            // there: neither a score, nor among the values that set the row's units.
            if (key0 + kKeyTile > wave_all || hd[193] != 0.0f) {
                vmax = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const f4 bad = *reinterpret_cast<const f4*>(hd + 128 + 32 * u + 2 * j + 4 * hf);
                        const f4 vs = *reinterpret_cast<const f4*>(hd + 64 + 32 * u + 2 * j + 4 * hf);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int k = key0 + 32 * u + 2 * j + 4 * hf + e;
                            const bool out = k > last || bad[e] != 0.0f;
                            x[u][j + e] = out ? -INFINITY : x[u][j + e];
                            vmax = fmaxf(vmax, out ? 0.0f : vs[e]);
                        }
                    }
                vmax = max_halves(vmax);
            }
            const auto largest = [&] {
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 16; j += 2) top = fmaxf(fmaxf(top, x[u][j]), x[u][j + 1]);
                return max_halves(top);
            };
            // The reference moves only once a row's scores pass it by kSlack.
            const auto move = [&] {
                const float top = largest();
                const bool moves = (top - m) * rowf > kSlack;
                const float f = moves ? fast_exp2((m - top) * rowf) : 1.0f;
                m = moves ? top : m;
                return f;
            };
            // Rarely a row's units change, its reference with them; here, since a branch behind
            // the next scores' matrix instructions would keep the softmax from running beside them.
            if (__any(vmax > nu * 8.0f || (vmax > 0.0f && vmax <= nu * 0x1p-4f))) {
                const float f = move();
                l *= f;
                peak *= f;
                const float now = next_nu(nu, vmax, peak, least), alpha = f * (nu / now);
                unit = __builtin_log2f(kPScale / now);
                nu = now;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
            }
            scores(sk[par ^ 1]);
            const float f = move();
            peak = fmaxf(peak * f, nu);
            const float ref = m == -INFINITY ? 0.0f : m;
            float base = __builtin_fmaf(-ref, rowf, unit);
            // m rowf is rounded once here, by less than half while it is below 2^22; past that
            // the difference is taken first, else the largest weight would be 2 to that error.
            if (__any(__builtin_fabsf(ref) * rowf > 0x1p22f)) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[u][j] -= ref;
                base = unit;
            }
            float sum = 0.0f;
            h8 ph[4], pl[two ? 4 : 1];
#pragma unroll
            for (int g = 0; g < 4; ++g) {  // 16 keys
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = fast_exp2(__builtin_fmaf(x[g >> 1][8 * (g & 1) + j], rowf, base));
                    sum += w[j];
                }
                const f4 s0 = *reinterpret_cast<const f4*>(hd + 64 + 16 * g + 4 * hf);
                const f4 s1 = *reinterpret_cast<const f4*>(hd + 64 + 16 * g + 8 + 4 * hf);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] *= s0[j];
                    w[4 + j] *= s1[j];
                }
                if constexpr (two) split8(w, ph[g], pl[g]);
                else ph[g] = round8(w);
            }
            l = __builtin_fmaf(sum, nu * (1.0f / kPScale), l * f);
            if (__any(f != 1.0f)) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] *= f;
            }
            const h8* p = reinterpret_cast<const h8*>(sv[par]) + lane;
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const h8 v = p[64 * (g * (D / 32) + i)];
                    o[i] = mfma32(v, ph[g], o[i]);
                    if constexpr (two) o[i] = mfma32(v, pl[g], o[i]);
                }
        }
    };
    if constexpr (DT == kF16) {
        if (seen_by(first) < kTwoTerms) run(std::true_type());
        else run(std::false_type());
    } else {
        run(std::bool_constant<SPLIT>());
    }
    wait_loads<0>();  // none may land in LDS that is another workgroup's

    if (!has_row) return;
    l = sum_halves(l);
    const int64_t orow = (int64_t)tok * a.Hq + head, prow = (int64_t)split * a.T * a.Hq + orow;
    float f = nu * (1.0f / kPScale);
    if (hf == 0) mark_row(a, split, orow, m * rowf, l);
    if (a.nrows == 1) f *= l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const int d = 32 * i + 2 * j + 4 * hf;
            const f4 v = {o[i][j] * f, o[i][j + 1] * f, o[i][j + 2] * f, o[i][j + 3] * f};
            if (a.nrows > 1) *reinterpret_cast<f4*>(a.rpart + prow * D + d) = v;
            else store4(a.out, DT, tok * a.o_token + head * a.o_head + d, v);
        }
}

// Rows up to which 16 a workgroup over the same keys are faster than 128 (us over
// 16000 keys, INT8, bf16: 8 / 16 tokens of 4 heads of 128 to a key head 29 / 42
// against 51 / 53; 8 / 16 tokens of 6 heads of 256 39 / 59 against 85 / 96).
constexpr int few_rows(int D) { return D == 256 ? 128 : 64; }
constexpr int64_t kMostBlocks = 1 << 23;  // of 256 threads: a grid has fewer than 2^32

// Splits, by the keys that the table has room for.  Single tokens: a split's keys cost
// a workgroup no more than its start does while they are few, and one long sequence
// among short ones must not be one workgroup's; so as many as bring a workgroup's keys
// down to kSplitMin while compute units are idle, and to kSplitKeys at least.  Chunks:
// the number that wastes the least of the last round of workgroups, each split
// of at least kSplitRows keys.
constexpr int kSplitMin = 64, kSplitMixed = 1024, kSplitKeys = 2048, kSplitRows = 512, kSplitMost = 64;

// The splits of a row joined: D/4 lanes a split and NG splits of a row at a
// time, their sums then in the order of the splits.  First the rows that
// attn_keys_kernel split, then the other kernels'.
template <int D, int NG>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    constexpr int L = D / 4, RW = 256 / L / NG;  // rows a workgroup
    __shared__ __align__(16) float sv[NG > 1 ? 256 / L : 1][D];
    __shared__ float sw[256 / L][kSplitMost];
    const int part = threadIdx.x / L, g = part % NG, d = 4 * (threadIdx.x % L);
    int64_t row = (int64_t)blockIdx.x * RW + part / NG;
    const int64_t nk = a.nkeys > 1 ? a.krows : 0;
    const bool keys = row < nk;
    const int64_t n = keys ? nk : (int64_t)a.T * a.Hq;  // rows of this kind
    if (!keys) row -= nk;
    const int nsplit = keys ? a.nkeys : a.nrows;
    const f2* const ml = keys ? a.kml : a.rml;
    const float* const sums = keys ? a.kpart : a.rpart;
    int tok = 0, head = 0;
    bool mine = row < n && nsplit > 1;
    if (keys && a.kper) {
        const int r = (int)(row % a.kper), h = (int)(row / a.kper % a.H), b = (int)(row / a.kper / a.H);
        const Seq sq = sequence(a, b);
        mine = (int64_t)sq.n * a.G <= a.few && r < sq.n * a.G;
        tok = sq.q0 + r / a.G;
        head = h * a.G + r % a.G;
    } else if (mine) {
        tok = (int)(row / a.Hq);
        head = (int)(row % a.Hq);
        mine = !(a.cu && (tok < a.cu[0] || tok >= a.cu[a.B])) && !(ml[row].y < 0.0f);
    }
    f4 v = {0, 0, 0, 0};
    float sum = 0.0f;
    // The splits' maxima and sums first, one or more a lane; sw: a split's weight.
    {
        constexpr int PER = kSplitMost / L;
        const int lane = threadIdx.x % L;
        f2 x[PER];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int s = lane + L * i;
            x[i] = mine && s < nsplit ? ml[s * n + row] : (f2){-INFINITY, 0.0f};
            top = fmaxf(top, x[i].x);
        }
#pragma unroll
        for (int st = 1; st < L; st *= 2) top = fmaxf(top, __shfl_xor(top, st));
        const float safe = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float f = fast_exp2(x[i].x - safe);
            sum += x[i].y == 0.0f && x[i].x == -INFINITY ? 0.0f : f * x[i].y;
            // An empty split's sums add nothing and are not read: marked by a weight below zero.
            sw[part][lane + L * i] = x[i].y == 0.0f && x[i].x == -INFINITY ? -1.0f : f;
        }
#pragma unroll
        for (int st = 1; st < L; st *= 2) sum += __shfl_xor(sum, st);
    }
    if (mine) {
#pragma unroll 8
        for (int s = g; s < nsplit; s += NG) {
            const float f = sw[part][s];
            if (f < 0.0f) continue;
            v += *reinterpret_cast<const f4*>(sums + (s * n + row) * D + d) * f;
        }
    }
    if constexpr (NG > 1) {
        *reinterpret_cast<f4*>(&sv[part][d]) = v;
        __syncthreads();
        if (g > 0) return;
#pragma unroll
        for (int i = 1; i < NG; ++i) v += *reinterpret_cast<const f4*>(&sv[part + i][d]);
    }
    if (!mine) return;
    v *= sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    store4(a.out, a.dt, tok * a.o_token + head * a.o_head + d, v);
}

// ------------------------------------------------------------------ host

struct AttnPlan {
    int keys, ntile16, rows, nslots;  // which kernels run, workgroups a sequence, slots of the rows kernels
    int lone;                        // the keys kernel's sequences are mostly of one token
    int nkeys, nrows;                // splits of the keys: of the two kinds of kernels
    int64_t krows;                   // rows that attn_keys_kernel has sums for where it splits
    int kper;                        // of each sequence and key head; 0: of each token and head
    int tiles, by_seq, direct;       // of an unpacked copy, 0: none; one for each sequence; attn_rows_kernel runs
    size_t copy, kpart, rpart, bytes;  // of the copies, of the two kinds' sums (without maxima), of the workspace
};

// Copies are made for calls of kUnpackRows rows or more (heads of 256, whose sums in
// fp32 leave attn_rows_kernel no registers for the unpacking, of kUnpackRows256: over
// 2000 keys 109 -> 72 us at 768 rows, 95 -> 62 at 192, bf16 60 -> 58 and 52 -> 51;
// heads of 128 are even at 512): of every sequence where
// they have kUnpackMean rows on average, else of those of kBigRows or more; at
// most kUnpackMost bytes.
constexpr int kUnpackRows = 512, kUnpackRows256 = 64, kUnpackMean = 64;
constexpr size_t kUnpackMost = (size_t)4 << 30;
// Bytes that the split rows' sums of either kind of kernel may take: a table of many
// columns asks for many splits, and a call may have many rows.
constexpr size_t kPartMost = (size_t)512 << 20;

AttnPlan plan_attn(int T, int B, int Hq, int H, int D, bool cu, int64_t capacity, int dtype, int n_cu) {
    const int G = Hq / H;
    AttnPlan p{};
    const int few = few_rows(D);
    const size_t row_bytes = (size_t)D * 4 + 8;  // a row's sums, maximum and sum of one split
    p.rows = cu ? (int64_t)T * G > few : G > few;
    // One sequence alone is never worth a second launch that may find nothing to do.
    p.keys = G <= few && !(p.rows && B == 1);
    p.nslots = cu ? (int)((int64_t)T * G / kRowTile) + B : B * ((G + kRowTile - 1) / kRowTile);
    p.nkeys = p.nrows = 1;
    if (p.keys) {
        p.ntile16 = (int)((std::min<int64_t>(few, (cu ? (int64_t)T : 1) * G) + 15) / 16);
        const int64_t wgs = (int64_t)B * H * (cu ? 1 : p.ntile16);
        // With chunks among the sequences the single tokens are not what fills the units,
        // but one of a long context must not outlast the chunks.
        const int64_t fill = (2 * n_cu + wgs - 1) / wgs;
        const bool mixed = (int64_t)T * G > few * (int64_t)B;
        p.lone = p.ntile16 == 1 || mixed;
        const int64_t idle = mixed ? std::min<int64_t>(16, capacity / kSplitMixed) : std::min(fill, capacity / kSplitMin);
        // The sequences' rows by themselves where that is fewer than all of the call's: one
        // long chunk beside single tokens has no sums here.
        const int64_t kper = std::min<int64_t>(few, (int64_t)T * G), by_seq = (int64_t)B * H * kper;
        p.krows = (int64_t)T * Hq;
        if (cu && by_seq < p.krows) {
            p.krows = by_seq;
            p.kper = (int)kper;
        }
        const int64_t blocks = kMostBlocks / ((int64_t)B * H * p.ntile16), room = (int64_t)(kPartMost / (p.krows * row_bytes));
        const int64_t most = std::max<int64_t>(1, std::min({(int64_t)kSplitMost, blocks, room}));
        p.nkeys = (int)std::max<int64_t>(1, std::min(std::max(idle, capacity / kSplitKeys), most));
    }
    if (p.rows) {
        const int64_t wgs = (int64_t)p.nslots * H, room = (int64_t)n_cu * (D == 256 || (D == 128 && dtype == kF32) ? 1 : 2);
        // A prompt's workgroups, the longest first, fill the last round by themselves.
        const bool causal = wgs >= room && 2 * (int64_t)T >= capacity * B;
        double best = 1e30;
        const auto may = [&](int64_t s) {
            return s * kSplitRows <= capacity && wgs < 4 * room && !causal && s * wgs <= kMostBlocks &&
                   (size_t)s * T * Hq * row_bytes <= kPartMost;
        };
        for (int64_t s = 1; s <= 16 && (s == 1 || may(s)); ++s) {
            const double cost = (double)((wgs * s + room - 1) / room) / s * (1.0 + 0.02 * (s - 1));
            if (cost < best) {
                best = cost;
                p.nrows = (int)s;
            }
        }
    }
    p.direct = p.rows;
    if (p.rows && (int64_t)T * G >= (D == 256 ? kUnpackRows256 : kUnpackRows)) {
        const int64_t tiles = (capacity + kKeyTile - 1) / kKeyTile, some = (int64_t)T * G / kBigRows + 1;
        const size_t one = (size_t)H * tiles * (kKeyTile * D * 4 + kHead);
        p.by_seq = (int64_t)T * G >= (int64_t)kUnpackMean * B && (one == 0 || (size_t)B <= kUnpackMost / one);
        const int64_t copies = p.by_seq ? B : some;
        if (one > 0 && (size_t)copies <= kUnpackMost / one) {
            p.tiles = (int)tiles;
            p.copy = copies * one;
            p.direct = !p.by_seq;
        }
    }
    const size_t nk = p.nkeys > 1 ? (size_t)p.nkeys * p.krows : 0, nr = p.nrows > 1 ? (size_t)p.nrows * T * Hq : 0;
    p.kpart = nk * D * 4;
    p.rpart = nr * D * 4;
    p.bytes = p.copy + (nk + nr) * row_bytes;
    return p;
}

int cu_count() {
    static int n[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (n[dev] == 0) {
        int v = 0;
        n[dev] = hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0 ? v : 256;
    }
    return n[dev];
}

template <int D, int KIND, int DT>
void launch3(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    const unsigned keys = p.keys ? (unsigned)a.B * a.H * a.ntile16 * a.nkeys : 0;
    const unsigned unpack = (unsigned)std::min<int64_t>((int64_t)a.B * a.H * a.tiles, 2048);
    // At one workgroup a unit the copy would go at half its rate.
    const bool alone = p.lone && keys_per_unit(D, DT, true) == 1;
    if (keys && unpack && !alone) {
        attn_keys_unpack_kernel<D, KIND, DT><<<keys + unpack, 256, 0, st>>>(a, keys);
    } else {
        constexpr bool kLone = keys_per_unit(D, DT, true) != keys_per_unit(D, DT, false);
        if (keys && p.lone) attn_keys_kernel<D, KIND, DT, kLone><<<keys, 256, 0, st>>>(a);
        else if (keys) attn_keys_kernel<D, KIND, DT, false><<<keys, 256, 0, st>>>(a);
        if (unpack) attn_unpack_kernel<D, KIND><<<unpack, 256, 0, st>>>(a);
    }
    if (p.direct) attn_rows_kernel<D, KIND, DT><<<(unsigned)a.nslots * a.H * a.nrows, 256, 0, st>>>(a);
    if (p.tiles) attn_tiles_kernel<D, DT><<<(unsigned)a.nslots * a.H * a.nrows, 256, 0, st>>>(a);
}

template <int D, int KIND>
void launch2(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    if (a.dt == kF32) launch3<D, KIND, kF32>(a, p, st);
    else if (a.dt == kBF16) launch3<D, KIND, kBF16>(a, p, st);
    else launch3<D, KIND, kF16>(a, p, st);
}

template <int D>
void launch1(const AttnArgs& a, const AttnPlan& p, int kind, hipStream_t st) {
    if (kind == kInt8) launch2<D, kInt8>(a, p, st);
    else launch2<D, kFp8>(a, p, st);
    if (a.nkeys > 1 || a.nrows > 1) {
        // Few rows: all of a workgroup's lanes for one, so that many splits are read at once.
        constexpr int NG = 256 / (D / 4);
        const int64_t n = (a.nkeys > 1 ? a.krows : 0) + (a.nrows > 1 ? (int64_t)a.T * a.Hq : 0);
        if (n <= 2048) attn_join_kernel<D, NG><<<(unsigned)n, 256, 0, st>>>(a);
        else attn_join_kernel<D, 1><<<(unsigned)((n + NG - 1) / NG), 256, 0, st>>>(a);
    }
}

bool check_shape(const i4_kv_cache* c, int T, int B, int heads, int table_w, bool has_cu, int* pshift) {
    if (!c || (c->kind != kInt8 && c->kind != kFp8)) {
        bq_set_error("paged_attention: needs a cache of kind 0 (INT8) or 1 (e4m3)");
        return false;
    }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        bq_set_error("paged_attention: head_dim must be 64, 128 or 256, got %d", c->head_dim);
        return false;
    }
    int s = 4;
    while (s < 10 && (1 << s) != c->page_size) ++s;
    if ((1 << s) != c->page_size || c->num_pages < 1 || c->kv_heads < 1 || c->kv_heads > 4096 ||
        c->num_pages > (INT32_MAX >> s)) {
        bq_set_error("paged_attention: needs a page size of 16 to 1024 that is a power of two, at least one page, 1 to "
                     "4096 heads and fewer than 2^31 slots (got page size %d, %d pages, %d heads)",
                     c->page_size, c->num_pages, c->kv_heads);
        return false;
    }
    if (T < 0 || B < 0 || heads < 1 || heads > 65536 || heads % c->kv_heads || table_w < 0 ||
        table_w > (INT32_MAX >> s) || (!has_cu && T != B)) {
        bq_set_error("paged_attention: needs query heads in multiples of the %d key-value heads, and one token a "
                     "sequence where no offsets are given (got %d tokens, %d sequences, %d heads, %d table columns)",
                     c->kv_heads, T, B, heads, table_w);
        return false;
    }
    // A launch has fewer than 2^24 workgroups (eight a sequence and head at most here), and keys are counted in 32
    // bits with some room.
    if ((int64_t)T * heads > (1 << 28) || (int64_t)B * c->kv_heads > kMostBlocks / 8 || table_w > ((1 << 30) >> s)) {
        bq_set_error("paged_attention: %d tokens of %d heads in %d sequences of up to %d pages are too much for one call", T,
                     heads, B, table_w);
        return false;
    }
    *pshift = s;
    return true;
}

}  // namespace

extern "C" {

int64_t i4_paged_attention_workspace(int kv_heads, int page_size, int head_dim, int T, int B, int heads, int dtype,
                                     int table_w, int has_cu) {
    i4_kv_cache c{};
    c.num_pages = 1;
    c.kv_heads = kv_heads;
    c.page_size = page_size;
    c.head_dim = head_dim;
    const i4_kv_cache* cache = &c;
    int ps = 0;
    if (!check_shape(cache, T, B, heads, table_w, has_cu != 0, &ps)) return -2;
    if (T == 0 || B == 0) return 0;
    return (int64_t)plan_attn(T, B, heads, cache->kv_heads, cache->head_dim, has_cu != 0, (int64_t)table_w << ps, dtype,
                              cu_count())
        .bytes;
}

int i4_paged_attention_dev(const i4_kv_cache* cache, const void* dQ, int64_t q_token, int64_t q_head, int T, int heads,
                           int dtype, const int32_t* dTable, int64_t table_row, int table_w, const int32_t* dKvLens,
                           const int32_t* dCu, int B, float scale, void* dOut, int64_t o_token, int64_t o_head,
                           void* dWork, int64_t work_bytes, void* stream) {
    int ps = 0;
    if (!check_shape(cache, T, B, heads, table_w, dCu != nullptr, &ps)) return -2;
    if (dtype < kF32 || dtype > kF16 || !(scale > 0.0f) || scale > 1e30f) {
        bq_set_error("paged_attention: needs a type of 0 to 2 and a positive finite scale (got %d, %g)", dtype, scale);
        return -2;
    }
    if (T == 0 || B == 0) return 0;
    if (!cache->k || !cache->v || !cache->k_scale || !cache->v_scale || !dQ || !dOut || !dKvLens ||
        (table_w > 0 && !dTable)) {
        bq_set_error("paged_attention: null device pointer");
        return -2;
    }
    AttnArgs a{};
    a.q = dQ;
    a.out = dOut;
    a.q_token = q_token;
    a.q_head = q_head;
    a.o_token = o_token;
    a.o_head = o_head;
    a.kp = static_cast<const uint8_t*>(cache->k);
    a.vp = static_cast<const uint8_t*>(cache->v);
    a.ks = cache->k_scale;
    a.vs = cache->v_scale;
    a.table = dTable;
    a.table_row = table_row;
    a.table_w = table_w;
    a.kv_lens = dKvLens;
    a.cu = dCu;
    a.T = T;
    a.B = B;
    a.Hq = heads;
    a.H = cache->kv_heads;
    a.G = heads / cache->kv_heads;
    a.P = cache->num_pages;
    a.pshift = ps;
    a.dt = dtype;
    a.scale = scale * kLog2e;
    const AttnPlan p =
        plan_attn(T, B, heads, a.H, cache->head_dim, dCu != nullptr, (int64_t)table_w << ps, dtype, cu_count());
    if (p.bytes > 0 && (!dWork || work_bytes < (int64_t)p.bytes)) {
        bq_set_error("paged_attention: needs a workspace of %zu bytes, got %lld", p.bytes, (long long)work_bytes);
        return -4;
    }
    a.nkeys = p.nkeys;
    a.few = p.keys ? few_rows(cache->head_dim) : 0;
    a.by_seq = p.by_seq;
    a.big = !p.tiles ? INT32_MAX : p.by_seq ? a.few + 1 : kBigRows;
    a.nrows = p.nrows;
    a.ntile16 = p.ntile16;
    a.nslots = p.nslots;
    a.tiles = p.tiles;
    a.unpacked = static_cast<uint8_t*>(dWork);
    uint8_t* const sums = static_cast<uint8_t*>(dWork) + p.copy;
    a.kpart = reinterpret_cast<float*>(sums);
    a.rpart = reinterpret_cast<float*>(sums + p.kpart);
    a.kml = reinterpret_cast<f2*>(sums + p.kpart + p.rpart);
    a.rml = a.kml + (p.nkeys > 1 ? p.nkeys * p.krows : 0);
    a.krows = p.krows;
    a.kper = p.kper;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (cache->head_dim == 64) launch1<64>(a, p, cache->kind, st);
    else if (cache->head_dim == 128) launch1<128>(a, p, cache->kind, st);
    else launch1<256>(a, p, cache->kind, st);
    return launched("paged_attention") ? 0 : -5;
}

}  // extern "C"
