// Attention of trees of drafted tokens over the quantized paged cache.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
//
// for the n nodes i of each sequence's tree, whose keys and values are the last n
// in the cache; j goes over the keys before them, node i's ancestors and node i.
//
// Numerics are those of the causal kernels (paged_attn.hip): the cache's numbers
// enter both products exactly, as fp16; fp32 queries and their weights are two fp16
// terms, as are fp16's weights; bf16's weights are one.  Sums, maxima and
// partial sums are fp32.
//
// A tree has tens of rows a key-value head (nodes times the query heads of one),
// which all see the same keys but for the tree itself.  So a workgroup takes up
// to 128 rows and a share of the keys: each key is loaded and unpacked once for
// all of them.  WR of its four waves take 32 rows each, and where the rows are
// fewer the waves share out a tile's keys instead (4 / WR groups, joined at the
// end).  Tiles go from the last keys to the first, so that the tree comes first and
// a lane follows its node's parents down once: a tile's mask is the 32 bits that
// it passes.  Tiles before the tree have no mask.
#include "attn_common.h"

#include <algorithm>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

constexpr int kTreeNodes = 1024;

struct TreeArgs {
    const void* q;
    void* out;
    int64_t q_token, q_head, o_token, o_head;  // element strides
    const uint8_t* kp;
    const uint8_t* vp;
    const float* ks;
    const float* vs;
    const int32_t* table;
    const int32_t* kv_lens;
    const int32_t* cu;  // null: one node a sequence
    const int32_t* parents;
    float* part;        // [splits][T * Hq][D] where keys are split
    f2* ml;             // [splits][T * Hq]: maximum and sum
    int64_t table_row;
    int T, B, Hq, H, G, P, pshift, table_w, nslots, splits, chunk;  // chunk: keys a split
    float scale;  // softmax scale * log2(e)
};

struct Seq {
    int q0, n, kv;  // first node, nodes, keys
};

__device__ inline Seq sequence(const TreeArgs& a, int b) {
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

// The RT rows of a slot: their sequence (-1: none) and the first of them.  Sequence b's
// tiles take the slots from cu[b] * G / RT + b on, which leaves room for all
// without a pass over the lengths.
template <int RT>
__device__ inline int rows_of_slot(const TreeArgs& a, int slot, Seq& sq, int& first) {
    const int per = (a.G + RT - 1) / RT;
    int b = 0;
    if (a.cu) {
        int hi = a.B;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            const int64_t start = (int64_t)min(max(a.cu[mid], 0), a.T) * a.G / RT + mid;
            if (start <= slot) b = mid;
            else hi = mid;
        }
    } else {
        b = slot / per;
    }
    sq = sequence(a, b);
    const int64_t rows = (int64_t)sq.n * a.G;
    const int64_t at = (slot - (a.cu ? (int64_t)sq.q0 * a.G / RT + b : (int64_t)b * per)) * RT;
    first = (int)at;
    return at < 0 || at >= rows ? -1 : b;
}

// Splits of a sequence: a tree that is too large has one, which says so.
__device__ inline int splits_of(const TreeArgs& a, const Seq& sq) {
    return sq.n > kTreeNodes ? 1 : max((sq.kv + a.chunk - 1) / a.chunk, 1);
}

// A row's queries as operands (values 16 s + 8 (lane / 32) + 0..7 for slab s,
// from element `at` on), scaled; returns what a score is worth in log2.
template <int D, int DT>
__device__ inline float load_queries(const TreeArgs& a, int64_t at, h8* hi, h8* lo) {
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

// Keys of a tile: 32 a wave where the waves share them out, else 64.
constexpr int tile_keys(int WR) { return WR == 1 ? 128 : 64; }
constexpr int row_k(int D) { return D + 8; }   // LDS rows of a key and of its values: reads of one
constexpr int row_v(int D) { return D + 16; }  // instruction fall on unlike banks
constexpr int per_unit(int D, int DT) { return D == 256 ? 1 : D == 128 && DT == kF32 ? 1 : 2; }

template <int D, int KIND, int DT, int WR>
__global__ __launch_bounds__(256, per_unit(D, DT)) void tree_keys_kernel(TreeArgs a) {
    constexpr bool SPLIT = DT == kF32, PSPLIT = DT != kBF16;  // two terms of the queries, and of the weights
    constexpr int WK = 4 / WR, RT = 32 * WR, KT = tile_keys(WR), KW = KT / WK, U = KW / 32;
    constexpr int KS = row_k(D), VS = row_v(D);
    constexpr int NC = KT * D / 4096;  // 16-byte chunks a thread loads of a tile's keys (and of its values)
    constexpr int per_row = D / 16;
    constexpr int kBytes = std::max(KT * (KS + VS) * 2, (WK - 1) * WR * D * 128);
    __shared__ __align__(16) uint8_t lds[kBytes];
    __shared__ __align__(16) float sks[KT], svs[KT];
    __shared__ float smax[KT / 32], sm[4][32], sl[4][32], sf[4][32];
    __shared__ uint32_t svalid[KT / 32];
    __shared__ int16_t up[kTreeNodes];
    _Float16 *const sk = reinterpret_cast<_Float16*>(lds), *const sv = sk + KT * KS;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, hf = lane >> 5, rg = wave % WR, kg = wave / WR;
    const int h = blockIdx.x % a.H, ss = blockIdx.x / a.H, split = ss % a.splits, slot = ss / a.splits;
    Seq sq;
    int first;
    const int b = rows_of_slot<RT>(a, slot, sq, first);
    if (b < 0) return;
    const int nsplit = splits_of(a, sq);
    if (split >= nsplit) return;
    const int rows = (int)min((int64_t)sq.n * a.G, (int64_t)first + RT);
    const int row = first + 32 * rg + r32;
    const bool has_row = row < rows, spoilt = sq.n > kTreeNodes;
    const int node = has_row ? row / a.G : 0, tok = sq.q0 + node, head = h * a.G + (has_row ? row % a.G : 0);
    const int ctx = sq.kv - sq.n;  // place of node 0; below zero where the cache lacks the first nodes

    const int k0 = split * a.chunk, k1 = spoilt ? 0 : min(k0 + a.chunk, sq.kv);
    const int t0 = k0 / KT, t1 = (k1 + KT - 1) / KT;
    int t = t1 - 1;
    const int32_t* table = a.table + b * a.table_row;

    u4 kraw[NC], vraw[NC];
    int64_t grow[NC];
    float ksc = 0.0f, vsc = 0.0f;
    bool sc_bad = true;
    // Cache row of the 16 keys from `key` on; -1 where the sequence or its table has none.
    const auto group_row = [&](int key) -> int64_t {
        const int page = table[min(key, sq.kv - 1) >> a.pshift];
        const bool is = key < sq.kv && page >= 0 && page < a.P;
        return is ? (((int64_t)page * a.H + h) << a.pshift) + (key & ((1 << a.pshift) - 1)) : -1;
    };
    const auto load = [&](int tile) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int kr = (wave * 64 + 256 * i) / per_row;  // the wave's first row of this pass
            grow[i] = group_row(KT * tile + (kr & ~15));
            const int64_t at = (grow[i] < 0 ? 0 : grow[i]) + ((tid + 256 * i) / per_row & 15);
            kraw[i] = *reinterpret_cast<const u4*>(a.kp + at * D + 16 * (tid % per_row));
            vraw[i] = *reinterpret_cast<const u4*>(a.vp + at * D + 16 * (tid % per_row));
        }
        if (tid < KT) {
            const int64_t at = group_row(KT * tile + (tid & ~15));
            sc_bad = at < 0 || KT * tile + tid >= sq.kv;
            ksc = sc_bad ? 0.0f : a.ks[at + (tid & 15)];
            vsc = sc_bad ? 0.0f : a.vs[at + (tid & 15)];
        }
    };
    if (t >= t0) load(t);
    if (k1 > ctx)
        for (int i = tid; i < min(sq.n, kTreeNodes); i += 256) {
            const int p = a.parents[sq.q0 + i];
            up[i] = (int16_t)(p >= 0 && p < i ? p : -1);
        }

    h8 qh[D / 16], ql[SPLIT ? D / 16 : 1];
    const float rowf = load_queries<D, DT>(a, tok * a.q_token + head * a.q_head + 8 * hf, qh, ql);

    f16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
    // A tile's weights are computed in units in which a probability of 1 is 2^9 / nu, at
    // most 2^119 of those eight, so that a lane's add up to less than fp32 holds.
    constexpr float least = 0x1p-110f;
    float m = -INFINITY, l = 0.0f, nu = least, peak = 0.0f, unit = __builtin_log2f(kPScale / least);
    int at_node = has_row ? node : -1;  // the next of the row's node and its ancestors

    for (; t >= t0; --t) {
        const int key0 = KT * t;
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
        if (tid < KT) {
            // A value scale of NaN goes with the key's, whose score a row that does
            // not see the key leaves out; times a probability of zero it would not.
            const bool nan = vsc != vsc;
            sks[tid] = nan ? vsc : ksc;
            svs[tid] = nan ? 0.0f : vsc;
            float vmax = nan ? 0.0f : vsc;
#pragma unroll
            for (int st = 1; st < 32; st *= 2) vmax = fmaxf(vmax, __shfl_xor(vmax, st));
            const uint64_t valid = __ballot(!sc_bad);
            if ((lane & 31) == 0) {
                smax[tid >> 5] = vmax;
                svalid[tid >> 5] = (uint32_t)(valid >> (lane & 32));
            }
        }
        __syncthreads();
        if (t > t0) load(t - 1);

        f16 s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < 16; ++j) s[u][j] = 0.0f;
            const _Float16* p = sk + (KW * kg + 32 * u + r32) * KS + 8 * hf;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const h8 k = *reinterpret_cast<const h8*>(p + 16 * i);
                s[u] = mfma32(k, qh[i], s[u]);
                if constexpr (SPLIT) s[u] = mfma32(k, ql[i], s[u]);
            }
        }
        // Scores times the key scales; result register j holds key 8 (j / 4) + 4 hf + j % 4.
        float vmax = 0.0f;
        bool all = key0 + KT <= ctx;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vmax = fmaxf(vmax, smax[U * kg + u]);
            all = all && svalid[U * kg + u] == 0xFFFFFFFFu;
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const f4 sc = *reinterpret_cast<const f4*>(sks + KW * kg + 32 * u + 2 * j + 4 * hf);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[u][j + e] *= sc[e];
            }
        }
        if (!all) {
            vmax = 0.0f;
#pragma unroll
            for (int u = U - 1; u >= 0; --u) {
                // The keys of these 32 that the row sees: those before the tree, and the nodes that
                // its path to the root passes.
                const int n0 = key0 + KW * kg + 32 * u - ctx;  // the first one's node
                uint32_t bits = n0 <= -32 ? 0xFFFFFFFFu : n0 < 0 ? (1u << -n0) - 1 : 0u;
                if (n0 + 32 > 0) {
                    while (at_node >= n0 + 32) at_node = up[at_node];
                    while (at_node >= max(n0, 0)) {
                        bits |= 1u << (at_node - n0);
                        at_node = up[at_node];
                    }
                }
                bits &= has_row ? svalid[U * kg + u] : 0u;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int k = 8 * (j / 4) + 4 * hf + j % 4;
                    const bool out = !(bits >> k & 1);
                    s[u][j] = out ? -INFINITY : s[u][j];
                    vmax = fmaxf(vmax, out ? 0.0f : svs[KW * kg + 32 * u + k]);
                }
            }
            vmax = max_halves(vmax);
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 16; j += 2) top = fmaxf(fmaxf(top, s[u][j]), s[u][j + 1]);
        top = max_halves(top);
        // The reference moves only once a row's scores pass it by kSlack, its units where the
        // values' size leaves their range.
        const bool moves = (top - m) * rowf > kSlack;
        float f = moves ? fast_exp2((m - top) * rowf) : 1.0f;
        m = moves ? top : m;
        l *= f;
        peak *= f;
        if (__any(vmax > nu * 8.0f || (vmax > 0.0f && vmax <= nu * 0x1p-4f))) {
            const float now = next_nu(nu, vmax, peak, least);
            f *= nu / now;
            unit = __builtin_log2f(kPScale / now);
            nu = now;
        }
        peak = fmaxf(peak, nu);
        if (__any(f != 1.0f)) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float bias = __builtin_fmaf(-ref, rowf, unit);
        // m rowf is rounded once here, by less than half while it is below 2^22; past that
        // the difference is taken first, else the largest weight would be 2 to that error.
        if (__any(__builtin_fabsf(ref) * rowf > 0x1p22f)) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 16; ++j) s[u][j] -= ref;
            bias = unit;
        }
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int g = 0; g < 2; ++g) {  // 16 keys
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = fast_exp2(__builtin_fmaf(s[u][8 * g + j], rowf, bias));
                    sum += w[j];
                }
                const float* const vp = svs + KW * kg + 32 * u + 16 * g + 4 * hf;
                const f4 s0 = *reinterpret_cast<const f4*>(vp), s1 = *reinterpret_cast<const f4*>(vp + 8);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] *= s0[j];
                    w[4 + j] *= s1[j];
                }
                h8 ph, pl;
                if constexpr (PSPLIT) split8(w, ph, pl);
                else ph = round8(w);
                const int i16 = lane & 15;
                const _Float16* p =
                    sv + (KW * kg + 32 * u + 16 * g + 4 * hf + (i16 >> 2)) * VS + 16 * (r32 >> 4) + 4 * (i16 & 3);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const h8 v = mx::join(read_tr(p + 32 * i), read_tr(p + 32 * i + 8 * VS));
                    o[i] = mfma32(v, ph, o[i]);
                    if constexpr (PSPLIT) o[i] = mfma32(v, pl, o[i]);
                }
            }
        l = __builtin_fmaf(sum, nu * (1.0f / kPScale), l);
    }

    l = sum_halves(l);
    float f = nu * (1.0f / kPScale), mlog = m * rowf;
    if constexpr (WK > 1) {
        // The groups' sums, joined in their order.
        __syncthreads();
        float* const so = reinterpret_cast<float*>(lds);
        constexpr int N = D / 2;  // a lane's sums
        if (hf == 0) {
            sm[wave][r32] = mlog;
            sl[wave][r32] = l;
            sf[wave][r32] = f;
        }
        if (kg > 0) {
            float* const mine = so + ((kg - 1) * WR + rg) * N * 64 + lane;
#pragma unroll
            for (int i = 0; i < N; ++i) mine[64 * i] = o[i / 16][i % 16];
        }
        __syncthreads();
        if (kg > 0) return;
        float top = mlog;
#pragma unroll
        for (int g = 1; g < WK; ++g) top = fmaxf(top, sm[g * WR + rg][r32]);
        const float safe = top == -INFINITY ? 0.0f : top;
        const float f0 = fast_exp2(mlog - safe);
        l *= f0;
        f *= f0;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= f;
        f = 1.0f;
#pragma unroll
        for (int g = 1; g < WK; ++g) {
            const float e = fast_exp2(sm[g * WR + rg][r32] - safe), w = e * sf[g * WR + rg][r32];
            l += e * sl[g * WR + rg][r32];
            const float* const its = so + ((g - 1) * WR + rg) * N * 64 + lane;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i / 16][i % 16] += w * its[64 * i];
        }
        mlog = top;
    }
    if (!has_row) return;
    const int64_t orow = (int64_t)tok * a.Hq + head, prow = (int64_t)split * a.T * a.Hq + orow;
    if (nsplit > 1) {
        if (hf == 0) a.ml[prow] = (f2){mlog, l};
    } else {
        f *= spoilt ? __builtin_nanf("") : l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const int d = 32 * i + 2 * j + 4 * hf;
            const f4 v = {o[i][j] * f, o[i][j + 1] * f, o[i][j + 2] * f, o[i][j + 3] * f};
            if (nsplit > 1) *reinterpret_cast<f4*>(a.part + prow * D + d) = v;
            else store4(a.out, DT, tok * a.o_token + head * a.o_head + d, v);
        }
}

// The splits of a row joined, in their order: a wave a row.
template <int D, int DT>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a) {
    constexpr int L = D / 4, NG = 64 / L;  // lanes a split, splits at a time
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * 4 + wave, n = (int64_t)a.T * a.Hq;
    if (row >= n) return;
    const int tok = (int)(row / a.Hq), head = (int)(row - (int64_t)tok * a.Hq);
    int b = tok;
    if (a.cu) {
        int hi = a.B;
        b = 0;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (a.cu[mid] <= tok) b = mid;
            else hi = mid;
        }
    }
    const Seq sq = sequence(a, b);
    const int nsplit = splits_of(a, sq);
    if (tok < sq.q0 || tok >= sq.q0 + sq.n || nsplit == 1) return;
    float top = -INFINITY;
    for (int s = lane; s < nsplit; s += 64) top = fmaxf(top, a.ml[s * n + row].x);
    top = max_wave(top);
    const float safe = top == -INFINITY ? 0.0f : top;
    f4 v = {0, 0, 0, 0};
    float sum = 0.0f;
    const int g = lane / L, d = 4 * (lane % L);
#pragma unroll 4
    for (int s = g; s < nsplit; s += NG) {
        const f2 x = a.ml[s * n + row];
        const f4 y = *reinterpret_cast<const f4*>(a.part + (s * n + row) * D + d);
        const bool none = x.y == 0.0f && x.x == -INFINITY;
        const float f = none ? 0.0f : fast_exp2(x.x - safe);
        sum += none ? 0.0f : f * x.y;
        v += none ? (f4){0, 0, 0, 0} : y * f;
    }
#pragma unroll
    for (int st = L; st < 64; st *= 2) {
        sum += __shfl_xor(sum, st);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], st);
    }
    if (g > 0) return;
    v *= sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    store4(a.out, DT, tok * a.o_token + head * a.o_head + d, v);
}

// ------------------------------------------------------------------ host

constexpr int64_t kMostBlocks = 1 << 23;  // of 256 threads: a grid has fewer than 2^32
constexpr size_t kPartMost = (size_t)512 << 20;
constexpr int kMostSplits = 1 << 16;

struct Plan {
    int wr, nslots, splits, chunk;
    size_t part, bytes;
};

// Rows a workgroup by the mean tree; keys a split so that there are a few workgroups
// for each place on the units while a split has its start's worth of keys.
Plan plan_tree(int T, int B, int Hq, int H, int D, bool cu, int64_t capacity, int dtype, int n_cu) {
    Plan p{};
    const int G = Hq / H;
    const int64_t mean = (((int64_t)T + B - 1) / B) * G;
    p.wr = mean <= 32 ? 1 : mean <= 64 ? 2 : 4;
    const int RT = 32 * p.wr, KT = tile_keys(p.wr);
    p.nslots = (int)(cu ? (int64_t)T * G / RT + B : (int64_t)B * ((G + RT - 1) / RT));
    const int64_t tiles = (int64_t)B * ((mean + RT - 1) / RT) * H, room = (int64_t)n_cu * per_unit(D, dtype);
    int64_t splits = std::max<int64_t>(1, (4 * room + tiles - 1) / tiles);
    int64_t chunk = (capacity + splits - 1) / splits;
    chunk = std::max<int64_t>(chunk, 128);
    const int64_t row_bytes = (int64_t)T * Hq * (D * 4 + 8);
    const int64_t most = std::max<int64_t>(
        1, std::min<int64_t>({(int64_t)kPartMost / row_bytes, kMostBlocks / ((int64_t)p.nslots * H), (int64_t)kMostSplits}));
    chunk = std::max(chunk, (capacity + most - 1) / most);
    chunk = (chunk + KT - 1) / KT * KT;
    p.chunk = (int)std::min<int64_t>(chunk, 1 << 30);
    p.splits = (int)std::max<int64_t>(1, (capacity + p.chunk - 1) / p.chunk);
    if (p.splits > 1) {
        p.part = (size_t)p.splits * T * Hq * D * 4;
        p.bytes = p.part + (size_t)p.splits * T * Hq * 8;
    }
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
void launch3(const TreeArgs& a, const Plan& p, hipStream_t st) {
    const unsigned blocks = (unsigned)((int64_t)a.nslots * a.H * a.splits);
    if (p.wr == 1) tree_keys_kernel<D, KIND, DT, 1><<<blocks, 256, 0, st>>>(a);
    else if (p.wr == 2) tree_keys_kernel<D, KIND, DT, 2><<<blocks, 256, 0, st>>>(a);
    else tree_keys_kernel<D, KIND, DT, 4><<<blocks, 256, 0, st>>>(a);
    if (a.splits > 1) tree_join_kernel<D, DT><<<(unsigned)(((int64_t)a.T * a.Hq + 3) / 4), 256, 0, st>>>(a);
}

template <int D, int KIND>
void launch2(const TreeArgs& a, const Plan& p, int dt, hipStream_t st) {
    if (dt == kF32) launch3<D, KIND, kF32>(a, p, st);
    else if (dt == kBF16) launch3<D, KIND, kBF16>(a, p, st);
    else launch3<D, KIND, kF16>(a, p, st);
}

template <int D>
void launch1(const TreeArgs& a, const Plan& p, int kind, int dt, hipStream_t st) {
    if (kind == kInt8) launch2<D, kInt8>(a, p, dt, st);
    else launch2<D, kFp8>(a, p, dt, st);
}

bool check_shape(const i4_kv_cache* c, int T, int B, int heads, int table_w, bool has_cu, int* pshift) {
    if (!c || (c->kind != kInt8 && c->kind != kFp8)) {
        bq_set_error("tree_attention: needs a cache of kind 0 (INT8) or 1 (e4m3)");
        return false;
    }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        bq_set_error("tree_attention: head_dim must be 64, 128 or 256, got %d", c->head_dim);
        return false;
    }
    int s = 4;
    while (s < 10 && (1 << s) != c->page_size) ++s;
    if ((1 << s) != c->page_size || c->num_pages < 1 || c->kv_heads < 1 || c->kv_heads > 4096 ||
        c->num_pages > (INT32_MAX >> s)) {
        bq_set_error("tree_attention: needs a page size of 16 to 1024 that is a power of two, at least one page, 1 to "
                     "4096 heads and fewer than 2^31 slots (got page size %d, %d pages, %d heads)",
                     c->page_size, c->num_pages, c->kv_heads);
        return false;
    }
    if (T < 0 || B < 0 || heads < 1 || heads > 65536 || heads % c->kv_heads || table_w < 0 ||
        table_w > ((1 << 30) >> s) || (!has_cu && T != B)) {
        bq_set_error("tree_attention: needs query heads in multiples of the %d key-value heads, tables of up to 2^30 keys "
                     "and one node a sequence where no offsets are given (got %d nodes, %d sequences, %d heads, %d table "
                     "columns)",
                     c->kv_heads, T, B, heads, table_w);
        return false;
    }
    // A launch has fewer than 2^24 workgroups: one for each 32 rows, and one a sequence and head.
    if ((int64_t)T * heads > (1 << 26) || (int64_t)B * c->kv_heads > kMostBlocks / 4) {
        bq_set_error("tree_attention: %d nodes of %d heads in %d sequences are too much for one call", T, heads, B);
        return false;
    }
    *pshift = s;
    return true;
}

}  // namespace

extern "C" {

int64_t i4_tree_attention_workspace(int kv_heads, int page_size, int head_dim, int T, int B, int heads, int dtype,
                                    int table_w, int has_cu) {
    i4_kv_cache c{};
    c.num_pages = 1;
    c.kv_heads = kv_heads;
    c.page_size = page_size;
    c.head_dim = head_dim;
    int ps = 0;
    if (!check_shape(&c, T, B, heads, table_w, has_cu != 0, &ps)) return -2;
    if (T == 0 || B == 0) return 0;
    return (int64_t)plan_tree(T, B, heads, kv_heads, head_dim, has_cu != 0, (int64_t)table_w << ps, dtype, cu_count()).bytes;
}

int i4_tree_attention_dev(const i4_kv_cache* cache, const void* dQ, int64_t q_token, int64_t q_head, int T, int heads,
                          int dtype, const int32_t* dTable, int64_t table_row, int table_w, const int32_t* dKvLens,
                          const int32_t* dCu, int B, const int32_t* dParents, float scale, void* dOut, int64_t o_token,
                          int64_t o_head, void* dWork, int64_t work_bytes, void* stream) {
    int ps = 0;
    if (!check_shape(cache, T, B, heads, table_w, dCu != nullptr, &ps)) return -2;
    if (dtype < kF32 || dtype > kF16 || !(scale > 0.0f) || scale > 1e30f) {
        bq_set_error("tree_attention: needs a type of 0 to 2 and a positive finite scale (got %d, %g)", dtype, scale);
        return -2;
    }
    if (T == 0 || B == 0) return 0;
    if (!cache->k || !cache->v || !cache->k_scale || !cache->v_scale || !dQ || !dOut || !dKvLens || !dParents ||
        (table_w > 0 && !dTable)) {
        bq_set_error("tree_attention: null device pointer");
        return -2;
    }
    TreeArgs a{};
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
    a.parents = dParents;
    a.T = T;
    a.B = B;
    a.Hq = heads;
    a.H = cache->kv_heads;
    a.G = heads / cache->kv_heads;
    a.P = cache->num_pages;
    a.pshift = ps;
    a.scale = scale * kLog2e;
    const Plan p = plan_tree(T, B, heads, a.H, cache->head_dim, dCu != nullptr, (int64_t)table_w << ps, dtype, cu_count());
    if (p.bytes > 0 && (!dWork || work_bytes < (int64_t)p.bytes)) {
        bq_set_error("tree_attention: needs a workspace of %zu bytes, got %lld", p.bytes, (long long)work_bytes);
        return -4;
    }
    a.nslots = p.nslots;
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.part = static_cast<float*>(dWork);
    a.ml = reinterpret_cast<f2*>(static_cast<uint8_t*>(dWork) + p.part);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (cache->head_dim == 64) launch1<64>(a, p, cache->kind, dtype, st);
    else if (cache->head_dim == 128) launch1<128>(a, p, cache->kind, dtype, st);
    else launch1<256>(a, p, cache->kind, dtype, st);
    return launched("tree_attention") ? 0 : -5;
}

}  // extern "C"
