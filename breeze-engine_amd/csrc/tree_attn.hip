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
// which all see the same keys but for the tree itself.  So a workgroup takes 32, 64 or
// 128 rows and a share of the keys: each key is loaded and unpacked once for
// all of them.  A wave takes 16 or 32 of the rows, and where that leaves waves over
// they share out a tile's keys, joined at the end.  Tiles go from the last keys to the
// first, so that the tree comes first and a lane follows its node's parents down once: a
// tile's mask is the 32 bits that it passes.  Tiles before the tree have no mask.
//
// The tiles of all units (a sequence, a key-value head, up to 128 rows), one unit
// after another, are cut into equal shares, one a workgroup, whatever the sequences'
// lengths, which the host does not read; each workgroup sums up the lengths for
// itself.  A unit that is cut leaves its parts' sums to tree_join_kernel.
//
// What bounds it.  Few rows of many sequences: HBM, less what unpacking does not hide (8
// nodes of each of 64 sequences behind 100 to 16000 keys, 32/8 heads of 128, e4m3, bf16:
// 151 us, 0.7 of a copy's rate).  From about 64 rows on, issue: of a compute unit's cycles
// (32 nodes of 16 sequences, 51 us, of which the join is 12) vector instructions take
// half, matrix instructions 0.29, LDS 0.4, and a wave waits a third of its time, at two
// waves a SIMD, which is what the registers hold.  Tried there and no faster: two LDS
// buffers and one barrier a tile, the next tile's loads among the products, waves started
// half a tile apart.  One sequence: latency (12 nodes behind 4100 keys 26 us: two
// launches, five dependent reads, 82 KB of sums a share written and read).
#include "attn_common.h"

#include <algorithm>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

typedef int i2 __attribute__((ext_vector_type(2)));

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
    float* part;        // [2 shares][rows a unit][D]: sums of cut units, a share's first and last one
    f2* ml;             // [2 shares][rows a unit]: maximum and sum
    i2* shares;         // [slots][H]: a unit's first and last share
    int64_t table_row;
    int T, B, H, G, P, pshift, table_w, nslots, grid;  // grid: shares
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

// Lane `who`'s value, as the scalar unit's.
__device__ inline int64_t lane_of(int64_t x, int who) {
    const int lo = __builtin_amdgcn_readlane((int)x, who), hi = __builtin_amdgcn_readlane((int)(x >> 32), who);
    return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}
// The sum over a wave's lanes up to this one.
__device__ inline int64_t scan_wave(int64_t x) {
    const auto step = [&](auto control, auto rows) {  // adds the lane's below, or a row's last one's; 0 where there is none
        const int lo = __builtin_amdgcn_update_dpp(0, (int)x, decltype(control)::value, decltype(rows)::value, 0xF, true);
        const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), decltype(control)::value, decltype(rows)::value, 0xF, true);
        x += (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
    };
    step(std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xF>());  // row_shr:1, 2, 4, 8 within 16 lanes
    step(std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xF>());
    step(std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xF>());
    step(std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xF>());
    step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xA>());  // row_bcast:15 to rows 1 and 3
    step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xC>());  // row_bcast:31 to rows 2 and 3
    return x;
}

// x / y of whole numbers up to 2^53: the fp64 quotient is rounded to a whole number
// only where it is one.  A tenth of the instructions of a division in 64-bit integers.
__device__ inline int64_t over(int64_t x, int64_t y) { return (int64_t)((double)x / (double)y); }

// Tiles of a sequence's keys; one where it has none, or where its tree is too large, which says so.
__device__ inline int tiles_of(const Seq& sq, int KT) {
    return sq.n > kTreeNodes ? 1 : max((sq.kv + KT - 1) / KT, 1);
}

// R rows a wave: 32 on the 32x32x16 instructions, 16 on the 16x16x32 ones.  A lane's
// row is its number modulo R, its part `c` the rest: 64 / R parts hold 8 values each
// of a slab of an operand, and quads of a result, keys or values QS q + 4 c + 0..3.
template <int R>
struct Shape;
template <>
struct Shape<32> {
    typedef f16 Acc;
    static constexpr int kSlab = 16, kQuads = 4, kStep = 8;  // an operand's depth; a result's quads, their step
    static __device__ inline f16 mfma(h8 a, h8 b, f16 c) { return mfma32(a, b, c); }
};
template <>
struct Shape<16> {
    typedef f4 Acc;
    static constexpr int kSlab = 32, kQuads = 1, kStep = 16;
    static __device__ inline f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <int R>
__device__ inline float max_parts(float x) { return R == 32 ? max_halves(x) : max_halves(max_rows16(x)); }
template <int R>
__device__ inline float sum_parts(float x) { return R == 32 ? sum_halves(x) : sum_halves(sum_rows16(x)); }

// A row's queries as they lie in memory: values kSlab s + 8 c + 0..7 for slab s, from
// element `at` on.
template <int D, int DT, int R>
struct RawQueries {
    static constexpr int kSlab = Shape<R>::kSlab, N = D / kSlab;
    u4 w[N][DT == kF32 ? 2 : 1];
    __device__ inline void load(const void* q, int64_t at) {
#pragma unroll
        for (int s = 0; s < N; ++s) {
            if constexpr (DT == kF32) {
                const u4* const p = reinterpret_cast<const u4*>(static_cast<const float*>(q) + at + kSlab * s);
                w[s][0] = p[0];
                w[s][1] = p[1];
            } else {  // rows are 8-byte aligned
                const u2* const p = reinterpret_cast<const u2*>(static_cast<const uint16_t*>(q) + at + kSlab * s);
                const u2 x = p[0], y = p[1];
                w[s][0] = (u4){x.x, x.y, y.x, y.y};
            }
        }
    }
    // As operands, scaled; returns what a score is worth in log2.
    __device__ inline float operands(float scale, h8* hi, h8* lo) const {
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == kF32) {
                    top = max(max(top, w[s][0][j] & 0x7FFFFFFFu), w[s][1][j] & 0x7FFFFFFFu);
                } else {
                    top = max(max(top, w[s][0][j] << 16 & 0x7FFF0000u), w[s][0][j] & 0x7FFF0000u);
                }
            }
        top = lane_max_u32(top, 32);
        if constexpr (R == 16) top = lane_max_u32(top, 16);
        if constexpr (DT == kF16) {  // halves order like their magnitudes
            const uint16_t bits = (uint16_t)(top >> 16);
            top = f_bits((float)__builtin_bit_cast(_Float16, bits));
        }
        const float up = row_scale(top);
#pragma unroll
        for (int s = 0; s < N; ++s) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == kF32) {
                    x[j] = bits_f(w[s][0][j]) * up;
                    x[4 + j] = bits_f(w[s][1][j]) * up;
                } else {
                    const uint32_t b = w[s][0][j];
                    const h2 h = __builtin_bit_cast(h2, b);
                    x[2 * j] = (DT == kBF16 ? bf_lo(b) : (float)h[0]) * up;
                    x[2 * j + 1] = (DT == kBF16 ? bf_hi(b) : (float)h[1]) * up;
                }
            }
            if constexpr (DT == kF32) split8(x, hi[s], lo[s]);
            else hi[s] = round8(x);
        }
        return score_worth(scale, up);
    }
};

// How a workgroup of W waves takes a unit of RT rows: R rows a wave, W / (RT / R) waves
// along the KT keys of a tile.
//
// Rows of 16: a wave's sums and queries are half as large, and up to three workgroups share
// a compute unit (per_unit), whose loads hide one another's waits.  Rows of 32 read a key from LDS half as
// often; they are for 128 rows of 64 and 128 values (32 nodes of 16 sequences, bf16: 51 us; 57 with
// 16 rows a wave, 70 with eight waves of 32).  Units of 64 rows were so once (10 nodes of
// 64 sequences, bf16: 207 us, 162 now).  With heads of 256 a wave's sums of 32 rows would
// leave no registers for a second wave.
template <int D, int RT>
struct Tiling {
    static constexpr int R = D == 256 || RT <= 64 ? 16 : 32, WR = RT / R;
    static constexpr int W = D == 256 && RT > 32 ? 8 : 4, WK = W / WR;
    static constexpr int KT = 64, KW = KT / WK;
    static constexpr int KS = D + 8, VS = D + (R == 32 ? 32 : 16);  // LDS rows of a key and of its values: reads of one instruction fall on unlike banks
    static_assert(KW >= 32, "a wave takes blocks of 32 keys");
};
// Workgroups a compute unit: three where the registers hold them, two of 128 rows or of fp32's
// 64, with heads of 256 two of 32 rows and one of 128.  Heads of 128, 64 rows: fp32 spills 28 registers a lane at three
// (10 nodes of 64 sequences 226 us, 198 at two), bf16 7 (162, 181).  32 rows: fp32 11
// (8 nodes of 64 sequences 175, 191 at two), bf16 2 (151, 173).
template <int D, int RT, int DT>
constexpr int per_unit() { return D == 256 ? RT > 32 ? 1 : 2 : RT > 64 || (DT == kF32 && RT > 32) ? 2 : 3; }

// The order of a stretch of code: `n` instructions of a kind next.  Left to itself the
// compiler reads each operand from LDS right before its matrix instruction, and
// every one waits out the read.
template <int KIND, int N>
__device__ __forceinline__ void next_are() {
    if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(KIND, N, 0);
}
constexpr int kValu = 2, kMatrix = 8, kLdsRead = 0x100;
// Keeps what a branch hardly ever does from being done, and left unused, every time.
__device__ __forceinline__ void stay_branch() { asm volatile(""); }

// Tiles a share at least: each share of a cut unit has its sums to write and to join.  12 nodes
// behind 4100 keys, heads of 256, fp32: 26.4 us; with one 27.4, three 28.2, four 31.5.
constexpr int kLeastTiles = 2;

// The share that this wave's workgroup has of all units' tiles: tiles [pos, end), the
// first in sequence b, whose first tile is `base`; `per` tiles a share.  Every wave
// sums up all sequences' tiles for itself, 256 a round.
struct Share {
    int64_t pos, end, per, base;
    int b;
    Seq sq;
};
template <int RT, int KT>
__device__ inline Share share_of(const TreeArgs& a, int id) {
    constexpr int N = 4;  // sequences a lane and round
    const int lane = threadIdx.x & 63;
    Seq s[N];
    int64_t n[N], upto, all;
    const auto round = [&](int b0) {
        int64_t mine = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] = sequence(a, min(b0 + N * lane + j, a.B - 1));
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int tiles = b0 + N * lane + j < a.B ? tiles_of(s[j], KT) : 0;
            n[j] = (int64_t)((uint32_t)(s[j].n * a.G + RT - 1) / RT * a.H) * tiles;
            mine += n[j];
        }
        upto = scan_wave(mine);
        all = lane_of(upto, 63);
        upto -= mine;  // before this lane's
    };
    Share w;
    int64_t total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64 * N) {
        round(b0);
        total += all;
    }
    w.per = max(over(total + a.grid - 1, a.grid), (int64_t)kLeastTiles);
    w.pos = id * w.per;
    w.end = min(w.pos + w.per, total);
    if (w.pos >= w.end) return w;
    int64_t before = 0;
    for (int b0 = 0;; b0 += 64 * N) {
        if (a.B > 64 * N) round(b0);
        upto += before;
        before += all;
        if (w.pos < before) {
            bool is = false;
            int64_t first = 0;
            int b = 0, q0 = 0, rows = 0, kv = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (w.pos >= upto && w.pos < upto + n[j]) {
                    is = true;
                    first = upto;
                    b = b0 + N * lane + j;
                    q0 = s[j].q0;
                    rows = s[j].n;
                    kv = s[j].kv;
                }
                upto += n[j];
            }
            const int who = __builtin_ctzll(__ballot(is));
            w.base = lane_of(first, who);
            w.b = __builtin_amdgcn_readlane(b, who);
            w.sq = {__builtin_amdgcn_readlane(q0, who), __builtin_amdgcn_readlane(rows, who), __builtin_amdgcn_readlane(kv, who)};
            return w;
        }
    }
}

template <int D, int KIND, int DT, int RT>
__global__ __launch_bounds__((64 * Tiling<D, RT>::W), (per_unit<D, RT, DT>() * Tiling<D, RT>::W / 4)) void tree_keys_kernel(TreeArgs a) {
    typedef Tiling<D, RT> T;
    constexpr bool SPLIT = DT == kF32, PSPLIT = DT != kBF16;  // two terms of the queries, and of the weights
    constexpr int R = T::R, W = T::W, WR = T::WR, WK = T::WK, KT = T::KT, KW = T::KW, KS = T::KS, VS = T::VS;
    constexpr int THREADS = 64 * W, U = KW / 32;    // blocks of 32 keys a wave
    constexpr int NC = KT * D / (16 * THREADS);     // 16-byte chunks a thread loads of a tile's keys (and of its values)
    constexpr int NG = KT / 16;                     // groups of 16 keys, each in one page
    constexpr int per_row = D / 16;
    constexpr int SL = D / Shape<R>::kSlab, NA = D / R, NQ = Shape<R>::kQuads, QS = Shape<R>::kStep;
    constexpr int J = R / 2;                        // scores a lane has of 32 keys
    constexpr int kBytes = std::max(KT * (KS + VS) * 2, (WK - 1) * RT * D * 4);
    typedef typename Shape<R>::Acc Acc;
    __shared__ __align__(16) uint8_t lds[kBytes];
    __shared__ __align__(16) float sks[KT], svs[KT];
    __shared__ float sm[W][R], sl[W][R], sf[W][R];
    __shared__ __align__(16) float smax[KT / 32];      // of each 32 keys' value scales
    __shared__ __align__(16) uint32_t svalid[KT / 32];  // the keys that are there, a bit each
    __shared__ int16_t up[kTreeNodes];
    _Float16 *const sk = reinterpret_cast<_Float16*>(lds), *const sv = sk + KT * KS;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & (R - 1), c = lane / R, rg = wave % WR, kg = wave / WR, r16 = lane & 15;
    // Neighbouring shares lie on one XCD each, whose cache has a unit's keys for its next rows.
    const int id = (blockIdx.x & 7) * (a.grid >> 3) + (blockIdx.x >> 3);
    Share w = share_of<RT, KT>(a, id);

    while (w.pos < w.end) {
        // A unit: rows of one key-value head; its tiles [t0, t1) are this share's.
        const Seq sq = w.sq;
        const int ntile = tiles_of(sq, KT), nrow = (uint32_t)(sq.n * a.G + RT - 1) / RT;
        const int its = (int)over(w.pos - w.base, ntile), h = its / nrow, first = (its - h * nrow) * RT;
        const int64_t began = w.base + (int64_t)its * ntile;
        const int t0 = (int)(w.pos - began), t1 = (int)min((int64_t)ntile, t0 + (w.end - w.pos));
        const bool whole = t0 == 0 && t1 == ntile, spoilt = sq.n > kTreeNodes;
        const int rows = min(sq.n * a.G, first + RT), row = first + R * rg + r;
        const bool has_row = row < rows;
        // Lanes past the rows repeat the unit's first: no other workgroup writes that one meanwhile,
        // where the output is q.
        const int like = has_row ? row : first, node = like / a.G, tok = sq.q0 + node, head = h * a.G + like % a.G;
        const int ctx = sq.kv - sq.n;  // place of node 0; below zero where the cache lacks the first nodes
        const int32_t* const table = a.table + w.b * a.table_row;
        int t = spoilt || sq.kv == 0 ? t0 - 1 : t1 - 1;

        // The pages of a tile's groups of 16 keys, one a lane, as the table has them: nothing
        // waits for them here.
        const auto pages_of = [&](int tile) {
            return table[min(max(KT * tile + 16 * (lane / (64 / NG)), 0), sq.kv - 1) >> a.pshift];
        };
        int pages = 0, pages_in = 0;  // of the tile that is loaded next, of the one in registers
        if (t >= t0) pages = pages_of(t);
        RawQueries<D, DT, R> raw;
        const bool wave_rows = first + R * rg < rows;
        raw.load(a.q, tok * a.q_token + head * a.q_head + 8 * c);

        // A lane's place in the 16 keys that a wave's pass begins with, the same in all passes.
        static_assert(THREADS / per_row % 16 == 0 && KT == 64, "passes of whole groups; a key a lane");
        const uint32_t own = (tid / per_row & 15) * D + 16 * (tid % per_row);
        u4 kraw[NC], vraw[NC];
        float ksc = 0.0f, vsc = 0.0f;
        bool sc_bad = true;
        const auto load = [&](int tile) {
            // -1 where the sequence has no key or the cache no such page.
            pages_in = KT * tile + 16 * (lane / (64 / NG)) < sq.kv && (uint32_t)pages < (uint32_t)a.P ? pages : -1;
            const auto row_of = [&](int page, int key) {  // cache row of a group's first key
                return (((int64_t)max(page, 0) * a.H + h) << a.pshift) + (key & ((1 << a.pshift) - 1));
            };
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int g = (wave * 64 + THREADS * i) / per_row >> 4;  // the wave's group of this pass
                const int64_t at = row_of(__builtin_amdgcn_readlane(pages_in, 64 / NG * g), KT * tile + 16 * g) * D;
                kraw[i] = *reinterpret_cast<const u4*>(a.kp + at + own);
                vraw[i] = *reinterpret_cast<const u4*>(a.vp + at + own);
            }
            if (wave < 3) {  // a key a lane: its key's scale, its value's, whether it is there
                sc_bad = pages_in < 0 || KT * tile + lane >= sq.kv;
                if (wave < 2) {
                    const int64_t at = row_of(pages_in, KT * tile + (lane & ~15)) + (lane & 15);
                    if (wave == 0) ksc = a.ks[at];
                    vsc = a.vs[at];
                }
            }
            pages = pages_of(tile - 1);
        };
        if (t >= t0) load(t);
        if (t0 == 0 && tid == 0) {
            const int slot = (a.cu ? (int)((int64_t)sq.q0 * a.G / RT) + w.b : w.b * nrow) + first / RT;
            a.shares[(int64_t)slot * a.H + h] = (i2){id, (int)over(began + ntile - 1, w.per)};
        }
        __syncthreads();  // the last unit's reads are over
        if (t1 * KT > ctx)
            for (int i = tid; i < min(sq.n, kTreeNodes); i += THREADS) {
                const int p = a.parents[sq.q0 + i];
                up[i] = (int16_t)(p >= 0 && p < i ? p : -1);
            }

        h8 qh[SL], ql[SPLIT ? SL : 1];
        const float rowf = raw.operands(a.scale, qh, ql);

        Acc o[NA];
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < 4 * NQ; ++j) o[i][j] = 0.0f;
        // A tile's weights are computed in units in which a probability of 1 is 2^9 / nu, at
        // most 2^119 of those eight, so that a lane's add up to less than fp32 holds.
        constexpr float least = 0x1p-110f;
        float m = -INFINITY, l = 0.0f, nu = least, peak = 0.0f, unit = __builtin_log2f(kPScale / least);
        int at_node = has_row ? node : -1;  // the next of the row's node and its ancestors

        // The tile in registers to LDS.
        const auto unpack = [&](int key0) {
            if (KIND == kFp8 && (key0 + KT > sq.kv || __any(pages_in < 0))) {  // bytes of rows that no key is in may be NaN
                stay_branch();
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    const int page = __builtin_amdgcn_readlane(pages_in, 64 / NG * ((wave * 64 + THREADS * i) / per_row >> 4));
                    if (page < 0 || key0 + (tid + THREADS * i) / per_row >= sq.kv) kraw[i] = vraw[i] = (u4){0, 0, 0, 0};
                }
            }
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int kr = (tid + THREADS * i) / per_row, col = 16 * (tid % per_row);
                const u4 kw = kraw[i], vw = vraw[i];
                h8* kd = reinterpret_cast<h8*>(sk + kr * KS + col);
                h8* vd = reinterpret_cast<h8*>(sv + kr * VS + col);
                // Eight lanes of sixteen write their second half first: all at once they fall on unlike
                // banks.  Rows of 128 values do not need it (keys), or lose less to the banks (values).
                const int one = D == 128 ? 0 : lane >> 3 & 1;
                kd[one] = unpack8<KIND>(one ? kw.z : kw.x, one ? kw.w : kw.y);
                kd[1 - one] = unpack8<KIND>(one ? kw.x : kw.z, one ? kw.y : kw.w);
                vd[one] = unpack8<KIND>(one ? vw.z : vw.x, one ? vw.w : vw.y);
                vd[1 - one] = unpack8<KIND>(one ? vw.x : vw.z, one ? vw.y : vw.w);
            }
            // A wave each for the keys' scales, the values' and what is there: all wait for the last.
            // A value scale of NaN goes with the key's, whose score a row that does
            // not see the key leaves out; times a probability of zero it would not.
            const bool nan = vsc != vsc;
            if (wave == 0) {
                sks[lane] = sc_bad ? 0.0f : nan ? vsc : ksc;
            } else if (wave == 1) {
                const float v = sc_bad || nan ? 0.0f : vsc;
                svs[lane] = v;
                const float vmax = max_rows16(max_16(v));  // of 32 keys
                if ((lane & 31) == 0) smax[lane >> 5] = vmax;
            } else if (wave == 2) {
                const uint64_t valid = __ballot(!sc_bad);
                if ((lane & 31) == 0) svalid[lane >> 5] = (uint32_t)(valid >> (lane & 32));
            }
        };
        for (; t >= t0; --t) {
            const int key0 = KT * t;
            __syncthreads();  // the last tile's reads are over
            unpack(key0);
            __syncthreads();
            if (t > t0) load(t - 1);
            if (!wave_rows) continue;

            // Scores: a lane's j-th of a block of 32 keys is key QS (j / 4) + 4 c + j % 4.
            constexpr int KB = KW / R, NK = SL * KB, TERMS = SPLIT ? 2 : 1;  // blocks of R keys, operands of K
            float x[U][J], vmax = 0.0f;
            uint32_t valid[U], every = ~0u;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                vmax = fmaxf(vmax, smax[U * kg + u]);
                valid[u] = svalid[U * kg + u];
                every &= valid[u];
            }
            {
                Acc s[KB];
                h8 k[NK];
#pragma unroll
                for (int n = 0; n < NK; ++n)
                    k[n] = *reinterpret_cast<const h8*>(sk + (KW * kg + R * (n % KB) + r) * KS + 8 * c + Shape<R>::kSlab * (n / KB));
                f4 sc[U * J / 4];
#pragma unroll
                for (int n = 0; n < U * J / 4; ++n)
                    sc[n] = *reinterpret_cast<const f4*>(sks + KW * kg + 32 * (n / (J / 4)) + QS * (n % (J / 4)) + 4 * c);
#pragma unroll
                for (int v = 0; v < KB; ++v)
#pragma unroll
                    for (int j = 0; j < 4 * NQ; ++j) s[v][j] = 0.0f;
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    s[n % KB] = Shape<R>::mfma(k[n], qh[n / KB], s[n % KB]);
                    if constexpr (SPLIT) s[n % KB] = Shape<R>::mfma(k[n], ql[n / KB], s[n % KB]);
                }
                // Times the key scales.
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < J; ++j) x[u][j] = s[(J * u + j) / (4 * NQ)][j % (4 * NQ)] * sc[(J * u + j) / 4][j % 4];
                constexpr int AHEAD = 6, NS = U * J / 4;
                next_are<kLdsRead, 2 + AHEAD>();
#pragma unroll
                for (int n = 0; n < NK - AHEAD; ++n) {
                    next_are<kMatrix, TERMS>();
                    next_are<kLdsRead, 1>();
                }
#pragma unroll
                for (int n = 0; n < AHEAD; ++n) {
                    next_are<kMatrix, TERMS>();
                    next_are<kLdsRead, (NS + AHEAD - 1) / AHEAD>();
                }
            }
            if (key0 + KT > ctx || __builtin_amdgcn_readfirstlane(every) != ~0u) {
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
                    bits &= has_row ? valid[u] : 0u;
                    bits >>= 4 * c;
#pragma unroll
                    for (int j = 0; j < J; j += 4) {
                        const f4 vs = *reinterpret_cast<const f4*>(svs + KW * kg + 32 * u + QS * (j / 4) + 4 * c);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool out = !(bits >> (QS * (j / 4) + e) & 1);
                            x[u][j + e] = out ? -INFINITY : x[u][j + e];
                            vmax = fmaxf(vmax, out ? 0.0f : vs[e]);
                        }
                    }
                }
                vmax = max_parts<R>(vmax);
            }
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < J; j += 2) top = fmaxf(fmaxf(top, x[u][j]), x[u][j + 1]);
            top = max_parts<R>(top);
            // The reference moves only once a row's scores pass it by kSlack, its units where the
            // values' size leaves their range.
            const bool moves = (top - m) * rowf > kSlack;
            const bool other = vmax > nu * 8.0f || (vmax > 0.0f && vmax <= nu * 0x1p-4f);
            if (__any(moves || other)) {
                float f = moves ? fast_exp2((m - top) * rowf) : 1.0f;
                m = moves ? top : m;
                l *= f;
                peak *= f;
                const float now = next_nu(nu, vmax, peak, least);
                f *= nu / now;
                unit = __builtin_log2f(kPScale / now);
                nu = now;
#pragma unroll
                for (int i = 0; i < NA; ++i) o[i] *= f;
            }
            peak = fmaxf(peak, nu);
            const float ref = m == -INFINITY ? 0.0f : m;
            float bias = __builtin_fmaf(-ref, rowf, unit);
            // m rowf is rounded once here, by less than half while it is below 2^22; past that
            // the difference is taken first, else the largest weight would be 2 to that error.
            if (__any(__builtin_fabsf(ref) * rowf > 0x1p22f)) {
                stay_branch();
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < J; ++j) x[u][j] -= ref;
                bias = unit;
            }
            __builtin_amdgcn_s_setprio(1);
            float sum = 0.0f;
            // Eight of a lane's scores make an operand of the weights, for a group of 512 / R keys.
            constexpr int GS = U * J / 8, NV = GS * NA;
#pragma unroll
            for (int g = 0; g < GS; ++g) {
                const int k0 = KW * kg + (512 / R) * g + 4 * c;  // of the first quad; the second QS on
                const f4 s0 = *reinterpret_cast<const f4*>(svs + k0), s1 = *reinterpret_cast<const f4*>(svs + k0 + QS);
                const _Float16* p = sv + (k0 + (r16 >> 2)) * VS + 16 * (r >> 4) + 4 * (r16 & 3);
                h8 v[NA];
#pragma unroll
                for (int i = 0; i < NA; ++i) v[i] = mx::join(read_tr(p + R * i), read_tr(p + R * i + QS * VS));
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    y[j] = fast_exp2(__builtin_fmaf(x[8 * g / J][8 * g % J + j], rowf, bias));
                    sum += y[j];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] *= s0[j];
                    y[4 + j] *= s1[j];
                }
                h8 ph, pl;
                if constexpr (PSPLIT) split8(y, ph, pl);
                else ph = round8(y);
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    o[i] = Shape<R>::mfma(v[i], ph, o[i]);
                    if constexpr (PSPLIT) o[i] = Shape<R>::mfma(v[i], pl, o[i]);
                }
            }
            {
                // The values' operands some instructions ahead; a group's weights beside the matrix
                // instructions of the one before.
                constexpr int AHEAD = 4, VALU = PSPLIT ? 60 : 40, PT = PSPLIT ? 2 : 1;
                next_are<kLdsRead, 2 * AHEAD + 2>();
                next_are<kValu, VALU>();
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    next_are<kMatrix, PT>();
                    next_are<kLdsRead, 2>();
                    next_are<kValu, (VALU + NA - 1) / NA>();
                }
            }
            __builtin_amdgcn_s_setprio(0);
            l = __builtin_fmaf(sum, nu * (1.0f / kPScale), l);
        }

        l = sum_parts<R>(l);
        float f = nu * (1.0f / kPScale), mlog = m * rowf;
        if constexpr (WK > 1) {
            // The groups' sums, joined in their order.
            __syncthreads();
            f4* const so = reinterpret_cast<f4*>(lds);
            if (c == 0) {
                sm[wave][r] = mlog;
                sl[wave][r] = l;
                sf[wave][r] = f;
            }
            if (kg > 0) {
                f4* const mine = so + ((kg - 1) * WR + rg) * NA * NQ * 64 + lane;
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        mine[64 * (i * NQ + q)] = (f4){o[i][4 * q], o[i][4 * q + 1], o[i][4 * q + 2], o[i][4 * q + 3]};
            }
            __syncthreads();
            float top = mlog;
#pragma unroll
            for (int g = 1; g < WK; ++g) top = fmaxf(top, sm[g * WR + rg][r]);
            const float safe = top == -INFINITY ? 0.0f : top;
            const float f0 = fast_exp2(mlog - safe);
            l *= f0;
            f *= f0;
            if (kg == 0) {
#pragma unroll
                for (int i = 0; i < NA; ++i) o[i] *= f;
#pragma unroll
                for (int g = 1; g < WK; ++g) {
                    const float e = fast_exp2(sm[g * WR + rg][r] - safe), by = e * sf[g * WR + rg][r];
                    l += e * sl[g * WR + rg][r];
                    const f4* const from = so + ((g - 1) * WR + rg) * NA * NQ * 64 + lane;
#pragma unroll
                    for (int i = 0; i < NA; ++i)
#pragma unroll
                        for (int q = 0; q < NQ; ++q) {
                            const f4 v = from[64 * (i * NQ + q)] * by;
#pragma unroll
                            for (int e4 = 0; e4 < 4; ++e4) o[i][4 * q + e4] += v[e4];
                        }
                }
            }
            f = 1.0f;
            mlog = top;
        }
        if (wave_rows && kg == 0) {
            if (!whole) {
                // A share's first unit may have begun in an earlier one; its last may go on.  A part is kept
                // in the lanes' order, 1 KB an instruction.
                const int64_t part = 2 * id + (t0 == 0);
                if (c == 0) a.ml[part * RT + R * rg + r] = (f2){mlog, l};
                f4* const to = reinterpret_cast<f4*>(a.part + part * RT * D) + rg * NA * NQ * 64 + lane;
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        to[64 * (i * NQ + q)] = (f4){o[i][4 * q] * f, o[i][4 * q + 1] * f, o[i][4 * q + 2] * f, o[i][4 * q + 3] * f};
            } else if (has_row) {
                f *= spoilt ? __builtin_nanf("") : l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        put4<DT>(a.out, tok * a.o_token + head * a.o_head + R * i + 8 * q + 4 * c,
                                 (f4){o[i][4 * q] * f, o[i][4 * q + 1] * f, o[i][4 * q + 2] * f, o[i][4 * q + 3] * f});
            }
        }
        w.pos += t1 - t0;
        if (w.pos < w.end && w.pos >= w.base + (int64_t)nrow * a.H * ntile) {  // on to the next sequence that has rows
            w.base = w.pos;
            do {
                w.sq = sequence(a, ++w.b);
            } while (w.sq.n == 0);
        }
    }
}

// The RT rows of a slot: their sequence (-1: none) and the first of them.  Sequence b's
// units take the slots from cu[b] * G / RT + b on, which leaves room for all
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

// The parts of a unit that was cut joined, in their order.  A wave takes QN quads of
// the values of R rows, each of which a part has in 1 KB; where there are few units,
// one quad, and the four waves of a workgroup a quarter of its parts each.
template <int D, int DT, int RT, bool FEW>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a) {
    typedef Tiling<D, RT> T;
    constexpr int R = T::R, NQ = Shape<R>::kQuads, N = D / R * NQ, NG = FEW ? 4 : 1, QN = FEW ? 1 : 2;
    __shared__ __align__(16) f4 sv[FEW ? 192 : 1];
    __shared__ float ssum[FEW ? 192 : 1], stop[FEW ? 256 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & (R - 1), c = lane / R, slot = blockIdx.x / a.H, h = blockIdx.x - slot * a.H;
    const int item = (FEW ? blockIdx.y : 4 * blockIdx.y + wave) * QN, rg = item / N, quad = item % N;
    Seq sq;
    int first;
    if (rows_of_slot<RT>(a, slot, sq, first) < 0) return;
    const i2 share = a.shares[blockIdx.x];
    const int rows = sq.n * a.G, row = first + R * rg + r;
    if (share[1] <= share[0] || first + R * rg >= rows) return;
    const auto part_of = [&](int s) { return (int64_t)(2 * s + (s == share[0])); };
    float top = -INFINITY, sum = 0.0f;
    f4 v[QN];
#pragma unroll
    for (int i = 0; i < QN; ++i) v[i] = (f4){0, 0, 0, 0};
    constexpr int AT = 8;  // parts whose reads are on their way at once
    for (int s0 = share[0] + (FEW ? wave : 0); s0 <= share[1]; s0 += AT * NG) {
        f2 x[AT];
        f4 y[AT][QN];
#pragma unroll
        for (int j = 0; j < AT; ++j) {
            const int s = s0 + j * NG;
            x[j] = (f2){-INFINITY, 0.0f};
#pragma unroll
            for (int i = 0; i < QN; ++i) y[j][i] = (f4){0, 0, 0, 0};
            if (s > share[1]) continue;
            const int64_t part = part_of(s);
            x[j] = a.ml[part * RT + R * rg + r];
#pragma unroll
            for (int i = 0; i < QN; ++i)
                y[j][i] = reinterpret_cast<const f4*>(a.part + part * RT * D)[(rg * N + quad + i) * 64 + lane];
        }
        float now = top;
#pragma unroll
        for (int j = 0; j < AT; ++j) now = fmaxf(now, x[j].x);
        const float safe = now == -INFINITY ? 0.0f : now, old = fast_exp2(top - safe);
        top = now;
        sum *= old;
#pragma unroll
        for (int i = 0; i < QN; ++i) v[i] *= old;
#pragma unroll
        for (int j = 0; j < AT; ++j) {
            const float f = fast_exp2(x[j].x - safe);  // a part that saw nothing: zeros times 0
            sum += f * x[j].y;
#pragma unroll
            for (int i = 0; i < QN; ++i) v[i] += y[j][i] * f;
        }
    }
    if constexpr (FEW) {  // the four waves' parts relative to one maximum
        stop[threadIdx.x] = top;
        __syncthreads();
        float all = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) all = fmaxf(all, stop[64 * i + lane]);
        const float f = fast_exp2(top - (all == -INFINITY ? 0.0f : all));
        sum *= f;
        v[0] *= f;
    }
    if constexpr (FEW) {
        if (wave > 0) {
            sv[threadIdx.x - 64] = v[0];
            ssum[threadIdx.x - 64] = sum;
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            v[0] += sv[64 * i + lane];
            sum += ssum[64 * i + lane];
        }
    }
    if (row >= rows) return;
    const float f = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    const int tok = sq.q0 + row / a.G, head = h * a.G + row % a.G;
#pragma unroll
    for (int i = 0; i < QN; ++i)
        put4<DT>(a.out, tok * a.o_token + head * a.o_head + R * ((quad + i) / NQ) + 8 * ((quad + i) % NQ) + 4 * c, v[i] * f);
}

// ------------------------------------------------------------------ host

struct Plan {
    int rt, nslots, grid;
    int64_t join;              // workgroups of the join, 0: nothing is cut
    size_t ml, shares, bytes;  // offsets of the maxima and of the shares, and the whole
};

// The join's grid.  At one tile a sequence there is none.  12 nodes behind 4100 keys (4 units): 26.4 us, 29.6 by
// the other; 10 nodes of 16 sequences (128): 34, 35.
constexpr int kFewUnits = 32;
template <int D, int RT>
dim3 join_grid(int64_t units, int64_t capacity) {
    constexpr unsigned items = RT * D / 256;  // quads of a wave's rows
    static_assert(items % 8 == 0, "a workgroup of the join takes eight");
    if (capacity <= Tiling<D, RT>::KT) return dim3(0, 0);
    return dim3((unsigned)units, units <= kFewUnits ? items : items / 8);
}

// A share for each place on the units, fewer where the table has fewer tiles.
template <int D, int RT>
Plan plan_rows(int T, int B, int H, int G, int dt, bool cu, int64_t capacity, int n_cu) {
    typedef Tiling<D, RT> L;
    Plan p{};
    p.rt = RT;
    p.nslots = (int)(cu ? (int64_t)T * G / RT + B : (int64_t)B * ((G + RT - 1) / RT));
    const dim3 join = join_grid<D, RT>((int64_t)p.nslots * H, capacity);
    p.join = (int64_t)join.x * join.y;
    const int64_t tiles = (int64_t)p.nslots * H * std::max<int64_t>(1, (capacity + L::KT - 1) / L::KT);
    const int64_t room = (int64_t)n_cu * (dt == kF32 ? per_unit<D, RT, kF32>() : per_unit<D, RT, kBF16>());
    p.grid = (int)((std::min(room, (tiles + kLeastTiles - 1) / kLeastTiles) + 7) / 8 * 8);
    p.ml = (size_t)p.grid * 2 * RT * D * 4;
    p.shares = p.ml + (size_t)p.grid * 2 * RT * 8;
    p.bytes = p.shares + (size_t)p.nslots * H * 8;
    return p;
}

// Rows a unit by the mean tree: the fewest that hold it, as what a unit lacks of rows is worked out
// all the same, and a tree of two units has its keys loaded and unpacked twice.  us with one step
// more and one less: 32 rows (8 nodes of 64 sequences, heads of 128, bf16) 151, 195 by units of
// 64; 64 rows (16 of 16) 43, 43 by 128; 40 rows (10 of 64) 162, 215 by 128, 235 by 32; 128 rows (32 of 16) 52, 61 by 64.
// Heads of 256 have no units of 64: 48 rows (8 of 64) 202 by 128, 218 by 64, 241 by 32.
template <int D>
Plan plan_tree(int T, int B, int H, int G, int dt, bool cu, int64_t capacity, int n_cu) {
    const int64_t mean = (((int64_t)T + B - 1) / B) * G;
    if (mean <= 32) return plan_rows<D, 32>(T, B, H, G, dt, cu, capacity, n_cu);
    if constexpr (D < 256) {
        if (mean <= 64) return plan_rows<D, 64>(T, B, H, G, dt, cu, capacity, n_cu);
    }
    return plan_rows<D, 128>(T, B, H, G, dt, cu, capacity, n_cu);
}

Plan plan_of(int T, int B, int heads, int H, int D, int dt, bool cu, int64_t capacity, int n_cu) {
    const int G = heads / H;
    return D == 64    ? plan_tree<64>(T, B, H, G, dt, cu, capacity, n_cu)
           : D == 128 ? plan_tree<128>(T, B, H, G, dt, cu, capacity, n_cu)
                      : plan_tree<256>(T, B, H, G, dt, cu, capacity, n_cu);
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

template <int D, int KIND, int DT, int RT>
void launch4(const TreeArgs& a, hipStream_t st) {
    typedef Tiling<D, RT> L;
    tree_keys_kernel<D, KIND, DT, RT><<<(unsigned)a.grid, 64 * L::W, 0, st>>>(a);
    const dim3 join = join_grid<D, RT>((int64_t)a.nslots * a.H, (int64_t)a.table_w << a.pshift);
    if (join.x == 0) return;
    if (join.x <= kFewUnits) tree_join_kernel<D, DT, RT, true><<<join, 256, 0, st>>>(a);
    else tree_join_kernel<D, DT, RT, false><<<join, 256, 0, st>>>(a);
}

template <int D, int KIND, int DT>
void launch3(const TreeArgs& a, const Plan& p, hipStream_t st) {
    if constexpr (D < 256) {
        if (p.rt == 64) return launch4<D, KIND, DT, 64>(a, st);
    }
    if (p.rt == 32) launch4<D, KIND, DT, 32>(a, st);
    else launch4<D, KIND, DT, 128>(a, st);
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
    // Rows and units are counted in 32 bits.
    if ((int64_t)T * heads > (1 << 24) || (int64_t)B * c->kv_heads > (1 << 20)) {
        bq_set_error("tree_attention: %d nodes of %d heads in %d sequences are too much for one call", T, heads, B);
        return false;
    }
    *pshift = s;
    return true;
}

// A launch has fewer than 2^24 workgroups.  The join's are the most, up to 16 a unit.
bool check_launch(const Plan& p, int T, int B, int heads) {
    if (p.join < (1 << 24)) return true;
    bq_set_error("tree_attention: %d nodes of %d heads in %d sequences are too much for one call (%lld workgroups)", T, heads,
                 B, (long long)p.join);
    return false;
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
    const Plan p = plan_of(T, B, heads, kv_heads, head_dim, dtype, has_cu != 0, (int64_t)table_w << ps, cu_count());
    return check_launch(p, T, B, heads) ? (int64_t)p.bytes : -2;
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
    a.H = cache->kv_heads;
    a.G = heads / cache->kv_heads;
    a.P = cache->num_pages;
    a.pshift = ps;
    a.scale = scale * kLog2e;
    const Plan p = plan_of(T, B, heads, a.H, cache->head_dim, dtype, dCu != nullptr, (int64_t)table_w << ps, cu_count());
    if (!check_launch(p, T, B, heads)) return -2;
    if (p.bytes > 0 && (!dWork || work_bytes < (int64_t)p.bytes)) {
        bq_set_error("tree_attention: needs a workspace of %zu bytes, got %lld", p.bytes, (long long)work_bytes);
        return -4;
    }
    a.nslots = p.nslots;
    a.grid = p.grid;
    a.part = static_cast<float*>(dWork);
    a.ml = reinterpret_cast<f2*>(static_cast<uint8_t*>(dWork) + p.ml);
    a.shares = reinterpret_cast<i2*>(static_cast<uint8_t*>(dWork) + p.shares);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (cache->head_dim == 64) launch1<64>(a, p, cache->kind, dtype, st);
    else if (cache->head_dim == 128) launch1<128>(a, p, cache->kind, dtype, st);
    else launch1<256>(a, p, cache->kind, dtype, st);
    return launched("tree_attention") ? 0 : -5;
}

}  // extern "C"
