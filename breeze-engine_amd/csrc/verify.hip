// Drafted tokens against the target's scores: down each sequence's tree with given
// random numbers, and the next token drawn.
//
// At node v, with p = softmax(logits[v] / temperature) and the drafted children
// c_1, c_2, .. of v in order, the chance of what is left is R = G / S with G = p
// and S = 1 at first.  Child c is taken where
//   u_c q(c) / Q < G(c) / S;
// else G(c) becomes zero and, where the draft's probabilities q are given,
//   A += S / Q,   G = max(p - A q, 0),   S = sum G,   Q = sum q,   but for the rejected.
// That is the rejection rule's residual max(R - q / Q, 0) / sum, sibling by sibling:
// every step takes a multiple of the same q off, so p and one number A are all it
// needs.  Q, 1 at first, is summed up along with G: 1 less the rejected tokens' q would be
// what fp32 left of the row's sum, where the draft gave them nearly everything (1 - 10^-7 to
// one token: 19% off).  Without q a child is the draft's whole chance (q(c) / Q = 1) and only the
// rejected ones leave.  Where no child is taken, or there is none, the first token
// whose running sum of G passes u_0 S is drawn.  Then every token is distributed as
// the target's own.
//
// A random number may fall next to a border between two tokens, of which a
// vocabulary has 10^5: weights and sums are fp64, so that it falls on the wrong
// side with a chance near 10^-10.
//
// verify_rows_kernel takes one pass over all rows, for each of their pieces of 2048
// scores the largest and the sum of exponentials relative to it: HBM, and fp64
// vector work of nearly the same time, which is what half types take.  verify_walk_kernel goes down, one workgroup a
// sequence: first what every node's pieces add up to, a node a wave, and every child's
// score, then the walk itself in LDS; to draw it reads one piece again.  The first
// residual of each sequence, a pass over the row that stands alone on its path, is
// spread over all units (verify_rest_kernel), between the two halves of the walk; any
// further one of a tree is its workgroup's alone.
//
// 640 nodes over 151936 tokens, fp32: rows 87 to 97 us (389 MB, 4.0 to 4.5 TB/s; a sum of a
// GiB reads 4.0), bf16 92; walk of 16 sequences of 40 nodes 18; 12 nodes: 5.7 and 12.  A walk is latency:
// five dependent reads of memory, a fp64 exponential and sum over a node's pieces, a few
// LDS reads a child.  24 sequences of 3 to 9 nodes over 32003 tokens with a draft, bf16: rows 9,
// walk 12, residual 9, walk 12, each a launch.  16 trees of 32 nodes, four children a node, over
// 151936 tokens with a draft, fp32: 143 the whole call (paths of 4), 167 where the draft is farther off
// and more siblings are rejected; 95 without the draft.
#include "mix_common.h"

#include <algorithm>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

constexpr int kPiece = 2048, kPieces = 1024;  // scores a piece; pieces of a row at most
constexpr int kTreeNodes = 1024;
constexpr int kWalk = 512;                    // threads of a walk; 1024 spill 18 to 126 registers a lane (52 us where a draft's call takes 43.5)

struct Piece {
    double sum;
    float top;  // NaN: a NaN or +infinity among them
    int at;
};

// Where a walk stands before its first residual.
struct Walk {
    double A, top, one;
    int node, m, child, going;
};

// G, and the draft's q, of the tokens that are left, summed up.
struct Left {
    double g, q;
};

struct VerArgs {
    const void* logits;
    int64_t row;  // element strides of a row
    const float* draft;
    int64_t draft_row;
    const int32_t* tokens;
    const int32_t* parents;
    const float* uniforms;
    const int32_t* cu;  // null: one node a sequence
    const int32_t* kv_lens;  // null: all sequences take part
    const float* temps; // null: `temp` for all
    float temp;
    int32_t* out;
    int32_t* path;
    int32_t* counts;
    Piece* pieces;  // [T][np]
    f2* own;        // [T]: each node's own score, and the draft's probability, at its parent
    Walk* walks;    // [B], with a draft
    Left* rest;     // [B][np], with a draft
    int T, V, B, np;
};

typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(2)));

template <int DT>
constexpr int vec() { return DT == kF32 ? 4 : 8; }

template <int DT>
__device__ inline float score(const void* p, int64_t i) {
    if constexpr (DT == kF32) return static_cast<const float*>(p)[i];
    const uint16_t w = static_cast<const uint16_t*>(p)[i];
    return DT == kBF16 ? bf_lo(w) : (float)__builtin_bit_cast(_Float16, w);
}

// A lane's scores of a piece, N at a time: the v-th are scores (64 v + lane) * N on.  Rows
// lie at any address of their type's alignment.  Past the row's end: -infinity.
template <int DT, int N = vec<DT>()>
__device__ inline void load_piece(const void* logits, int64_t row, int V, int piece, int lane, float* x) {
    constexpr int L = kPiece / 64 / N, PER = vec<DT>();  // of 16 bytes
#pragma unroll
    for (int v = 0; v < L; ++v)
#pragma unroll
        for (int k = 0; k < N; k += PER) {
            const int i = piece * kPiece + (64 * v + lane) * N + k;
            if (i + PER <= V) {
                const u4a w =
                    *reinterpret_cast<const u4a*>(static_cast<const uint8_t*>(logits) + (row + i) * (DT == kF32 ? 4 : 2));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t b = w[j];  // bit_cast of a vector's element itself would take its first
                    if constexpr (DT == kF32) {
                        x[N * v + k + j] = bits_f(b);
                    } else {
                        const h2 h = __builtin_bit_cast(h2, b);
                        x[N * v + k + 2 * j] = DT == kBF16 ? bf_lo(b) : (float)h[0];
                        x[N * v + k + 2 * j + 1] = DT == kBF16 ? bf_hi(b) : (float)h[1];
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < PER; ++j) x[N * v + k + j] = i + j < V ? score<DT>(logits, row + i + j) : -INFINITY;
            }
        }
}

// A lane's value as DPP control CONTROL moves it, 0 where nothing comes.
template <int CONTROL, int ROWS>
__device__ inline double moved(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CONTROL, ROWS, 0xF, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CONTROL, ROWS, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}
// The sum over a wave's lanes up to this one.
__device__ inline double scan_wave(double x) {
    x += moved<0x111, 0xF>(x);  // row_shr:1, 2, 4, 8 within 16 lanes
    x += moved<0x112, 0xF>(x);
    x += moved<0x114, 0xF>(x);
    x += moved<0x118, 0xF>(x);
    x += moved<0x142, 0xA>(x);  // row_bcast:15 to rows 1 and 3
    x += moved<0x143, 0xC>(x);  // row_bcast:31 to rows 2 and 3
    return x;
}
__device__ inline double of_lane(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline double sum_wave(double x) { return of_lane(scan_wave(x), 63); }
__device__ inline int min_wave(int x) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) x = min(x, __shfl_xor(x, s));
    return x;
}

// exp((x - top) / temperature) with scale = log2(e) / temperature: 2^t, t = (x - top)
// scale, at most 0, as 2^n times 2^r with n the nearest whole number and |r| at most a
// half, whose Taylor series in r ln(2) is taken up to the eleventh power (7e-15 is left
// out).  -infinity gives zero, and so does all that is below fp64's range.  Two thirds of
// a general exponential's instructions.
__device__ inline double weight(float x, double top, double scale) {
    const double t = __builtin_fmax(((double)x - top) * scale, -1080.0), n = __builtin_rint(t), r = t - n;
    double p = 4.4455382718708115e-10;  // ln(2)^11 / 11!, and so on down
    p = __builtin_fma(p, r, 7.0549116208011233e-9);
    p = __builtin_fma(p, r, 1.0178086009239699e-7);
    p = __builtin_fma(p, r, 1.3215486790144309e-6);
    p = __builtin_fma(p, r, 1.5252733804059840e-5);
    p = __builtin_fma(p, r, 1.5403530393381609e-4);
    p = __builtin_fma(p, r, 1.3333558146428443e-3);
    p = __builtin_fma(p, r, 9.6181291076284772e-3);
    p = __builtin_fma(p, r, 5.5504108664821580e-2);
    p = __builtin_fma(p, r, 2.4022650695910071e-1);
    p = __builtin_fma(p, r, 6.9314718055994531e-1);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// What the wave's lanes wrote to LDS is there for all of them.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
constexpr double kLog2e64 = 1.4426950408889634;

struct Seq {
    int q0, n;
};
__device__ inline Seq sequence(const VerArgs& a, int b) {
    if (!a.cu) return {b, 1};
    const int q0 = min(max(a.cu[b], 0), a.T);
    return {q0, min(max(a.cu[b + 1], q0), a.T) - q0};
}
__device__ inline float temperature(const VerArgs& a, int b) { return a.temps ? a.temps[b] : a.temp; }

template <int DT>
__global__ __launch_bounds__(256) void verify_rows_kernel(VerArgs a) {
    constexpr int N = vec<DT>(), E = kPiece / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (a.np + 3) / 4, t = blockIdx.x / blocks, piece = (blockIdx.x - t * blocks) * 4 + wave;
    if (piece >= a.np) return;
    float x[E];
    load_piece<DT>(a.logits, t * a.row, a.V, piece, lane, x);
    const int b = a.cu ? last_of(a.B, [&](int i) { return a.cu[i] <= t; }) : t;
    const float temp = temperature(a, b);
    if (piece == 0 && lane == 0 && a.parents) {  // what the walk will ask of this node, while the scores are read anyway
        const int q0 = a.cu ? min(max(a.cu[b], 0), a.T) : t, up = a.parents[t], token = a.tokens[t];
        if (up >= 0 && up < t - q0 && token >= 0 && token < a.V)
            a.own[t] = (f2){score<DT>(a.logits, (q0 + up) * a.row + token),
                            a.draft ? a.draft[(q0 + up) * a.draft_row + token] : 1.0f};
    }
    float top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        top = fmaxf(top, x[i]);
        bad |= !(x[i] < INFINITY);
    }
    top = max_wave(top);
    bad = __any(bad);
    int at = INT32_MAX;
    double sum = 0.0;
    if (temp > 0.0f) {
        if (top > -INFINITY) {
            const double scale = kLog2e64 / (double)temp;
#pragma unroll
            for (int i = 0; i < E; ++i) sum += weight(x[i], top, scale);
        }
        sum = sum_wave(sum);
    } else {
#pragma unroll
        for (int i = E - 1; i >= 0; --i)
            if (x[i] == top) at = piece * kPiece + (64 * (i / N) + lane) * N + i % N;
        at = min_wave(at);
    }
    if (lane == 0) a.pieces[(int64_t)t * a.np + piece] = Piece{sum, bad ? __builtin_nanf("") : top, at};
}

// One row's weights: G of a node.
struct Row {
    double top, scale, one, A;  // one: 1 / the sum of exponentials
};

// G of a token of score x that the draft gives q.
template <bool DRAFT>
__device__ inline double share(const Row& r, float x, float q) {
    const double p = weight(x, r.top, r.scale) * r.one;
    if (!DRAFT || r.A == 0.0) return p;
    const double d = p - r.A * (double)q;
    return d > 0.0 ? d : d * 0.0;  // a draft's NaN or infinity shows
}

// A lane's weights of a piece of node t's row without the tokens in `gone` (a bit each):
// f(v, g, q) with those of scores (64 v + lane) * N on, for one v after another, and the
// draft's q, where it has taken a part off the row.
template <int DT, bool DRAFT, typename F>
__device__ inline void weights_of(const VerArgs& a, const Row& r, int t, int piece, int lane, const uint32_t* gone, F f) {
    constexpr int N = vec<DT>(), E = kPiece / 64;
    float x[E], q[DRAFT ? E : 1];
    load_piece<DT>(a.logits, t * a.row, a.V, piece, lane, x);
    if (DRAFT && r.A != 0.0) load_piece<kF32, N>(a.draft, t * a.draft_row, a.V, piece, lane, q);
#pragma unroll
    for (int v = 0; v < E / N; ++v) {
        double g[N], left[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int in = (64 * v + lane) * N + j, at = piece * kPiece + in;
            const bool is = at < a.V && !(gone[in >> 5] >> (in & 31) & 1);
            g[j] = is ? share<DRAFT>(r, x[N * v + j], DRAFT ? q[N * v + j] : 0.0f) : 0.0;
            left[j] = is && DRAFT ? (double)q[N * v + j] : 0.0;
        }
        f(v, g, left);
    }
}
// Their sums over the piece.
template <int DT, bool DRAFT>
__device__ inline Left left_of(const VerArgs& a, const Row& r, int t, int piece, int lane, const uint32_t* gone) {
    Left sum = {0.0, 0.0};
    weights_of<DT, DRAFT>(a, r, t, piece, lane, gone, [&](int, const double* g, const double* q) {
#pragma unroll
        for (int j = 0; j < vec<DT>(); ++j) {
            sum.g += g[j];
            if constexpr (DRAFT) sum.q += q[j];
        }
    });
    sum.g = sum_wave(sum.g);
    if constexpr (DRAFT) sum.q = sum_wave(sum.q);
    return sum;
}

// The sequences whose walk stands before its first residual, all pieces.
template <int DT>
__global__ __launch_bounds__(256) void verify_rest_kernel(VerArgs a) {
    __shared__ uint32_t gone[4][kPiece / 32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (a.np + 3) / 4, b = blockIdx.x / blocks, piece = (blockIdx.x - b * blocks) * 4 + wave;
    const Walk w = a.walks[b];
    if (!w.going) return;
    const Seq s = sequence(a, b);
    const int token = a.tokens[s.q0 + w.child], in = token - piece * kPiece;
    gone[wave][lane] = in >= 0 && in < kPiece && in >> 5 == lane ? 1u << (in & 31) : 0;
    __syncthreads();
    if (piece >= a.np) return;
    const Row r = {w.top, kLog2e64 / (double)temperature(a, b), w.one, w.A};
    const Left sum = left_of<DT, true>(a, r, s.q0 + w.node, piece, lane, gone[wave]);
    if (lane == 0) a.rest[(int64_t)b * a.np + piece] = sum;
}

// What a node's pieces add up to.
struct Node {
    double one;  // 1 / the sum of exponentials
    float top;   // NaN: no distribution
    int best;    // the largest score's token, at temperature 0
};

template <int DT, bool DRAFT, bool RESUME>
__global__ __launch_bounds__(kWalk) void verify_walk_kernel(VerArgs a) {
    constexpr int W = kWalk / 64, N = vec<DT>(), AT = 2;
    struct Child {
        int token;
        float u, score, q;  // its random number; its score, and the draft's probability, at its parent
    };
    __shared__ Node nodes[kTreeNodes];
    __shared__ Child children[kTreeNodes];
    __shared__ int parents[kTreeNodes], removed[kTreeNodes];
    __shared__ double removed_g[DRAFT ? 1 : kTreeNodes];  // what each had
    __shared__ double full[DRAFT ? 1 : kPieces];          // the pieces' sums with them
    __shared__ double mass[kPieces], sums[W];             // G's sums of the node's pieces
    __shared__ double draft_left[RESUME ? kPieces : 1];   // and q's
    __shared__ uint32_t gone[W][kPiece / 32];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Seq s = sequence(a, b);
    const float temp = temperature(a, b);
    Walk k = {0.0, 0.0, 1.0, 0, 1, 0, 0};
    if constexpr (RESUME) {
        k = a.walks[b];
        if (!k.going) return;
    } else {
        // Rows outside every sequence, and what this one's walk leaves: -1.
        const int from = b == 0 ? 0 : s.q0, to = b == a.B - 1 ? a.T : s.q0 + s.n;
        for (int i = from + tid; i < to; i += kWalk) a.out[i] = a.path[i] = -1;
        if (DRAFT && tid == 0) a.walks[b].going = 0;
        if (s.n == 0 || s.n > kTreeNodes || (a.kv_lens && a.kv_lens[b] < 0)) {
            if (tid == 0) a.counts[b] = 0;
            return;
        }
    }
    const bool greedy = temp == 0.0f, cold = !(temp >= 0.0f && temp < INFINITY);
    const double scale = kLog2e64 / (double)temp;
    for (int i = tid; i < s.n; i += kWalk) {
        const int up = a.parents ? a.parents[s.q0 + i] : -1;
        const f2 own = a.own[s.q0 + i];  // not a number where there is no parent: not read then
        parents[i] = up >= 0 && up < i ? up : -1;
        children[i] = Child{a.tokens[s.q0 + i], a.uniforms[s.q0 + i], own.x, own.y};
    }
    for (int i0 = wave * AT; i0 < s.n; i0 += W * AT) {  // AT nodes' first 128 pieces are on their way at once
        Piece p[AT][2];
#pragma unroll
        for (int n = 0; n < AT; ++n) {
            const Piece* const own = a.pieces + (int64_t)(s.q0 + min(i0 + n, s.n - 1)) * a.np;
#pragma unroll
            for (int j = 0; j < 2; ++j) p[n][j] = own[min(lane + 64 * j, a.np - 1)];
        }
#pragma unroll
        for (int n = 0; n < AT; ++n) {
            const int i = i0 + n;
            if (i >= s.n) continue;
            const Piece* const own = a.pieces + (int64_t)(s.q0 + i) * a.np;
            float top = -INFINITY;
            bool nan = false;
            const auto look = [&](const Piece& q) {
                top = fmaxf(top, q.top);
                nan |= q.top != q.top;
            };
            look(p[n][0]);
            look(p[n][1]);
            for (int j = lane + 128; j < a.np; j += 64) look(own[j]);
            top = max_wave(top);
            nan = cold || __any(nan) || !(top > -INFINITY);
            int best = INT32_MAX;
            double z = 0.0;
            const auto add = [&](const Piece& q) {
                if (greedy) best = q.top == top ? min(best, q.at) : best;
                else if (q.top > -INFINITY) z += q.sum * weight(q.top, top, scale);
            };
            if (!nan) {
                if (lane < a.np) add(p[n][0]);
                if (lane + 64 < a.np) add(p[n][1]);
                for (int j = lane + 128; j < a.np; j += 64) add(own[j]);
                if (greedy) best = min_wave(best);
                else z = sum_wave(z);
            }
            if (lane == 0) nodes[i] = Node{1.0 / z, nan ? __builtin_nanf("") : top, best};
        }
    }
    __syncthreads();
    // The walk is one wave's, but for residuals, which all take part in.
    constexpr int STEP = RESUME ? kWalk : 64;
    if (!RESUME && wave > 0) return;
    const auto sync = [] {
        if constexpr (RESUME) __syncthreads();
        else wave_sync();
    };
    if (!RESUME && lane == 0) a.path[s.q0] = 0;

    int node = k.node, m = k.m, cursor = k.node, nremoved = 0;
    double S = 1.0, Q = 1.0, base = 1.0;
    Row r = {0.0, scale, 1.0, 0.0};
    Node at = {1.0, 0.0f, 0};
    bool fresh = true, bad = false;

    // Over all pieces.
    const auto sum_of = [&](const double* of) {
        double x = 0.0;
        sync();
        for (int i = tid; i < a.np; i += STEP) x += of[i];
        x = sum_wave(x);
        if constexpr (RESUME) {
            __syncthreads();
            if (lane == 0) sums[wave] = x;
            __syncthreads();
            x = 0.0;
#pragma unroll
            for (int w = 0; w < W; ++w) x += sums[w];
        }
        return x;
    };
    // The bits of the removed tokens in a piece.
    const auto mark = [&](int piece) {
        gone[wave][lane] = 0;
        wave_sync();
        for (int i = lane; i < nremoved; i += 64) {
            const int in = removed[i] - piece * kPiece;
            if (in >= 0 && in < kPiece) atomicOr(&gone[wave][in >> 5], 1u << (in & 31));
        }
        wave_sync();
    };
    const auto piece_mass = [&](int piece) {
        mark(piece);
        const Left x = left_of<DT, DRAFT>(a, r, s.q0 + node, piece, lane, gone[wave]);
        if (lane == 0) {
            mass[piece] = x.g;
            if constexpr (RESUME) draft_left[piece] = x.q;
        }
    };
    // All pieces' masses at a node without a draft's part.  The removed tokens' shares are
    // taken off their piece's; where they leave less than 2^-10 of all that it had, however
    // many steps it took, the difference has lost its last bits, and the piece is summed up
    // anew.
    const auto masses = [&] {
        const Piece* const own = a.pieces + (int64_t)(s.q0 + node) * a.np;
        sync();
        for (int i = tid; i < a.np; i += STEP) {
            const Piece p = own[i];
            mass[i] = p.top > -INFINITY ? p.sum * weight(p.top, r.top, scale) * r.one : 0.0;
            if constexpr (!DRAFT) full[i] = mass[i];
        }
        sync();
        if constexpr (!DRAFT) {
            for (int i = 0; i < nremoved; ++i) {
                const int piece = removed[i] / kPiece;
                const double was = mass[piece], now = was - removed_g[i];
                sync();
                if (lane == 0 && was >= 0.0) mass[piece] = now < full[piece] * 0x1p-10 ? -1.0 : now;
                sync();
            }
            for (int i = 0; i < nremoved; ++i) {
                const int piece = removed[i] / kPiece;
                if (mass[piece] < 0.0) piece_mass(piece);
                sync();
            }
        }
    };

    if constexpr (RESUME) {
        cursor = k.child;
        r = {k.top, scale, k.one, k.A};
        for (int i = tid; i < a.np; i += STEP) {
            const Left x = a.rest[(int64_t)b * a.np + i];
            mass[i] = x.g;
            draft_left[i] = x.q;
        }
        if (tid == 0) removed[0] = children[k.child].token;
        nremoved = 1;
        S = sum_of(mass);
        Q = sum_of(draft_left);
        fresh = false;
    }
    for (;;) {  // every wave alike
        if (fresh) {
            at = nodes[node];
            bad = at.top != at.top;
            if (bad) break;
            r = {(double)at.top, scale, at.one, 0.0};
            nremoved = 0;
            S = Q = base = 1.0;
            cursor = node;
            fresh = false;
        }
        // The next child.
        int child = -1;
        for (int i = cursor + 1; i < s.n; i += 64) {
            const uint64_t hit = __ballot(i + lane < s.n && parents[min(i + lane, s.n - 1)] == node);
            if (hit) {
                child = i + __builtin_ctzll(hit);
                break;
            }
        }
        if (child < 0) break;
        cursor = child;
        const Child c = children[child];
        bool take = false;
        if (greedy) {
            take = c.token == at.best;
        } else {
            // A token that no vocabulary has, or an earlier sibling had, is passed over, and
            // so is one that the draft's probabilities have nothing left for.
            bool there = c.token >= 0 && c.token < a.V && Q > 0.0;
            for (int i = 0; i < nremoved && there; ++i) there = removed[i] != c.token;
            // A draft that gave the child no probability: nothing says what chance it had.
            bad = DRAFT && there && !(c.q >= 0.0f && c.q < INFINITY);
            if (bad) break;
            if (there) {
                const double g = share<DRAFT>(r, c.score, c.q);
                take = (double)c.u * (DRAFT ? (double)c.q / Q : 1.0) * S < g;
                if (!take) {
                    sync();
                    if (tid == 0) {
                        removed[nremoved] = c.token;
                        if constexpr (!DRAFT) removed_g[nremoved] = g;
                    }
                    ++nremoved;
                    sync();
                    if constexpr (!DRAFT) {
                        S -= g;
                        if (S < base * 0x1p-10) {
                            masses();
                            S = base = sum_of(mass);
                        }
                    } else {
                        r.A += S / Q;
                        if constexpr (!RESUME) {
                            if (lane == 0) {
                                a.walks[b] = Walk{r.A, r.top, r.one, node, m, child, 1};
                                a.counts[b] = m;
                            }
                            return;
                        } else {
                            for (int i = wave; i < a.np; i += W) piece_mass(i);
                            S = sum_of(mass);
                            Q = sum_of(draft_left);
                        }
                    }
                }
            }
        }
        if (take) {
            if (tid == 0) {
                a.out[s.q0 + m - 1] = c.token;
                a.path[s.q0 + m] = child;
            }
            node = child;
            ++m;
            fresh = true;
        }
    }
    if (tid == 0) a.counts[b] = m;
    if (bad || greedy) {
        if (tid == 0) a.out[s.q0 + m - 1] = bad ? -1 : at.best;
        return;
    }
    if (r.A == 0.0) masses();
    sync();
    if (wave > 0) return;
    // The piece that the running sum passes the random number in: each lane takes
    // consecutive ones.
    const int per = (a.np + 63) / 64, first = lane * per, last = min(first + per, a.np);
    double x = 0.0;
    for (int i = first; i < last; ++i) x += mass[i];
    const double until = scan_wave(x), total = of_lane(until, 63), goal = (double)children[0].u * total;
    double before = __shfl_up(until, 1);
    if (lane == 0) before = 0.0;
    int piece = -1;
    for (int i = first; i < last && piece < 0; ++i) {
        if (before + mass[i] > goal) piece = i;
        else before += mass[i];
    }
    const uint64_t has = __ballot(piece >= 0);
    if (!has || !(total > 0.0)) {
        if (lane == 0) a.out[s.q0 + m - 1] = -1;  // nothing is left, or not a number
        return;
    }
    const int who = __builtin_ctzll(has);
    piece = __builtin_amdgcn_readlane(piece, who);
    before = of_lane(before, who);
    mark(piece);
    int drawn = INT32_MAX, final = -1;  // and the last token that has any weight
    weights_of<DT, DRAFT>(a, r, s.q0 + node, piece, lane, gone[0], [&](int v, const double* g, const double*) {
        double own = 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j) own += g[j];
        const double upto = scan_wave(own);
        double run = before + (upto - own);
        before += of_lane(upto, 63);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = piece * kPiece + (64 * v + lane) * N + j;
            run += g[j];
            if (g[j] > 0.0) {
                if (run > goal) drawn = min(drawn, at);
                final = at;
            }
        }
    });
    drawn = min_wave(drawn);
    final = -min_wave(-final);
    if (lane == 0) a.out[s.q0 + m - 1] = drawn < INT32_MAX ? drawn : final;
}

template <int DT>
void launch(const VerArgs& a, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.np + 3) / 4);
    if (a.T > 0) verify_rows_kernel<DT><<<(unsigned)a.T * blocks, 256, 0, st>>>(a);
    if (!a.draft) {
        verify_walk_kernel<DT, false, false><<<a.B, kWalk, 0, st>>>(a);
        return;
    }
    verify_walk_kernel<DT, true, false><<<a.B, kWalk, 0, st>>>(a);
    verify_rest_kernel<DT><<<(unsigned)a.B * blocks, 256, 0, st>>>(a);
    verify_walk_kernel<DT, true, true><<<a.B, kWalk, 0, st>>>(a);
}

// A launch has fewer than 2^32 threads in a dimension: 64 a piece of a row, 512 a sequence.
bool check(int T, int V, int B, bool has_cu) {
    const int64_t np = ((int64_t)V + kPiece - 1) / kPiece;
    if (T < 0 || B < 0 || V < 1 || V > kPiece * kPieces || (!has_cu && T != B) || T * np > (1 << 23) ||
        B * np > (1 << 22)) {
        bq_set_error("verify: needs 1 to 2^21 scores a row, one node a sequence where no offsets are given, and no more "
                     "than 2^23 pieces of 2048 scores, half of them of sequences (got %d rows of %d, %d sequences)",
                     T, V, B);
        return false;
    }
    return true;
}

// The workspace's parts: where those after the pieces begin, and its end.
struct Parts {
    int64_t own, walks, rest, end;
};
Parts parts_of(int T, int V, int B, bool draft) {
    const int64_t np = (V + kPiece - 1) / kPiece;
    Parts p;
    p.own = T * np * (int64_t)sizeof(Piece);
    p.walks = p.own + T * (int64_t)sizeof(f2);
    p.rest = p.walks + (draft ? B * (int64_t)sizeof(Walk) : 0);
    p.end = p.rest + (draft ? B * np * (int64_t)sizeof(Left) : 0);
    return p;
}

}  // namespace

extern "C" {

int64_t i4_verify_workspace(int T, int V, int B, int has_cu, int has_draft) {
    if (!check(T, V, B, has_cu != 0)) return -2;
    return parts_of(T, V, B, has_draft != 0).end;
}

int i4_verify_lens_dev(const void* dLogits, int64_t row, int T, int V, int dtype, const int32_t* dTokens,
                       const int32_t* dParents, const float* dUniforms, const int32_t* dCu, int B,
                       const int32_t* dKvLens, const float* dTemps, float temperature, const float* dDraft,
                       int64_t draft_row, int32_t* dOut, int32_t* dPath, int32_t* dCounts, void* dWork,
                       int64_t work_bytes, void* stream) {
    if (!check(T, V, B, dCu != nullptr)) return -2;
    if (dtype < kF32 || dtype > kF16 || (!dTemps && !(temperature >= 0.0f && temperature < 1e30f))) {
        bq_set_error("verify: needs a type of 0 to 2 and a temperature of zero or more (got %d, %g)", dtype, temperature);
        return -2;
    }
    if (B == 0) return 0;
    if (!dCounts || (T > 0 && (!dLogits || !dTokens || !dUniforms || !dOut || !dPath))) {
        bq_set_error("verify: null device pointer");
        return -2;
    }
    VerArgs a{};
    const Parts at = parts_of(T, V, B, dDraft != nullptr);
    if (at.end > 0 && (!dWork || work_bytes < at.end)) {
        bq_set_error("verify: needs a workspace of %lld bytes, got %lld", (long long)at.end, (long long)work_bytes);
        return -4;
    }
    a.logits = dLogits;
    a.row = row;
    a.draft = dDraft;
    a.draft_row = draft_row;
    a.tokens = dTokens;
    a.parents = dParents;
    a.uniforms = dUniforms;
    a.cu = dCu;
    a.kv_lens = dKvLens;
    a.temps = dTemps;
    a.temp = temperature;
    a.out = dOut;
    a.path = dPath;
    a.counts = dCounts;
    a.pieces = static_cast<Piece*>(dWork);
    a.own = reinterpret_cast<f2*>(static_cast<uint8_t*>(dWork) + at.own);
    a.walks = reinterpret_cast<Walk*>(static_cast<uint8_t*>(dWork) + at.walks);
    a.rest = reinterpret_cast<Left*>(static_cast<uint8_t*>(dWork) + at.rest);
    a.T = T;
    a.V = V;
    a.B = B;
    a.np = (V + kPiece - 1) / kPiece;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    if (dtype == kF32) launch<kF32>(a, st);
    else if (dtype == kBF16) launch<kBF16>(a, st);
    else launch<kF16>(a, st);
    return launched("verify") ? 0 : -5;
}

int i4_verify_dev(const void* dLogits, int64_t row, int T, int V, int dtype, const int32_t* dTokens,
                  const int32_t* dParents, const float* dUniforms, const int32_t* dCu, int B, const float* dTemps,
                  float temperature, const float* dDraft, int64_t draft_row, int32_t* dOut, int32_t* dPath,
                  int32_t* dCounts, void* dWork, int64_t work_bytes, void* stream) {
    return i4_verify_lens_dev(dLogits, row, T, V, dtype, dTokens, dParents, dUniforms, dCu, B, nullptr, dTemps,
                              temperature, dDraft, draft_row, dOut, dPath, dCounts, dWork, work_bytes, stream);
}

}  // extern "C"
