// Drafted tokens against the target's scores: down each sequence's tree with given
// random numbers, and the next token drawn.
//
// At node v, with p = softmax(logits[v] / temperature) and the drafted children
// c_1, c_2, .. of v in order, the chance of what is left is R = G / S with G = p
// and S = 1 at first.  Child c is taken where
//   u_c q(c) / Q < G(c) / S;
// else G(c) becomes zero and, where the draft's probabilities q are given,
//   A += S / Q,   G = max(p - A q, 0) but for the rejected,   Q -= q(c),   S = sum G.
// That is the rejection rule's residual max(R - q / Q, 0) / sum, sibling by sibling:
// every step takes a multiple of the same q off, so p and one number A are all it
// needs.  Without q a child is the draft's whole chance (q(c) / Q = 1) and only the
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
// vector work of the same time.  verify_walk_kernel goes down, one workgroup a
// sequence, from what the pieces hold; to draw it reads one piece again.  The first
// residual of each sequence, a pass over the row that stands alone on its path, is
// spread over all units (verify_rest_kernel), between the two halves of the walk.
#include "mix_common.h"

#include <algorithm>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

constexpr int kPiece = 2048, kPieces = 1024;  // scores a piece; pieces of a row at most
constexpr int kTreeNodes = 1024;
constexpr int kWalk = 256;                    // threads of a walk; of one with residuals
constexpr int kWalkDraft = 1024;

struct Piece {
    double sum;
    float top;  // NaN: a NaN or +infinity among them
    int at;
};

// Where a walk stands before its first residual.
struct Walk {
    double A, Q, top, one;
    int node, m, child, going;
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
    const float* temps; // null: `temp` for all
    float temp;
    int32_t* out;
    int32_t* path;
    int32_t* counts;
    Piece* pieces;  // [T][np]
    Walk* walks;    // [B], with a draft
    double* rest;   // [B][np], with a draft
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

// A lane's scores of a piece: load v holds scores (64 v + lane) * VEC on.  Rows
// lie at any address of their type's alignment.  Past the row's end: -infinity.
template <int DT>
__device__ inline void load_piece(const void* logits, int64_t row, int V, int piece, int lane, float* x) {
    constexpr int N = vec<DT>(), L = kPiece / 64 / N;
#pragma unroll
    for (int v = 0; v < L; ++v) {
        const int i = piece * kPiece + (64 * v + lane) * N;
        if (i + N <= V) {
            const u4a w = *reinterpret_cast<const u4a*>(static_cast<const uint8_t*>(logits) + (row + i) * (DT == kF32 ? 4 : 2));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (DT == kF32) {
                    x[N * v + j] = bits_f(w[j]);
                } else {
                    const uint32_t b = w[j];  // bit_cast of a vector's element itself would take its first
                    const h2 h = __builtin_bit_cast(h2, b);
                    x[N * v + 2 * j] = DT == kBF16 ? bf_lo(w[j]) : (float)h[0];
                    x[N * v + 2 * j + 1] = DT == kBF16 ? bf_hi(w[j]) : (float)h[1];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[N * v + j] = i + j < V ? score<DT>(logits, row + i + j) : -INFINITY;
        }
    }
}

__device__ inline double sum_wave(double x) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) x += __shfl_xor(x, s);
    return x;
}
__device__ inline int min_wave(int x) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) x = min(x, __shfl_xor(x, s));
    return x;
}

// exp((x - top) / temperature); zero for -infinity.
__device__ inline double weight(float x, double top, double inv) { return exp(((double)x - top) * inv); }

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
    int b = t;
    if (a.cu) {
        int hi = a.B;
        b = 0;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (a.cu[mid] <= t) b = mid;
            else hi = mid;
        }
    }
    const float temp = temperature(a, b);
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
            const double inv = 1.0 / (double)temp;
#pragma unroll
            for (int i = 0; i < E; ++i) sum += weight(x[i], top, inv);
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
    double top, inv, one, A;  // one: 1 / the sum of exponentials
};

template <int DT, bool DRAFT>
__device__ inline double share(const VerArgs& a, const Row& r, float x, const float* q) {
    const double p = weight(x, r.top, r.inv) * r.one;
    if (!DRAFT || r.A == 0.0) return p;
    const double d = p - r.A * (double)*q;
    return d > 0.0 ? d : d * 0.0;  // a draft's NaN or infinity shows
}

// A lane's weights of a piece of node t's row without the tokens in `gone`
// (a bit each; null: none), in load_piece's order.
template <int DT, bool DRAFT>
__device__ inline void weights_of(const VerArgs& a, const Row& r, int t, int piece, int lane, const uint32_t* gone,
                                  double* g) {
    constexpr int N = vec<DT>(), E = kPiece / 64;
    float x[E];
    load_piece<DT>(a.logits, t * a.row, a.V, piece, lane, x);
    const float* const q = DRAFT ? a.draft + t * a.draft_row : nullptr;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int in = (64 * (i / N) + lane) * N + i % N, at = piece * kPiece + in;
        const bool is = at < a.V && !(gone && (gone[in >> 5] >> (in & 31) & 1));
        g[i] = is ? share<DT, DRAFT>(a, r, x[i], DRAFT ? q + at : nullptr) : 0.0;
    }
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
    const Row r = {w.top, 1.0 / (double)temperature(a, b), w.one, w.A};
    double g[kPiece / 64], sum = 0.0;
    weights_of<DT, true>(a, r, s.q0 + w.node, piece, lane, gone[wave], g);
#pragma unroll
    for (int i = 0; i < kPiece / 64; ++i) sum += g[i];
    sum = sum_wave(sum);
    if (lane == 0) a.rest[(int64_t)b * a.np + piece] = sum;
}

template <int DT, bool DRAFT, bool RESUME, int THREADS>
__global__ __launch_bounds__(THREADS) void verify_walk_kernel(VerArgs a) {
    constexpr int W = THREADS / 64, N = vec<DT>(), E = kPiece / 64;
    __shared__ int parents[kTreeNodes], removed[kTreeNodes];
    __shared__ double mass[kPieces];  // G's sums of the node's pieces
    __shared__ double sums[W];
    __shared__ float tops[W];
    __shared__ int ats[W], bads[W];
    __shared__ uint32_t gone[W][kPiece / 32];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Seq s = sequence(a, b);
    Walk k = {0.0, 1.0, 0.0, 1.0, 0, 1, 0, 0};
    if constexpr (RESUME) {
        k = a.walks[b];
        if (!k.going) return;
    } else {
        // Rows outside every sequence, and what this one's walk leaves: -1.
        const int from = b == 0 ? 0 : s.q0, to = b == a.B - 1 ? a.T : s.q0 + s.n;
        for (int i = from + tid; i < to; i += THREADS) a.out[i] = a.path[i] = -1;
        if (DRAFT && tid == 0) a.walks[b].going = 0;
        if (s.n == 0 || s.n > kTreeNodes) {
            if (tid == 0) a.counts[b] = 0;
            return;
        }
    }
    for (int i = tid; i < s.n; i += THREADS) parents[i] = a.parents ? a.parents[s.q0 + i] : -1;
    __syncthreads();
    if (!RESUME && tid == 0) a.path[s.q0] = 0;
    const float temp = temperature(a, b);
    const bool greedy = temp == 0.0f;
    const double inv = 1.0 / (double)temp;

    int node = k.node, m = k.m, cursor = k.node, nremoved = 0, best = -1;
    double S = 1.0, Q = 1.0, base = 1.0;
    Row r = {0.0, inv, 1.0, 0.0};
    bool fresh = true, bad = !(temp >= 0.0f) || temp > 3e38f;

    const auto block_sum = [&](double x) {
        x = sum_wave(x);
        __syncthreads();
        if (lane == 0) sums[wave] = x;
        __syncthreads();
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < W; ++w) all += sums[w];
        return all;
    };
    const auto mass_sum = [&] {
        double x = 0.0;
        __syncthreads();
        for (int i = tid; i < a.np; i += THREADS) x += mass[i];
        return block_sum(x);
    };
    // The bits of the removed tokens in a piece.
    const auto mark = [&](int piece) {
        gone[wave][lane] = 0;
        __builtin_amdgcn_wave_barrier();
        for (int i = lane; i < nremoved; i += 64) {
            const int in = removed[i] - piece * kPiece;
            if (in >= 0 && in < kPiece) atomicOr(&gone[wave][in >> 5], 1u << (in & 31));
        }
        __builtin_amdgcn_wave_barrier();
    };
    const auto piece_mass = [&](int piece) {
        double g[E], x = 0.0;
        mark(piece);
        weights_of<DT, DRAFT>(a, r, s.q0 + node, piece, lane, gone[wave], g);
#pragma unroll
        for (int i = 0; i < E; ++i) x += g[i];
        x = sum_wave(x);
        if (lane == 0) mass[piece] = x;
    };
    // The sums of the pieces that removed tokens are in, without them.
    const auto remove = [&] {
        __syncthreads();
        for (int i = wave; i < nremoved; i += W) piece_mass(removed[i] / kPiece);
        return mass_sum();
    };

    if constexpr (RESUME) {
        cursor = k.child;
        r = {k.top, inv, k.one, k.A};
        Q = k.Q;
        for (int i = tid; i < a.np; i += THREADS) mass[i] = a.rest[(int64_t)b * a.np + i];
        if (tid == 0) removed[0] = a.tokens[s.q0 + k.child];
        const int gone0 = a.tokens[s.q0 + k.child];
        nremoved = gone0 >= 0 && gone0 < a.V;
        __syncthreads();
        S = base = mass_sum();
        fresh = false;
    }
    for (;;) {
        if (fresh) {
            // The node's own probabilities.
            const Piece* const own = a.pieces + (int64_t)(s.q0 + node) * a.np;
            float top = -INFINITY;
            int at = INT32_MAX;
            bool nan = false;
            for (int i = tid; i < a.np; i += THREADS) {
                const Piece p = own[i];
                nan |= p.top != p.top;
                if (p.top > top) {  // pieces come in order: the first of equal ones stays
                    top = p.top;
                    at = p.at;
                }
            }
            const float wave_top = max_wave(top);
            at = min_wave(top == wave_top ? at : INT32_MAX);
            nan = __any(nan);
            __syncthreads();
            if (lane == 0) {
                tops[wave] = wave_top;
                ats[wave] = at;
                bads[wave] = nan;
            }
            __syncthreads();
            top = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                top = fmaxf(top, tops[w]);
                bad |= bads[w] != 0;
            }
            best = INT32_MAX;
#pragma unroll
            for (int w = 0; w < W; ++w) best = tops[w] == top ? min(best, ats[w]) : best;
            bad |= !(top > -INFINITY);
            if (bad) break;
            r = {(double)top, inv, 1.0, 0.0};
            nremoved = 0;
            if (!greedy) {
                double z = 0.0;
                for (int i = tid; i < a.np; i += THREADS) {
                    const Piece p = own[i];
                    mass[i] = p.top > -INFINITY ? p.sum * weight(p.top, r.top, inv) : 0.0;
                    z += mass[i];
                }
                r.one = 1.0 / block_sum(z);
                for (int i = tid; i < a.np; i += THREADS) mass[i] *= r.one;
                S = Q = base = 1.0;
            }
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
        const int token = a.tokens[s.q0 + child];
        const bool real = token >= 0 && token < a.V;
        bool take = false;
        if (greedy) {
            take = token == best;
        } else {
            // A token that no vocabulary has, or an earlier sibling had, is passed over, and
            // so is one that the draft's probabilities have nothing left for.
            bool there = real && Q > 0.0;
            for (int i = 0; i < nremoved && there; ++i) there = removed[i] != token;
            if (there) {
                const int64_t t = s.q0 + node;
                const float x = score<DT>(a.logits, t * a.row + token), q = DRAFT ? a.draft[t * a.draft_row + token] : 1.0f;
                const double g = share<DT, DRAFT>(a, r, x, &q);
                take = (double)a.uniforms[s.q0 + child] * (DRAFT ? (double)q / Q : 1.0) * S < g;
                if (!take) {
                    if (tid == 0) removed[nremoved] = token;
                    ++nremoved;
                    __syncthreads();
                    if constexpr (!DRAFT) {
                        S -= g;
                        if (S < base * 0x1p-10) S = base = remove();  // the difference has lost its last bits
                    } else {
                        r.A += S / Q;
                        Q -= (double)q;
                        if constexpr (!RESUME) {
                            if (tid == 0) {
                                a.walks[b] = Walk{r.A, Q, r.top, r.one, node, m, child, 1};
                                a.counts[b] = m;
                            }
                            return;
                        } else {
                            for (int i = wave; i < a.np; i += W) piece_mass(i);
                            S = mass_sum();
                        }
                    }
                }
            }
        }
        if (take) {
            if (tid == 0) {
                a.out[s.q0 + m - 1] = token;
                a.path[s.q0 + m] = child;
            }
            node = child;
            ++m;
            fresh = true;
        }
    }
    if (tid == 0) a.counts[b] = m;
    if (bad || greedy) {
        if (tid == 0) a.out[s.q0 + m - 1] = bad ? -1 : best;
        return;
    }
    if (!DRAFT && nremoved > 0) remove();
    __syncthreads();
    if (wave > 0) return;
    // The piece that the running sum passes the random number in: each lane takes
    // consecutive ones.
    const int per = (a.np + 63) / 64, first = lane * per, last = min(first + per, a.np);
    double x = 0.0;
    for (int i = first; i < last; ++i) x += mass[i];
    double until = x;
#pragma unroll
    for (int st = 1; st < 64; st *= 2) {
        const double y = __shfl_up(until, st);
        if (lane >= st) until += y;
    }
    const double total = __shfl(until, 63), goal = (double)a.uniforms[s.q0] * total;
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
    piece = __shfl(piece, who);
    before = __shfl(before, who);
    mark(piece);
    double g[E];
    weights_of<DT, DRAFT>(a, r, s.q0 + node, piece, lane, gone[0], g);
    int drawn = INT32_MAX, final = -1;  // and the last token that has any weight
#pragma unroll
    for (int v = 0; v < E / N; ++v) {
        double own = 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j) own += g[N * v + j];
        double upto = own;
#pragma unroll
        for (int st = 1; st < 64; st *= 2) {
            const double y = __shfl_up(upto, st);
            if (lane >= st) upto += y;
        }
        double run = before + (upto - own);
        before += __shfl(upto, 63);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = piece * kPiece + (64 * v + lane) * N + j;
            run += g[N * v + j];
            if (g[N * v + j] > 0.0) {
                if (run > goal) drawn = min(drawn, at);
                final = at;
            }
        }
    }
    drawn = min_wave(drawn);
    final = -min_wave(-final);
    if (lane == 0) a.out[s.q0 + m - 1] = drawn < INT32_MAX ? drawn : final;
}

template <int DT>
void launch(const VerArgs& a, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.np + 3) / 4);
    if (a.T > 0) verify_rows_kernel<DT><<<(unsigned)a.T * blocks, 256, 0, st>>>(a);
    if (!a.draft) {
        verify_walk_kernel<DT, false, false, kWalk><<<a.B, kWalk, 0, st>>>(a);
        return;
    }
    verify_walk_kernel<DT, true, false, kWalk><<<a.B, kWalk, 0, st>>>(a);
    verify_rest_kernel<DT><<<(unsigned)a.B * blocks, 256, 0, st>>>(a);
    verify_walk_kernel<DT, true, true, kWalkDraft><<<a.B, kWalkDraft, 0, st>>>(a);
}

bool check(int T, int V, int B, bool has_cu) {
    const int64_t np = ((int64_t)V + kPiece - 1) / kPiece;
    if (T < 0 || B < 0 || V < 1 || V > kPiece * kPieces || (!has_cu && T != B) || T * np > (1 << 23) ||
        B * np > (1 << 23)) {
        bq_set_error("verify: needs 1 to 2^21 scores a row, one node a sequence where no offsets are given, and no more "
                     "than 2^23 pieces of 2048 scores (got %d rows of %d, %d sequences)",
                     T, V, B);
        return false;
    }
    return true;
}

int64_t sizes(int T, int V, int B, bool draft, int64_t* walks, int64_t* rest) {
    const int64_t np = (V + kPiece - 1) / kPiece;
    *walks = T * np * (int64_t)sizeof(Piece);
    *rest = *walks + (draft ? B * (int64_t)sizeof(Walk) : 0);
    return *rest + (draft ? B * np * 8 : 0);
}

}  // namespace

extern "C" {

int64_t i4_verify_workspace(int T, int V, int B, int has_cu, int has_draft) {
    if (!check(T, V, B, has_cu != 0)) return -2;
    int64_t walks, rest;
    return sizes(T, V, B, has_draft != 0, &walks, &rest);
}

int i4_verify_dev(const void* dLogits, int64_t row, int T, int V, int dtype, const int32_t* dTokens,
                  const int32_t* dParents, const float* dUniforms, const int32_t* dCu, int B, const float* dTemps,
                  float temperature, const float* dDraft, int64_t draft_row, int32_t* dOut, int32_t* dPath,
                  int32_t* dCounts, void* dWork, int64_t work_bytes, void* stream) {
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
    int64_t walks, rest;
    const int64_t need = sizes(T, V, B, dDraft != nullptr, &walks, &rest);
    if (need > 0 && (!dWork || work_bytes < need)) {
        bq_set_error("verify: needs a workspace of %lld bytes, got %lld", (long long)need, (long long)work_bytes);
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
    a.temps = dTemps;
    a.temp = temperature;
    a.out = dOut;
    a.path = dPath;
    a.counts = dCounts;
    a.pieces = static_cast<Piece*>(dWork);
    a.walks = reinterpret_cast<Walk*>(static_cast<uint8_t*>(dWork) + walks);
    a.rest = reinterpret_cast<double*>(static_cast<uint8_t*>(dWork) + rest);
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

}  // extern "C"
