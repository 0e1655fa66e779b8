// A batch's page table on the GPU: pages of a free stack given to sequences that
// grow, and taken back from those that shrink; new tokens' slots, positions and
// lengths.
//
// extend: sequence b has n_b new tokens behind len_b and needs
//   need_b = max(ceil((len_b + n_b) / page) - held_b, 0)
// pages more.  With N_b = need_0 + .. + need_b, its j-th new page is
// free[count - 1 - (N_b - need_b + j)], where N_b <= count; else it, and every
// later one that needs a page, gets none.  trim is the inverse: the k-th page
// given back (sequences in order, each one's columns in order) of R goes to
// free[count + R - 1 - k], so that pages given back at once come out again as
// they were.
//
// Whole numbers throughout, each worked out by one thread in a fixed order: no
// atomics.  The prefix sums take one workgroup, bound by the latency of four
// dependent reads; slots of many tokens are a second launch over all units.  64
// sequences of 16 tokens: extend 5.5 us on the GPU, trim 3.9 (both calls with the host's
// part 15); 13642 tokens of 7 prompts: 4.3, 3.3 for the slots, 4.2.
#include "mix_common.h"

#include <algorithm>

#include "../../include/breeze_qmm.h"

using namespace mx;

namespace {

constexpr int kScan = 1024;      // threads of the workgroup that sums
constexpr int kTreeNodes = 1024; // of a tree of drafted tokens

struct PageArgs {
    int32_t* table;
    int32_t* held;
    int32_t* free;
    int32_t* count;
    const int32_t* lens;
    const int32_t* cu;       // null: one token a sequence
    const int32_t* parents;  // null: chains
    int32_t* slots;
    int32_t* positions;
    int32_t* kv_lens;
    int T, B, cols, P, pshift;
};

struct New {
    int q0, n;  // first new token, and how many
};
__device__ inline New new_tokens(const PageArgs& a, int b) {
    if (!a.cu) return {b, 1};
    const int q0 = min(max(a.cu[b], 0), a.T);
    return {q0, min(max(a.cu[b + 1], q0), a.T) - q0};
}

// The sum over threads up to this one, `total` that over all.
template <typename I>
__device__ inline I scan_block(I x, I* lds, I& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const I y = __shfl_up(x, s);
        if (lane >= s) x += y;
    }
    __syncthreads();  // the last call's reads
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    I before = 0;
    total = 0;
    for (int w = 0; w < kScan / 64; ++w) {
        before += w < wave ? lds[w] : 0;
        total += lds[w];
    }
    return x + before;
}

// The thread that the k-th of all threads' items is; until: each one's last, plus one.
__device__ inline int owner(const int* until, int k) {
    int lo = 0, hi = kScan - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (until[mid] > k) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// A node's depth in its tree; up(i) gives node i's parent, if it comes before.
template <typename F>
__device__ inline int depth_of(int node, F up) {
    int depth = 0;
    for (;;) {
        const int p = up(node);
        if (p < 0 || p >= node) return depth;
        node = p;
        ++depth;
    }
}
// The slot of a sequence's place.
__device__ inline int slot_of(const PageArgs& a, int b, int place) {
    const int page = a.table[(int64_t)b * a.cols + (place >> a.pshift)];
    return page >= 0 && page < a.P ? (page << a.pshift) + (place & ((1 << a.pshift) - 1)) : -1;
}

// Tokens up to which the workgroup that sums places them too, and sequences: their
// offsets, lengths and parents are in LDS then, where a token finds its sequence
// and its depth.  64 sequences of 16 tokens, extend and trim: 15 us, 18 with the second launch.
constexpr int kHere = 2048;

__global__ __launch_bounds__(kScan) void pages_extend_kernel(PageArgs a, bool here) {
    __shared__ int64_t wide[kScan / 64];
    __shared__ int lds[kScan / 64], until[kScan], from[kScan];
    __shared__ int first[kScan], count[kScan], lens[kScan], grown[kScan], parents[kHere];  // of all sequences, where they are `here`
    if (here && a.parents)
        for (int t = threadIdx.x; t < a.T; t += kScan) parents[t] = a.parents[t];
    const int have = min(max(a.count[0], 0), a.P);
    int64_t asked = 0;
    int taken = 0;
    for (int b0 = 0; b0 < a.B; b0 += kScan) {
        const int b = b0 + threadIdx.x;
        int need = 0, held = 0;
        bool fits = false;
        int64_t end = 0;
        if (b < a.B) {
            const New s = new_tokens(a, b);
            const int len = a.lens[b];
            first[threadIdx.x] = s.q0;
            count[threadIdx.x] = s.n;
            lens[threadIdx.x] = len;
            held = min(max(a.held[b], 0), a.cols);
            end = (int64_t)len + s.n;
            const int64_t want = (end + (1 << a.pshift) - 1) >> a.pshift;
            fits = len >= 0 && want <= a.cols && !(a.parents && s.n > kTreeNodes);
            need = fits ? max((int)want - held, 0) : 0;
        }
        int64_t total;
        const int64_t upto = asked + scan_block<int64_t>(need, wide, total);
        asked += total;
        // Those that get pages have all that were asked for before them: the sums are one.
        const bool ok = fits && (need == 0 || upto <= have);
        int got;
        until[threadIdx.x] = scan_block<int>(ok ? need : 0, lds, got);
        from[threadIdx.x] = held;
        if (b < a.B) {
            if (ok && need > 0) a.held[b] = held + need;
            a.kv_lens[b] = ok ? (int)end : -1;
            grown[threadIdx.x] = ok;
        }
        __syncthreads();
        for (int k = threadIdx.x; k < got; k += kScan) {
            const int i = owner(until, k), j = k - (i > 0 ? until[i - 1] : 0);
            a.table[(int64_t)(b0 + i) * a.cols + from[i] + j] = a.free[have - 1 - taken - k];
        }
        taken += got;
    }
    if (threadIdx.x == 0) a.count[0] = have - taken;
    if (!here) return;
    __threadfence_block();
    __syncthreads();
    for (int t = threadIdx.x; t < a.T; t += kScan) {
        int lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int i = t - first[lo];
        int slot = -1, position = 0;
        if (i >= 0 && i < count[lo]) {
            const int q0 = first[lo];
            position = lens[lo] + (a.parents && count[lo] <= kTreeNodes ? depth_of(i, [&](int n) { return parents[q0 + n]; }) : i);
            if (grown[lo]) slot = slot_of(a, lo, lens[lo] + i);
        }
        a.slots[t] = slot;
        a.positions[t] = position;
    }
}

// 256 tokens a workgroup, each wave's found by its first one.
__global__ __launch_bounds__(256) void pages_slots_kernel(PageArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x, t0 = t & ~63;
    if (t0 >= a.T) return;
    int b = a.cu ? a.B > 0 ? last_of(a.B, [&](int i) { return a.cu[i] <= t0; }) : -1 : t;
    if (t >= a.T) return;
    int slot = -1, position = 0;
    if (b >= 0) {
        while (a.cu && b + 1 < a.B && a.cu[b + 1] <= t) ++b;  // the wave's later tokens may be later sequences'
        const New s = new_tokens(a, b);
        const int len = a.lens[b], i = t - s.q0;
        if (i >= 0 && i < s.n) {
            position = len + (a.parents && s.n <= kTreeNodes ? depth_of(i, [&](int n) { return a.parents[s.q0 + n]; }) : i);
            if (a.kv_lens[b] >= 0) slot = slot_of(a, b, len + i);
        }
    }
    a.slots[t] = slot;
    a.positions[t] = position;
}

__global__ __launch_bounds__(kScan) void pages_trim_kernel(PageArgs a) {
    __shared__ int lds[kScan / 64], until[kScan], from[kScan];
    const int have = min(max(a.count[0], 0), a.P);
    const auto gone_of = [&](int b, int& keep) {
        keep = 0;
        if (b >= a.B) return 0;
        const int held = min(max(a.held[b], 0), a.cols), len = a.lens[b];
        keep = len < 0 ? held : (int)min(((int64_t)len + (1 << a.pshift) - 1) >> a.pshift, (int64_t)held);
        return held - keep;
    };
    // All that are given back, first: the k-th of R goes to place R - 1 - k.
    int R = 0, before = 0;
    for (int b0 = 0; b0 < a.B; b0 += kScan) {
        int keep, total;
        scan_block<int>(gone_of(b0 + threadIdx.x, keep), lds, total);
        R += total;
    }
    for (int b0 = 0; b0 < a.B; b0 += kScan) {
        int keep, total;
        const int gone = gone_of(b0 + threadIdx.x, keep);
        until[threadIdx.x] = scan_block<int>(gone, lds, total);
        from[threadIdx.x] = keep;
        if (gone > 0) a.held[b0 + threadIdx.x] = keep;
        __syncthreads();
        for (int k = threadIdx.x; k < total; k += kScan) {
            const int i = owner(until, k), j = k - (i > 0 ? until[i - 1] : 0);
            int32_t* const at = a.table + (int64_t)(b0 + i) * a.cols + from[i] + j;
            const int64_t to = (int64_t)have + R - 1 - before - k;
            if (to < a.P) a.free[to] = *at;
            *at = -1;
        }
        before += total;
    }
    if (threadIdx.x == 0) a.count[0] = (int)min((int64_t)have + R, (int64_t)a.P);
}

int page_shift(int page) {
    int s = 4;
    while (s < 10 && (1 << s) != page) ++s;
    return (1 << s) == page ? s : -1;
}

bool check_pages(const char* what, PageArgs& a, int num_pages, int page_size, int B, int cols) {
    a.pshift = page_shift(page_size);
    // B * cols: a table's entries are counted in 32 bits.
    if (a.pshift < 0 || num_pages < 1 || num_pages > (INT32_MAX >> a.pshift) || B < 0 || B > (1 << 20) || cols < 0 ||
        cols > ((1 << 30) >> a.pshift) || (int64_t)B * cols > INT32_MAX) {
        bq_set_error("%s: needs a page size of 16 to 1024 that is a power of two, fewer than 2^31 slots, up to 2^20 "
                     "sequences and a table of fewer than 2^31 entries and 2^30 keys a sequence (got %d pages of %d, %d sequences, %d columns)",
                     what, num_pages, page_size, B, cols);
        return false;
    }
    if (B > 0 && (!a.table || !a.held || !a.free || !a.count || !a.lens)) {
        bq_set_error("%s: null device pointer", what);
        return false;
    }
    a.P = num_pages;
    a.B = B;
    a.cols = cols;
    return true;
}

}  // namespace

extern "C" {

int i4_pages_extend_dev(int32_t* dTable, int32_t* dHeld, int32_t* dFree, int32_t* dCount, int num_pages, int page_size,
                        int B, int cols, const int32_t* dLens, const int32_t* dCu, int T, const int32_t* dParents,
                        int32_t* dSlots, int32_t* dPositions, int32_t* dKvLens, void* stream) {
    PageArgs a{};
    a.table = dTable;
    a.held = dHeld;
    a.free = dFree;
    a.count = dCount;
    a.lens = dLens;
    if (!check_pages("pages_extend", a, num_pages, page_size, B, cols)) return -2;
    if (T < 0 || T > (1 << 30) || (!dCu && T != B) || (T > 0 && (!dSlots || !dPositions)) || (B > 0 && !dKvLens)) {
        bq_set_error("pages_extend: needs up to 2^30 tokens, one a sequence where no offsets are given, and places for "
                     "slots, positions and lengths (got %d tokens of %d sequences)",
                     T, B);
        return -2;
    }
    if (B == 0 && T == 0) return 0;
    a.cu = dCu;
    a.T = T;
    a.parents = dParents;
    a.slots = dSlots;
    a.positions = dPositions;
    a.kv_lens = dKvLens;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    const bool here = T <= kHere && B <= kScan;
    if (B > 0) pages_extend_kernel<<<1, kScan, 0, st>>>(a, here);
    if (T > 0 && (!here || B == 0)) pages_slots_kernel<<<(unsigned)((T + 255) / 256), 256, 0, st>>>(a);
    return launched("pages_extend") ? 0 : -5;
}

int i4_pages_trim_dev(int32_t* dTable, int32_t* dHeld, int32_t* dFree, int32_t* dCount, int num_pages, int page_size,
                      int B, int cols, const int32_t* dLens, void* stream) {
    PageArgs a{};
    a.table = dTable;
    a.held = dHeld;
    a.free = dFree;
    a.count = dCount;
    a.lens = dLens;
    if (!check_pages("pages_trim", a, num_pages, page_size, B, cols)) return -2;
    if (B == 0) return 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    (void)hipGetLastError();
    pages_trim_kernel<<<1, kScan, 0, st>>>(a);
    return launched("pages_trim") ? 0 : -5;
}

}  // extern "C"
