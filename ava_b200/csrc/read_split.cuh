// How a read over pages is cut into equal shares.
//
// The new tokens' rows of one request and key head (token-major, the heads that share the key head innermost) are cut into
// tiles of MR rows; a tile reads a stretch of keys, cut into units of KT keys.  All units of the call, in the order
// (request, key head, tile, keys), form one line, and every worker (a warp or a block) takes an equal piece of it, so the
// shares are even whatever the lengths are: one long sequence, a few long prompts or hundreds of ragged requests.  A
// worker's piece may begin or end inside a tile's stretch; those two ends go to the workspace as unnormalised sums with
// their running maximum, and a second kernel joins them (the read itself is then no different from one pass).  Stretches
// of at most SNAP units are never cut.  The lengths are read on the GPU, so the same launch fits any of them.
#pragma once

#include <cuda_runtime.h>

#include "serving.cuh"

namespace ava {
namespace split {

constexpr int ENTRIES = 2048;   // sums over requests kept in shared memory (each of several requests when there are more)

struct Request {
    int c, f, first, start;     // tokens stored, new tokens, first key that counts, first packed token
};

// What request r asks for; one whose lengths do not fit its arrays asks for nothing.
__device__ __forceinline__ Request request(const ReadArgs& a, int r, bool* bad) {
    Request q;
    q.start = a.q_start[r];
    const int end = a.q_start[r + 1];
    q.c = a.cached[r];
    q.first = a.first ? max(a.first[r], 0) : 0;
    q.f = end - q.start;
    const long long total = (long long)q.c + q.f;
    if (q.start < 0 || end < q.start || end > a.max_tokens || q.c < 0 || total > (long long)a.max_pages * a.s.page_size || total > 0x7ffffff0ll) {
        q.f = 0;
        *bad = true;
    }
    return q;
}

struct Stretch {
    int lo, hi;                 // keys some row of the tile sees: [lo, hi); none: hi <= lo
    int units;
};

template <int MR, int KT>
__device__ __forceinline__ Stretch stretch(const ReadArgs& a, const Request& q, int tile) {
    const int m0 = tile * MR, m1 = min(q.f * a.group, m0 + MR) - 1;
    const int i0 = m0 / a.group, i1 = m1 / a.group;
    Stretch s;
    s.hi = q.c + i1 + 1;
    s.lo = a.window > 0 ? max(q.first, q.c + i0 + 1 - a.window) : q.first;
    s.units = s.lo < s.hi ? (s.hi - 1) / KT - s.lo / KT + 1 : 1;   // a tile that sees nothing still has its zeros to write
    return s;
}

template <int MR>
__device__ __forceinline__ int tiles(const ReadArgs& a, const Request& q) {
    return (q.f * a.group + MR - 1) / MR;
}

template <int MR, int KT>
__device__ __forceinline__ long long request_units(const ReadArgs& a, int r, bool* bad) {
    const Request q = request(a, r, bad);
    long long n = 0;
    for (int t = 0, e = tiles<MR>(a, q); t < e; ++t) n += stretch<MR, KT>(a, q, t).units;
    return n * a.s.kv_heads;
}

// Where the line's requests begin: sums[e] units lie before request e * step (e = 0 .. entries), by all threads of a block.
struct Line {
    long long* sums;            // shared memory, ENTRIES + 1
    int entries, step;
    __device__ __forceinline__ long long total() const { return sums[entries]; }
};

template <int MR, int KT>
__device__ __forceinline__ Line line(const ReadArgs& a, long long* sums, bool* bad) {
    Line l;
    l.sums = sums;
    l.step = (a.rows + ENTRIES - 1) / ENTRIES;
    l.entries = (a.rows + l.step - 1) / l.step;
    for (int e = threadIdx.x; e < l.entries; e += blockDim.x) {
        long long n = 0;
        for (int r = e * l.step, end = min(a.rows, r + l.step); r < end; ++r) n += request_units<MR, KT>(a, r, bad);
        sums[e + 1] = n;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int per = (l.entries + 31) / 32, e0 = threadIdx.x * per, e1 = min(l.entries, e0 + per);
        long long n = 0;
        for (int e = e0; e < e1; ++e) n += sums[e + 1];
        long long inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, inc, o);
            if ((int)threadIdx.x >= o) inc += y;
        }
        n = inc - n;
        for (int e = e0; e < e1; ++e) {
            n += sums[e + 1];
            sums[e + 1] = n;
        }
        if (threadIdx.x == 0) sums[0] = 0;
    }
    __syncthreads();
    return l;
}

// A place on the line: a tile's stretch and where it begins.
struct Item {
    int r, head, tile;
    Request q;
    Stretch s;
    long long begin;            // the stretch's first unit
};

// The stretch that unit u lies in (u < total).
template <int MR, int KT>
__device__ __forceinline__ Item locate(const ReadArgs& a, const Line& l, long long u) {
    int lo = 0, hi = l.entries;
    while (hi - lo > 1) {       // the last entry whose sum is not above u: empty requests are passed over
        const int mid = (lo + hi) >> 1;
        if (l.sums[mid] <= u) lo = mid;
        else hi = mid;
    }
    Item it;
    bool bad = false;
    it.begin = l.sums[lo];
    it.r = lo * l.step;
    long long n = 0;
    for (;; ++it.r) {
        n = request_units<MR, KT>(a, it.r, &bad);
        if (u < it.begin + n) break;
        it.begin += n;
    }
    it.q = request(a, it.r, &bad);
    n /= a.s.kv_heads;
    it.head = (int)((u - it.begin) / n);
    it.begin += n * it.head;
    for (it.tile = 0;; ++it.tile) {
        it.s = stretch<MR, KT>(a, it.q, it.tile);
        if (u < it.begin + it.s.units) break;
        it.begin += it.s.units;
    }
    return it;
}

// The next stretch of the line (there is one).
template <int MR, int KT>
__device__ __forceinline__ void next(const ReadArgs& a, Item& it) {
    it.begin += it.s.units;
    if (++it.tile == tiles<MR>(a, it.q)) {
        it.tile = 0;
        if (++it.head == a.s.kv_heads) {
            it.head = 0;
            bool bad = false;
            do it.q = request(a, ++it.r, &bad);
            while (it.q.f == 0);
        }
    }
    it.s = stretch<MR, KT>(a, it.q, it.tile);
}

// The first unit of worker w's piece; one that would fall inside a stretch of at most SNAP units moves to its beginning.
template <int MR, int KT, int SNAP>
__device__ __forceinline__ long long piece(const ReadArgs& a, const Line& l, long long per, long long w, Item* it) {
    const long long u = w * per;
    if (u >= l.total()) return l.total();
    *it = locate<MR, KT>(a, l, u);
    return it->s.units <= SNAP ? it->begin : u;
}

// What the joining kernel is told by the worker in whose piece a cut stretch begins.
struct Cut {
    int r, head, tile;
    int workers;                // how many workers' pieces the stretch runs through; 0: this worker begins none
};

}  // namespace split
}  // namespace ava
