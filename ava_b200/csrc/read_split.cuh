// How a read over pages is cut into equal shares.
//
// The new tokens' rows of one request and key head (token-major, the heads that share the key head innermost) are cut into
// tiles of MR rows; a tile reads a stretch of keys, cut into units of KT keys.  All units of the call, in the order
// (request, key head, tile, keys), form one line, and every worker (a warp or a block) takes an equal piece of it, so the
// shares are even whatever the lengths are: one long sequence, a few long prompts or hundreds of ragged requests.  A
// worker's piece may begin or end inside a tile's stretch; those two ends go to the workspace as unnormalised sums with
// their running maximum, and a second kernel joins them (the read itself is then no different from one pass).  A tile also
// costs what lies around its keys (its queries, its results): START units more, in front of the stretch on the line.
// Stretches of at most SNAP units are never cut.  The lengths are read on the GPU, so the same launch fits any of them.
#pragma once

#include <cuda_runtime.h>

#include "serving.cuh"

namespace ava {
namespace split {

constexpr long long MOST_KEYS = 1ll << 29;   // of a request: a warp's tiles together stay within 32 bits of units
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
    if (q.start < 0 || end < q.start || end > a.max_tokens || q.c < 0 || total > (long long)a.max_pages * a.s.page_size || total >= MOST_KEYS) {
        q.f = 0;
        *bad = true;
    }
    return q;
}

struct Stretch {
    int lo, hi;                 // keys some row of the tile sees: [lo, hi); none: hi <= lo
    int units;
};

template <typename P>
__device__ __forceinline__ Stretch stretch(const ReadArgs& a, const Request& q, int tile) {
    const int m0 = tile * P::MR, m1 = min(q.f * a.group, m0 + P::MR) - 1;
    const int i0 = m0 / a.group, i1 = m1 / a.group;
    Stretch s;
    s.hi = q.c + i1 + 1;
    s.lo = a.window > 0 ? max(q.first, q.c + i0 + 1 - a.window) : q.first;
    s.units = s.lo < s.hi ? (s.hi - 1) / P::KT - s.lo / P::KT + 1 : 1;   // a tile that sees nothing still has its zeros to write
    return s;
}

template <typename P>
__device__ __forceinline__ int tiles(const ReadArgs& a, const Request& q) {
    return (q.f * a.group + P::MR - 1) / P::MR;
}

// What one key head of a request takes of the line: by one thread, and by a warp together (a prompt has many tiles).
template <typename P>
__device__ __forceinline__ long long head_units(const ReadArgs& a, const Request& q) {
    long long n = 0;
    for (int t = 0, e = tiles<P>(a, q); t < e; ++t) n += P::START + stretch<P>(a, q, t).units;
    return n;
}
template <typename P>
__device__ __forceinline__ long long head_units_warp(const ReadArgs& a, const Request& q) {
    const int e = tiles<P>(a, q), lane = threadIdx.x & 31;
    if (e <= 1) return e ? P::START + stretch<P>(a, q, 0).units : 0;
    long long n = 0;
    for (int t = lane; t < e; t += 32) n += P::START + stretch<P>(a, q, t).units;
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

// Where the line's requests begin: sums[e] units lie before request e * step (e = 0 .. entries), by all threads of a block.
struct Line {
    long long* sums;            // shared memory, ENTRIES + 1
    int entries, step;
    __device__ __forceinline__ long long total() const { return sums[entries]; }
};

template <typename P>
__device__ __forceinline__ Line line(const ReadArgs& a, long long* sums, bool* bad) {
    Line l;
    l.sums = sums;
    l.step = (a.rows + ENTRIES - 1) / ENTRIES;
    l.entries = (a.rows + l.step - 1) / l.step;
    if (a.rows < 128) {         // few requests: a warp each, a lane per tile
        for (int r = threadIdx.x >> 5; r < a.rows; r += blockDim.x >> 5) {
            const long long n = head_units_warp<P>(a, request(a, r, bad)) * a.s.kv_heads;
            if ((threadIdx.x & 31) == 0) sums[r + 1] = n;
        }
    } else {
        for (int e = threadIdx.x; e < l.entries; e += blockDim.x) {
            long long n = 0;
            for (int r = e * l.step, end = min(a.rows, r + l.step); r < end; ++r) n += head_units<P>(a, request(a, r, bad)) * a.s.kv_heads;
            sums[e + 1] = n;
        }
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
    long long begin;            // where the stretch's START units begin; its own follow
};

// The stretch that place u of the line lies in (u < total), by a warp together.  known (may be null): an item whose request
// need not be looked at again.
template <typename P>
__device__ __forceinline__ Item locate(const ReadArgs& a, const Line& l, long long u, const Item* known) {
    int lo = 0, hi = l.entries;
    while (hi - lo > 1) {       // the last entry whose sum is not above u: empty requests are passed over
        const int mid = (lo + hi) >> 1;
        if (l.sums[mid] <= u) lo = mid;
        else hi = mid;
    }
    Item it = {};
    bool bad = false;
    it.begin = l.sums[lo];
    it.r = lo * l.step;
    long long n = 0;
    for (;; ++it.r) {
        if (known && known->r == it.r) it.q = known->q;
        else it.q = request(a, it.r, &bad);
        n = l.step == 1 ? l.sums[lo + 1] - it.begin : head_units_warp<P>(a, it.q) * a.s.kv_heads;
        if (u < it.begin + n) break;
        it.begin += n;
    }
    n /= a.s.kv_heads;
    it.head = (int)((u - it.begin) / n);
    it.begin += n * it.head;
    const int e = tiles<P>(a, it.q), lane = threadIdx.x & 31;
    for (int t0 = 0;; t0 += 32) {   // 32 tiles at a time
        const int t = t0 + lane;
        const int own = t < e ? P::START + stretch<P>(a, it.q, t).units : 0;
        int inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, it.begin + inc > u);
        if (over) {
            const int k = __ffs(over) - 1;
            it.begin += __shfl_sync(0xffffffffu, inc - own, k);
            it.tile = t0 + k;
            break;
        }
        it.begin += __shfl_sync(0xffffffffu, inc, 31);
    }
    it.s = stretch<P>(a, it.q, it.tile);
    return it;
}

// The next stretch of the line (there is one).
template <typename P>
__device__ __forceinline__ void next(const ReadArgs& a, Item& it) {
    it.begin += P::START + it.s.units;
    if (++it.tile == tiles<P>(a, it.q)) {
        it.tile = 0;
        if (++it.head == a.s.kv_heads) {
            it.head = 0;
            bool bad = false;
            do it.q = request(a, ++it.r, &bad);
            while (it.q.f == 0);
        }
    }
    it.s = stretch<P>(a, it.q, it.tile);
}

// Where worker w's piece begins; a place inside a stretch of at most SNAP units, or within START + SNAP / 2 units of a
// stretch's beginning, moves to that beginning.
template <typename P>
__device__ __forceinline__ long long piece(const ReadArgs& a, const Line& l, long long per, long long w, Item* it, const Item* known = nullptr) {
    const long long u = w * per;
    if (u >= l.total()) return l.total();
    *it = locate<P>(a, l, u, known);
    return it->s.units <= P::SNAP || u <= it->begin + P::START + P::SNAP / 2 ? it->begin : u;
}

// A worker's run over one stretch, from place u of the line on: its units [from, to) of the stretch, and where it stops.
struct Share {
    int from, to;
    long long stop;
    bool whole;
};
template <typename P>
__device__ __forceinline__ Share share(const Item& it, long long u, long long end) {
    Share s;
    const long long first = it.begin + P::START;
    s.stop = min(end, first + it.s.units);
    s.from = u > first ? (int)(u - first) : 0;
    s.to = (int)(s.stop - first);
    s.whole = u == it.begin && s.to == it.s.units;
    return s;
}
// The worker whose piece the stretch's last unit lies in (a stretch that is cut: no beginning of a piece inside it has moved
// but to its own beginning).
template <typename P>
__device__ __forceinline__ long long last_worker(const Item& it, long long per) {
    return (it.begin + P::START + it.s.units - 1) / per;
}

// What the joining kernel is told by the worker in whose piece a cut stretch begins.
struct __align__(16) Cut {
    int workers;                // how many workers' pieces the stretch runs through; 0: this worker begins none
    int start, head, tile, rows;   // the request's first packed token, the key head, the tile and its rows
    int unused[3];
};

}  // namespace split
}  // namespace ava
