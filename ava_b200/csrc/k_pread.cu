// The read of new tokens over a store in pages, for a few rows per key head (decode steps, drafted runs) and for every
// store type, page size and layout: o = sum_j softmax_j(scale q . k_j) v_j.
//
// One pass with the running maximum and sum per row.  What bounds it is the store's bytes: every key and value is used by
// a handful of rows only, so the kernel is laid out around keeping loads in flight.  A warp is a worker of its own
// (read_split.cuh): it walks its piece of the line in steps of 16 keys, its own ring of 16-key stages in shared memory
// filled by asynchronous 16-byte copies several stages ahead; no barrier joins the warps of a block.  Pages are looked up
// a key at a time (lane = key), one step before their copies are issued, so any page size and any strides of whole 16
// bytes go; keys outside the stretch or on a page outside the store are written as zeros and never read.
// The products run on mma.sync (m16n8k16, bf16 in, f32 sums): 16 rows of queries stand in one operand (a request's tokens
// and the heads that share the key head), and tcgen05's 128-row tiles would be empty for 7 of 8 rows and more.
// f32 queries, f32 stores and the softmax weights of f32 queries are three bf16 limbs each (2^-24 of the value; a store's
// are made as its elements come out of shared memory), and of two limbed operands' nine products the six down to 2^-18 are
// taken.  Two limbs (2^-17) were not enough: an error of 2e-6 of the read where f32 sums leave 5e-7.
#include <cuda_runtime.h>

#include "ava_math.h"
#include "bf16_hw.cuh"
#include "kernels.cuh"
#include "read_split.cuh"
#include "serving.cuh"

namespace ava {

namespace {

constexpr int STEP = 16;                 // keys per stage
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;

__device__ __forceinline__ uint32_t s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_half(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
// the limbs of a pair: each the bf16 nearest to what the ones before leave over
__device__ __forceinline__ void limbs(float a, float b, uint32_t (&l)[1]) { l[0] = pack_bf16(a, b); }
__device__ __forceinline__ void limbs(float a, float b, uint32_t (&l)[3]) {
    l[0] = pack_bf16(a, b);
    a = __fsub_rn(a, low_half(l[0]));
    b = __fsub_rn(b, high_half(l[0]));
    l[1] = pack_bf16(a, b);
    l[2] = pack_bf16(__fsub_rn(a, low_half(l[1])), __fsub_rn(b, high_half(l[1])));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// a . b over the pairs of limbs whose product is at least 2^-18 of the leading one: high += the leading pair, low += the
// others.  The tensor cores' f32 sums are cut, not rounded, at every addition: one running sum over all limbs and keys
// lost 4e-6 of a read over 2048 keys, always towards 0.  So the small terms have a sum of their own, and no sum on the
// tensor cores runs over more than one step's keys.
template <int LA, int LB>
__device__ __forceinline__ void mma_limbs(float (&high)[4], float (&low)[4], const uint32_t (&a)[LA][4], const uint32_t (&b0)[LB], const uint32_t (&b1)[LB]) {
#pragma unroll
    for (int i = 0; i < LA; ++i)
#pragma unroll
        for (int j = 0; j < LB; ++j)
            if (i + j > 0 && i + j <= 2) mma16816(low, a[i], b0[j], b1[j]);
    mma16816(high, a[0], b0[0], b1[0]);
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// How a warp lays out its stage: 16 rows of HS elements of K, then of V; the 16-byte pieces of a row are rotated by the
// row so that eight rows' equal pieces lie in eight bank groups.
template <typename TS, int HS>
struct Stage {
    static constexpr int ROW = HS * (int)sizeof(TS), PIECES = ROW / 16, BYTES = 2 * STEP * ROW;
    static __device__ __forceinline__ uint32_t at(int key, int piece) {
        const int turn = PIECES >= 8 ? (key & 7) : ((key >> 1) & 3);
        return (uint32_t)(key * ROW + ((piece ^ turn) << 4));
    }
};

// tiles of MR rows, cut into stages; stretches of up to eight stages (128 keys) are not cut
template <int MT>
struct Plan {
    static constexpr int MR = 16 * MT, KT = STEP, START = 2, SNAP = 8;
};

// Workspace of one worker's piece: the two ends that may be cut (0: goes on from the worker before, 1: goes on in the
// next), each MR rows of HS sums, then the rows' maxima (of scores times log2 e) and sums.
template <int HS, int MR>
struct Ends {
    static constexpr int FLOATS = MR * (HS + 2);
};

template <typename TS, int L, int HS, int MT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) read_kernel(const ReadArgs a, float* __restrict__ ends, split::Cut* __restrict__ cuts, const int workers) {
    constexpr int MR = 16 * MT, KK = HS / 16, NB = HS / 8;
    constexpr bool F32S = sizeof(TS) == 4;
    constexpr int LS = F32S ? 3 : 1;   // limbs of the store's elements
    using St = Stage<TS, HS>;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ long long sums[split::ENTRIES + 1];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tq = lane & 3;
    bool bad_length = false, bad_page = false;
    using Pl = Plan<MT>;
    const split::Line line = split::line<Pl>(a, sums, &bad_length);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (bad_length && a.status && blockIdx.x == 0) atomicOr(a.status, AVA_PAGED_BAD_LENGTH);

    const int w = blockIdx.x * WARPS + warp;
    const long long per = max((line.total() + workers - 1) / workers, 1ll);
    split::Item it = {}, after = {};
    long long u = split::piece<Pl>(a, line, per, w, &it);
    const long long end = split::piece<Pl>(a, line, per, w + 1ll, &after);
    if (lane == 0) cuts[w].workers = 0;
    unsigned char* ring = smem + warp * STAGES * St::BYTES;
    const uint32_t ring_at = s32(ring);
    const float scale2 = a.scale * LOG2E;
    const bool paired = !((reinterpret_cast<uintptr_t>(a.out) & (a.bf16_q ? 3 : 7)) || (a.out_token_stride & 1) || (a.out_head_stride & 1));
    const int page_shift = (a.s.page_size & (a.s.page_size - 1)) ? -1 : __ffs(a.s.page_size) - 1;
    const TS* pool_k = static_cast<const TS*>(a.s.k);
    const TS* pool_v = static_cast<const TS*>(a.s.v);

    while (u < end) {
        const split::Share run = split::share<Pl>(it, u, end);
        const bool whole = run.whole;
        const int rows = min(it.q.f * a.group - it.tile * MR, MR);
        // this warp's keys of the stretch: from step t0 to t1 of the store's own 16-key steps
        const bool none = it.s.lo >= it.s.hi;
        const int t0 = none ? 0 : it.s.lo / STEP + run.from, t1 = none ? 0 : it.s.lo / STEP + run.to;
        const int32_t* pages = a.table + (int64_t)it.r * a.max_pages;
        const int64_t head_at = (int64_t)it.head * a.s.head_stride;

        // the place of key t * 16 + (lane & 15) in the pools, -1: none
        auto place = [&](int t) -> int64_t {
            const int j = t * STEP + (lane & 15);
            if (t >= t1 || j < it.s.lo || j >= it.s.hi) return -1;
            const int pi = page_shift >= 0 ? j >> page_shift : j / a.s.page_size;
            const int page = pages[pi];
            if (page < 0 || page >= a.s.n_pages) {
                bad_page = true;
                return -1;
            }
            return page * a.s.page_stride + (j - pi * a.s.page_size) * a.s.place_stride + head_at;
        };
        auto fetch = [&](int t, int64_t at) {
            const uint32_t dst = ring_at + (uint32_t)(((unsigned)(t - t0) % STAGES) * St::BYTES);
#pragma unroll
            for (int i = 0; i < St::PIECES / 2; ++i) {
                const int id = i * 32 + lane, key = id / St::PIECES, piece = id % St::PIECES;
                const int64_t from = __shfl_sync(0xffffffffu, at, key);
                const int64_t e = (from < 0 ? 0 : from) + piece * (16 / (int)sizeof(TS));
                copy16(dst + St::at(key, piece), pool_k + e, from >= 0);
                copy16(dst + STEP * St::ROW + St::at(key, piece), pool_v + e, from >= 0);
            }
        };
        __syncwarp();   // the stretch before has been read out of the ring by every lane
        int64_t coming = -1;
        if (t0 < t1) {
            int64_t at = place(t0);
#pragma unroll 1
            for (int s = 0; s < STAGES - 1; ++s) {
                const int64_t ahead = place(t0 + s + 1);
                if (t0 + s < t1) fetch(t0 + s, at);
                asm volatile("cp.async.commit_group;" ::: "memory");
                at = ahead;
            }
            coming = at;
        }

        // queries: row m = tile * MR + 16 mt + g (+ 8), channels 16 kk + 2 tq (+ 8)
        uint32_t qf[MT][KK][L][4];
        int pos[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int m = it.tile * MR + min(16 * mt + g + 8 * half, rows - 1);   // rows beyond the last repeat it: no mask of their own
                const int i = m / a.group, h = it.head * a.group + (m - i * a.group);
                pos[mt][half] = it.q.c + i;
                const int64_t at = (int64_t)(it.q.start + i) * a.q_token_stride + (int64_t)h * a.q_head_stride;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        const int64_t e = at + 16 * kk + 8 * o + 2 * tq;
                        if (L == 3) {
                            const float* q = static_cast<const float*>(a.q) + e;
                            uint32_t l[L];
                            limbs(q[0], q[1], l);
#pragma unroll
                            for (int x = 0; x < L; ++x) qf[mt][kk][x][2 * o + half] = l[x];
                        } else {
                            const uint16_t* q = static_cast<const uint16_t*>(a.q) + e;
                            qf[mt][kk][0][2 * o + half] = q[0] | ((uint32_t)q[1] << 16);
                        }
                    }
            }

        float acc[MT][NB][4], top[MT][2], sum[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            top[mt][0] = top[mt][1] = -INFINITY;
            sum[mt][0] = sum[mt][1] = 0.0f;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[mt][n][i] = 0.0f;
        }
        // keys that every row of the tile sees need no comparison
        const int all_from = a.window > 0 ? max(it.q.first, it.q.c + (it.tile * MR + rows - 1) / a.group + 1 - a.window) : it.q.first;
        const int all_to = it.q.c + (it.tile * MR) / a.group + 1;

#pragma unroll 1
        for (int t = t0; t < t1; ++t) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();
            {   // the stage read last is free: the step STAGES - 1 ahead goes into it
                const int ahead = t + STAGES - 1;
                if (ahead < t1) fetch(ahead, coming);
                asm volatile("cp.async.commit_group;" ::: "memory");
                coming = place(ahead + 1);
            }
            const uint32_t at_k = ring_at + (uint32_t)(((unsigned)(t - t0) % STAGES) * St::BYTES), at_v = at_k + STEP * St::ROW;
            const unsigned char* st = ring + (at_k - ring_at);

            float s[MT][2][4], sl[MT][2][4];   // leading products, the others
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[mt][n][i] = sl[mt][n][i] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                uint32_t b[4][LS];
                if constexpr (F32S) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const int ch = 16 * kk + 8 * o + 2 * tq;
                            const float2 x = *reinterpret_cast<const float2*>(st + St::at(8 * n + g, ch / 4) + (ch & 3) * 4);
                            limbs(x.x, x.y, b[2 * n + o]);
                        }
                } else {
                    uint32_t x[4];
                    ldmatrix4(at_k + St::at((lane & 7) + 8 * (lane >> 4), 2 * kk + ((lane >> 3) & 1)), x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i][0] = x[i];
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < 2; ++n) mma_limbs(s[mt][n], sl[mt][n], qf[mt][kk], b[2 * n], b[2 * n + 1]);
            }
            // scores in units of log2: hidden keys to -infinity, the running maximum, the weights
            const int j0 = t * STEP;
            const bool edge = j0 < all_from || j0 + STEP > all_to;
            uint32_t wf[MT][L][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[mt][n][i] = (L == 3 ? s[mt][n][i] + sl[mt][n][i] : s[mt][n][i]) * scale2;
                if (edge) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = j0 + 8 * n + 2 * tq + (i & 1), p = pos[mt][i >> 1];
                            if (j > p || j < it.q.first || (a.window > 0 && j <= p - a.window)) s[mt][n][i] = -INFINITY;
                        }
                }
                float high[2];
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    high[half] = fmaxf(fmaxf(s[mt][0][2 * half], s[mt][0][2 * half + 1]), fmaxf(s[mt][1][2 * half], s[mt][1][2 * half + 1]));
                if (__any_sync(0xffffffffu, high[0] > top[mt][0] || high[1] > top[mt][1])) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float x = fmaxf(high[half], __shfl_xor_sync(0xffffffffu, high[half], 1));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                        x = fmaxf(x, top[mt][half]);
                        const float f = top[mt][half] == -INFINITY ? 0.0f : exp2_fast(top[mt][half] - x);
                        top[mt][half] = x;
                        sum[mt][half] *= f;
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            acc[mt][n][2 * half] *= f;
                            acc[mt][n][2 * half + 1] *= f;
                        }
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float base = top[mt][half] == -INFINITY ? 0.0f : top[mt][half];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float x = exp2_fast(s[mt][n][2 * half] - base), y = exp2_fast(s[mt][n][2 * half + 1] - base);
                        sum[mt][half] += x + y;
                        uint32_t l[L];
                        limbs(x, y, l);
#pragma unroll
                        for (int i = 0; i < L; ++i) wf[mt][i][2 * n + half] = l[i];
                    }
                }
            }
#pragma unroll
            for (int n2 = 0; n2 < NB / 2; ++n2) {
                uint32_t b[4][LS];
                if constexpr (F32S) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const int ch = 16 * n2 + 8 * n + g, key = 8 * o + 2 * tq;
                            const unsigned char* v = st + STEP * St::ROW + (ch & 3) * 4;
                            limbs(*reinterpret_cast<const float*>(v + St::at(key, ch / 4)), *reinterpret_cast<const float*>(v + St::at(key + 1, ch / 4)), b[2 * n + o]);
                        }
                } else {
                    uint32_t x[4];
                    ldmatrix4_trans(at_v + St::at((lane & 7) + 8 * ((lane >> 3) & 1), 2 * n2 + (lane >> 4)), x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i][0] = x[i];
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        if constexpr (L == 3) {
                            float high[4] = {0.0f, 0.0f, 0.0f, 0.0f}, low[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_limbs(high, low, wf[mt], b[2 * n], b[2 * n + 1]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[mt][2 * n2 + n][i] += high[i] + low[i];
                        } else {
                            mma16816(acc[mt][2 * n2 + n], wf[mt][0], b[2 * n][0], b[2 * n + 1][0]);
                        }
                    }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // the rows' sums over the quad, then the read itself or this piece's end of it
        float* part = ends + ((int64_t)w * 2 + (u == it.begin ? 1 : 0)) * Ends<HS, MR>::FLOATS;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float l = sum[mt][half];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                const int row = 16 * mt + g + 8 * half;
                if (row >= rows) continue;
                if (whole) {
                    const float inv = l > 0.0f ? 1.0f / l : l;   // a sum that is NaN stays NaN
                    const int m = it.tile * MR + row, i = m / a.group, h = it.head * a.group + (m - i * a.group);
                    const int64_t to = (int64_t)(it.q.start + i) * a.out_token_stride + (int64_t)h * a.out_head_stride + 2 * tq;
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        const float x = acc[mt][n][2 * half] * inv, y = acc[mt][n][2 * half + 1] * inv;
                        if (L == 1) {
                            uint16_t* o = static_cast<uint16_t*>(a.out) + to + 8 * n;
                            const uint32_t v = pack_bf16(x, y);
                            if (paired) *reinterpret_cast<uint32_t*>(o) = v;
                            else {
                                o[0] = (uint16_t)v;
                                o[1] = (uint16_t)(v >> 16);
                            }
                        } else {
                            float* o = static_cast<float*>(a.out) + to + 8 * n;
                            if (paired) *reinterpret_cast<float2*>(o) = make_float2(x, y);
                            else {
                                o[0] = x;
                                o[1] = y;
                            }
                        }
                    }
                    if (a.lse && tq == 0) a.lse[(int64_t)(it.q.start + i) * a.heads + h] = l == 0.0f ? -INFINITY : (top[mt][half] + log2f(l)) * LN2;
                } else {
#pragma unroll
                    for (int n = 0; n < NB; ++n)
                        *reinterpret_cast<float2*>(part + row * HS + 8 * n + 2 * tq) = make_float2(acc[mt][n][2 * half], acc[mt][n][2 * half + 1]);
                    if (tq == 0) {
                        part[MR * HS + row] = top[mt][half];
                        part[MR * HS + MR + row] = l;
                    }
                }
            }
        if (!whole && u == it.begin && lane == 0) {
            cuts[w].r = it.r;
            cuts[w].head = it.head;
            cuts[w].tile = it.tile;
            cuts[w].workers = (int)split::last_worker<Pl>(it, per) - w + 1;
        }
        u = run.stop;
        if (u < end) split::next<Pl>(a, it);
    }
    if (__any_sync(0xffffffffu, bad_page) && lane == 0 && a.status) atomicOr(a.status, AVA_PAGED_BAD_PAGE);
}

// Joins the ends of the stretches that were cut: one block per worker, idle unless a cut stretch begins in its piece.
// With the parts' maxima m_i, sums l_i and mixes o_i: m = max m_i, out = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i.
constexpr int JOIN_WARPS = 8;
template <int HS, int MR>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const ReadArgs a, const float* __restrict__ ends, const split::Cut* __restrict__ cuts) {
    pdl_enter();
    const int w = blockIdx.x, n = cuts[w].workers;
    if (n == 0) return;
    constexpr int PER = HS / 32;
    __shared__ float part_o[JOIN_WARPS][HS], part_m[JOIN_WARPS], part_l[JOIN_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    bool bad = false;
    const split::Request q = split::request(a, cuts[w].r, &bad);
    const int head = cuts[w].head, tile = cuts[w].tile, rows = min(q.f * a.group - tile * MR, MR);
    for (int row = 0; row < rows; ++row) {
        float m = -INFINITY, l = 0.0f, o[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = 0.0f;
        for (int k = warp; k < n; k += JOIN_WARPS) {
            const float* part = ends + ((int64_t)(w + k) * 2 + (k == 0 ? 1 : 0)) * Ends<HS, MR>::FLOATS;
            const float mk = part[MR * HS + row], lk = part[MR * HS + MR + row], mn = fmaxf(m, mk);
            const float fo = m == -INFINITY ? 0.0f : exp2_fast(m - mn), fk = mk == -INFINITY ? 0.0f : exp2_fast(mk - mn);
            l = l * fo + lk * fk;
#pragma unroll
            for (int i = 0; i < PER; ++i) o[i] = o[i] * fo + part[row * HS + lane + 32 * i] * fk;
            m = mn;
        }
        if (lane == 0) {
            part_m[warp] = m;
            part_l[warp] = l;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) part_o[warp][lane + 32 * i] = o[i];
        __syncthreads();
        if (warp == 0) {
            m = part_m[0];
            for (int k = 1; k < JOIN_WARPS; ++k) m = fmaxf(m, part_m[k]);
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) o[i] = 0.0f;
            for (int k = 0; k < JOIN_WARPS; ++k) {
                const float f = part_m[k] == -INFINITY ? 0.0f : exp2_fast(part_m[k] - m);
                l += part_l[k] * f;
#pragma unroll
                for (int i = 0; i < PER; ++i) o[i] += part_o[k][lane + 32 * i] * f;
            }
            const float inv = l > 0.0f ? 1.0f / l : l;
            const int mm = tile * MR + row, i = mm / a.group, h = head * a.group + (mm - i * a.group);
            const int64_t to = (int64_t)(q.start + i) * a.out_token_stride + (int64_t)h * a.out_head_stride + lane;
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                if (a.bf16_q) static_cast<uint16_t*>(a.out)[to + 32 * c] = bf16_rn_hw(o[c] * inv);
                else static_cast<float*>(a.out)[to + 32 * c] = o[c] * inv;
            }
            if (a.lse && lane == 0) a.lse[(int64_t)(q.start + i) * a.heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
        }
        __syncthreads();
    }
}

constexpr int most_warps(int stage_bytes, int mt) { return mt > 1 ? 8 : stage_bytes <= 2048 ? 16 : stage_bytes <= 4096 ? 12 : stage_bytes <= 8192 ? 8 : 6; }
constexpr int most_stages(int stage_bytes, int mt) { return 196608 / (most_warps(stage_bytes, mt) * stage_bytes); }

template <typename TS, int L, int HS, int MT>
cudaError_t launch_one(cudaStream_t st, const ReadArgs& a, void* room, int sms) {
    constexpr int BYTES = Stage<TS, HS>::BYTES, WARPS = most_warps(BYTES, MT), STAGES = most_stages(BYTES, MT), MR = 16 * MT;
    const int workers = sms * WARPS;
    split::Cut* cuts = static_cast<split::Cut*>(room);
    float* ends = reinterpret_cast<float*>(cuts + workers);
    cudaError_t rc = launch_serving(read_kernel<TS, L, HS, MT, WARPS, STAGES>, dim3(sms), dim3(WARPS * 32), (size_t)WARPS * STAGES * BYTES, st, 1, a, ends, cuts, workers);
    if (rc != cudaSuccess) return rc;
    return launch_serving(join_kernel<HS, MR>, dim3(workers), dim3(JOIN_WARPS * 32), 0, st, 1, a, ends, cuts);
}

template <int HS>
cudaError_t launch_size(cudaStream_t st, const ReadArgs& a, void* room, int sms) {
    // Rows per key head that the host expects: one tile of 16 reads the store once for up to 16 of them, a tile of 32 for
    // twice as many (not with f32 queries of 128 channels: their limbs and sums would not stay in registers).
    const bool wide = (int64_t)a.max_fresh * a.group > 16;
    if (a.bf16_q) return wide ? launch_one<uint16_t, 1, HS, 2>(st, a, room, sms) : launch_one<uint16_t, 1, HS, 1>(st, a, room, sms);
    if (a.s.dtype == AVA_BF16) {
        if constexpr (HS < 128)
            if (wide) return launch_one<uint16_t, 3, HS, 2>(st, a, room, sms);
        return launch_one<uint16_t, 3, HS, 1>(st, a, room, sms);
    }
    if constexpr (HS < 128)
        if (wide) return launch_one<float, 3, HS, 2>(st, a, room, sms);
    return launch_one<float, 3, HS, 1>(st, a, room, sms);
}

}  // namespace

int64_t paged_read_workspace(int head_size, int sms) {
    // at most 16 workers on an SM, and at most 256 rows of their tiles (most_warps times 16 or 32)
    return (int64_t)sms * 16 * (int64_t)sizeof(split::Cut) + (int64_t)sms * 256 * 2 * (head_size + 2) * 4;
}

cudaError_t launch_paged_read(cudaStream_t st, const ReadArgs& a, void* room, int sms) {
    bool taken = false;
    const cudaError_t rc = launch_paged_read_tc(st, a, room, sms, &taken);
    if (taken || rc != cudaSuccess) return rc;
    if (a.s.head_size == 32) return launch_size<32>(st, a, room, sms);
    if (a.s.head_size == 64) return launch_size<64>(st, a, room, sms);
    return launch_size<128>(st, a, room, sms);
}

}  // namespace ava
