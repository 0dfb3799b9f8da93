// The read of new tokens over a store in pages, for a few rows per key head (decode steps, drafted runs) and for every
// store type, page size and layout: o = sum_j softmax_j(scale q . k_j) v_j.
//
// One pass with the running maximum and sum per row.  What bounds it is the store's bytes: every key and value is used by
// a handful of rows only, so the kernel is laid out around keeping loads in flight and few instructions around them.  A
// warp is a worker of its own (read_split.cuh): it walks its piece of the line in steps of 16 keys, its own ring of 16-key
// stages in shared memory filled several stages ahead; no barrier joins the warps of a block.  Pages of 8 or of a multiple
// of 16 keys come by TMA, one lane asking for 16 keys at a time (a page outside the store is a coordinate past the tensor's
// last page: zeros, nothing read); other page sizes and strides that do not nest by asynchronous 16-byte copies, every lane
// looking up a key.  Values of places that are no key of the stretch are written over with zeros.
// The products run on mma.sync (m16n8k16, bf16 in, f32 sums) with the keys on the long side: S^T = K Q^T and O^T = V^T P^T,
// so eight rows of queries (a request's tokens and the heads that share the key head) cost one operand of eight columns;
// with the queries on the long side a single decoded token paid for 16, and with tcgen05's 128-row tiles it would for 128.
// f32 queries, f32 stores and the softmax weights of f32 queries are three bf16 limbs each (2^-24 of the value; a store's
// are made as its elements come out of shared memory), and of two limbed operands' nine products the six down to 2^-18 are
// taken.  Two limbs (2^-17) were not enough: an error of 2e-6 of the read where f32 sums leave 5e-7.
// Measured (one B200, 6.57 TB/s copy): one token of 256 sequences of 1024 to 2048 keys, 12 heads of 64, f32 over bf16: 181 us
// for 1.12 GB, 0.93 of the copy rate; one token over 131072 keys 74 us, 0.83 (9 us pass until the first keys are multiplied,
// 5 us join the parts); drafted runs of up to 6 tokens of 64 requests over 8192 keys, 32 heads on 8 of 128, bf16: 257 us for
// 1.52 GB, 0.90.  Three short requests: 11.2 us, of which 4 lie before the first fetch (lengths, the line, the piece) and 3
// around the join.
#include <cuda.h>
#include <cuda_runtime.h>

#include "ava_math.h"
#include "bf16_hw.cuh"
#include "kernels.cuh"
#include "paged_map.cuh"
#include "read_join.cuh"
#include "read_split.cuh"
#include "serving.cuh"
#include "tc_common.cuh"

namespace ava {

namespace {

constexpr int STEP = 16;                 // keys per stage

using tcc::s32;
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
// The same with the first limb rounded towards 0: of a value near the type's largest it stays finite, and so does 0 times it
// (to nearest it would be infinite, in a place that nobody sees as well).  The other two still leave nothing over.
__device__ __forceinline__ void limbs_down(float a, float b, uint32_t (&l)[3]) {
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(l[0]) : "f"(b), "f"(a));
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

// the transpose of an 8 x 8 tile of bf16 held two to a lane
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// a word of f32, or of two bf16: whether any of it is not finite, and the word with that part 0
template <bool F32>
__device__ __forceinline__ bool not_finite(uint32_t x) {
    return (x & 0x7f800000u) == 0x7f800000u || (!F32 && (x & 0x7f80u) == 0x7f80u);
}
template <bool F32>
__device__ __forceinline__ uint32_t finite_only(uint32_t x) {
    if (F32) return not_finite<true>(x) ? 0u : x;
    return x & ~(((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u));
}

// How a warp lays out its stage: K, then V, each in columns of up to 128 bytes a key (what a TMA box with the swizzle of
// that width leaves): the 16-byte pieces of a column's row are rotated by the row, so that eight rows' equal pieces lie in
// eight bank groups.
template <typename TS, int HS>
struct Stage {
    static constexpr int ROW = HS * (int)sizeof(TS), SEG = ROW < 128 ? ROW : 128, PIECES = ROW / 16, PER_SEG = SEG / 16, POOL = STEP * ROW, BYTES = 2 * POOL;
    static __device__ __forceinline__ uint32_t at(int key, int piece) {
        const int turn = PER_SEG >= 8 ? (key & 7) : ((key >> 1) & 3);
        return (uint32_t)((piece / PER_SEG) * (STEP * SEG) + key * SEG + (((piece % PER_SEG) ^ turn) << 4));
    }
};

// tiles of MR rows, cut into stages; stretches of up to two stages (32 keys) are not cut.  (Up to eight: three requests of 64
// keys 14.6 us instead of 11.2, 200 of 100 keys 26.3 instead of 22.9: with few keys a warp's steps one after another cost more
// than joining; 256 of 1500 are the same.)
template <int NQ>
struct Plan {
    static constexpr int MR = 8 * NQ, KT = STEP, START = 2, SNAP = 2;
};

// How the keys come (box 0: by copies).
struct Coming {
    int box, heads_inside;
};

template <typename TS, int L, int HS, int NQ, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) read_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const ReadArgs a,
                                                           const Coming coming, float* __restrict__ ends, split::Cut* __restrict__ cuts, const int workers) {
    constexpr int MR = 8 * NQ, KK = HS / 16, MB = HS / 16;
    constexpr bool F32S = sizeof(TS) == 4;
    constexpr int LS = F32S ? 3 : 1;   // limbs of the store's elements
    using St = Stage<TS, HS>;
    extern __shared__ unsigned char raw[];
    unsigned char* smem = raw + ((1024u - (s32(raw) & 1023u)) & 1023u);
    __shared__ long long sums[split::ENTRIES + 1];
    __shared__ uint64_t bars[WARPS * STAGES];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tq = lane & 3;
    bool bad_length = false, bad_page = false, ok = true;
    if (threadIdx.x < WARPS * STAGES) tcc::bar_init(&bars[threadIdx.x], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    using Pl = Plan<NQ>;
    const split::Line line = split::line<Pl>(a, sums, &bad_length);   // (joins the block's threads)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (bad_length && a.status && blockIdx.x == 0) atomicOr(a.status, AVA_PAGED_BAD_LENGTH);

    const int w = blockIdx.x * WARPS + warp;
    const long long per = max((line.total() + workers - 1) / workers, 1ll);
    split::Item it = {}, after = {};
    it.r = -1;
    long long u = split::piece<Pl>(a, line, per, w, &it);
    const long long end = split::piece<Pl>(a, line, per, w + 1ll, &after, &it);
    if (lane == 0) cuts[w].workers = 0;
    unsigned char* ring = smem + warp * STAGES * St::BYTES;
    uint64_t* bar = bars + warp * STAGES;
    const uint32_t ring_at = s32(ring);
    uint32_t filled = 0;                 // stages asked for by TMA so far (their barriers' phases)
    const float scale2 = a.scale * LOG2E;
    const int page_shift = (a.s.page_size & (a.s.page_size - 1)) ? -1 : __ffs(a.s.page_size) - 1;
    const TS* pool_k = static_cast<const TS*>(a.s.k);
    const TS* pool_v = static_cast<const TS*>(a.s.v);

    while (u < end && ok) {
        const split::Share run = split::share<Pl>(it, u, end);
        const bool whole = run.whole;
        const int rows = min(it.q.f * a.group - it.tile * MR, MR);
        // this warp's keys of the stretch: from step t0 to t1 of the store's own 16-key steps
        const bool none = it.s.lo >= it.s.hi;
        const int t0 = none ? 0 : it.s.lo / STEP + run.from, t1 = none ? 0 : it.s.lo / STEP + run.to;
        const int32_t* pages = a.table + (int64_t)it.r * a.max_pages;
        const int64_t head_at = (int64_t)it.head * a.s.head_stride;
        const uint32_t first_filled = filled;

        // Where a step's keys lie.  By copies: the place of key t * 16 + (lane & 15) in the pools, -1: none.  By TMA: lane b's
        // box of the step, page * 2^32 + place.
        auto place = [&](int t) -> int64_t {
            if (coming.box) {
                const int j = t * STEP + (lane & 1) * coming.box;
                int page = a.s.n_pages, at = 0;
                if (t < t1 && (lane & 1) * coming.box < STEP && j < it.s.hi && j + coming.box > it.s.lo) {
                    const int pi = page_shift >= 0 ? j >> page_shift : j / a.s.page_size;
                    page = pages[pi];
                    at = j - pi * a.s.page_size;
                    if (page < 0 || page >= a.s.n_pages) {
                        bad_page = true;
                        page = a.s.n_pages;
                    }
                }
                return ((int64_t)page << 32) | (uint32_t)at;
            }
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
            const uint32_t slot = (unsigned)(t - t0) % STAGES, dst = ring_at + slot * St::BYTES;
            if (coming.box) {
                uint64_t* full = bar + filled % STAGES;   // (slots and barriers need not be the same ones: both turn in order)
                if (lane == 0) tcc::bar_expect(full, St::BYTES);
                __syncwarp();
                if (lane * coming.box < STEP) {           // one box of 16 keys, or two of 8
                    const int page = (int)(at >> 32), y = (int)(uint32_t)at;
#pragma unroll
                    for (int seg = 0; seg < St::ROW / St::SEG; ++seg) {
                        const uint32_t to = dst + seg * (STEP * St::SEG) + lane * coming.box * St::SEG;
                        const int x = seg * (St::SEG / (int)sizeof(TS));
                        tma_box(to, &map_k, x, coming.heads_inside ? it.head : y, coming.heads_inside ? y : it.head, page, full);
                        tma_box(to + St::POOL, &map_v, x, coming.heads_inside ? it.head : y, coming.heads_inside ? y : it.head, page, full);
                    }
                }
                ++filled;
                return;
            }
#pragma unroll
            for (int i = 0; i < St::PIECES / 2; ++i) {
                const int id = i * 32 + lane, key = id / St::PIECES, piece = id % St::PIECES;
                const int64_t from = __shfl_sync(0xffffffffu, at, key);
                const int64_t e = (from < 0 ? 0 : from) + piece * (16 / (int)sizeof(TS));
                copy16(dst + St::at(key, piece), pool_k + e, from >= 0);
                copy16(dst + St::POOL + St::at(key, piece), pool_v + e, from >= 0);
            }
        };
        __syncwarp();   // the stretch before has been read out of the ring by every lane
        int64_t ahead_at = -1;
        if (t0 < t1) {
            int64_t at = place(t0);
#pragma unroll 1
            for (int s = 0; s < STAGES - 1; ++s) {
                const int64_t next_at = place(t0 + s + 1);
                if (t0 + s < t1) fetch(t0 + s, at);
                asm volatile("cp.async.commit_group;" ::: "memory");
                at = next_at;
            }
            ahead_at = at;
        }

        // queries: column 8 nq + g of the tile (B operand: channels 16 kk + 2 tq (+ 8)); a lane's scores are of columns 2 tq, 2 tq + 1
        uint32_t qf[NQ][KK][2][L];
        int pos[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
                pos[nq][half] = it.q.c + (it.tile * MR + min(8 * nq + 2 * tq + half, rows - 1)) / a.group;   // columns beyond the last repeat it: no mask of their own
            const int m = it.tile * MR + min(8 * nq + g, rows - 1), i = m / a.group, h = it.head * a.group + (m - i * a.group);
            const int64_t at = (int64_t)(it.q.start + i) * a.q_token_stride + (int64_t)h * a.q_head_stride;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const int64_t e = at + 16 * kk + 8 * o + 2 * tq;
                    if constexpr (L == 3) {
                        const float* q = static_cast<const float*>(a.q) + e;
                        limbs(q[0], q[1], qf[nq][kk][o]);
                    } else {
                        const uint16_t* q = static_cast<const uint16_t*>(a.q) + e;
                        qf[nq][kk][o][0] = q[0] | ((uint32_t)q[1] << 16);
                    }
                }
        }

        float acc[NQ][MB][4], top[NQ][2], sum[NQ][2];   // acc: channels 16 mb + g (+ 8) of columns 2 tq, 2 tq + 1
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            top[nq][0] = top[nq][1] = -INFINITY;
            sum[nq][0] = sum[nq][1] = 0.0f;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[nq][mb][i] = 0.0f;
        }
        // keys that every row of the tile sees need no comparison
        const int all_from = a.window > 0 ? max(it.q.first, it.q.c + (it.tile * MR + rows - 1) / a.group + 1 - a.window) : it.q.first;
        const int all_to = it.q.c + (it.tile * MR) / a.group + 1;

#pragma unroll 1
        for (int t = t0; t < t1; ++t) {
            if (coming.box) {
                const uint32_t n = first_filled + (unsigned)(t - t0);
                ok = __all_sync(0xffffffffu, tcc::bar_wait(bar + n % STAGES, (n / STAGES) & 1));
                if (!ok) break;
            } else {
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
                __syncwarp();
            }
            {   // the stage read last is free: the step STAGES - 1 ahead goes into it
                const int ahead = t + STAGES - 1;
                if (ahead < t1) fetch(ahead, ahead_at);
                asm volatile("cp.async.commit_group;" ::: "memory");
                ahead_at = place(ahead + 1);
            }
            const uint32_t at_k = ring_at + (uint32_t)(((unsigned)(t - t0) % STAGES) * St::BYTES), at_v = at_k + St::POOL;
            unsigned char* st = ring + (at_k - ring_at);
            const int j0 = t * STEP;
            if (coming.box && (j0 < it.s.lo || j0 + STEP > it.s.hi)) {   // rows of V that are no key of the stretch
                for (int e = lane; e < STEP * St::PIECES; e += 32) {
                    const int key = e / St::PIECES;
                    if (j0 + key < it.s.lo || j0 + key >= it.s.hi) *reinterpret_cast<uint4*>(st + St::POOL + St::at(key, e % St::PIECES)) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the next copy into this stage comes after
                __syncwarp();
            }

            float s[NQ][4], sl[NQ][4];   // leading products, the others: keys g, g + 8 of columns 2 tq, 2 tq + 1
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nq][i] = sl[nq][i] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                uint32_t kf[LS][4];      // keys x channels: (g, 2 tq), (g + 8, 2 tq), (g, 2 tq + 8), (g + 8, 2 tq + 8)
                if constexpr (F32S) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int ch = 16 * kk + 8 * (i >> 1) + 2 * tq;
                        const float2 x = *reinterpret_cast<const float2*>(st + St::at(g + 8 * (i & 1), ch / 4) + (ch & 3) * 4);
                        uint32_t l[LS];
                        limbs(x.x, x.y, l);
#pragma unroll
                        for (int y = 0; y < LS; ++y) kf[y][i] = l[y];
                    }
                } else {
                    ldmatrix4(at_k + St::at((lane & 7) + 8 * ((lane >> 3) & 1), 2 * kk + (lane >> 4)), kf[0]);
                }
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) mma_limbs(s[nq], sl[nq], kf, qf[nq][kk][0], qf[nq][kk][1]);
            }
            // scores in units of log2: hidden keys to -infinity, the running maximum, the weights
            const bool edge = j0 < all_from || j0 + STEP > all_to;
            uint32_t wf[NQ][2][L];       // weights as the other operand: keys 2 tq, 2 tq + 1 (+ 8) of column g
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nq][i] = (L == 3 ? s[nq][i] + sl[nq][i] : s[nq][i]) * scale2;
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = j0 + g + 8 * (i >> 1), p = pos[nq][i & 1];
                        if (j > p || j < it.q.first || (a.window > 0 && j <= p - a.window)) s[nq][i] = -INFINITY;
                    }
                }
                const float high[2] = {fmaxf(s[nq][0], s[nq][2]), fmaxf(s[nq][1], s[nq][3])};
                if (__any_sync(0xffffffffu, high[0] > top[nq][0] || high[1] > top[nq][1])) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float x = high[half];
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                        x = fmaxf(x, top[nq][half]);
                        const float f = top[nq][half] == -INFINITY ? 0.0f : exp2_fast(top[nq][half] - x);
                        top[nq][half] = x;
                        sum[nq][half] *= f;
#pragma unroll
                        for (int mb = 0; mb < MB; ++mb) {
                            acc[nq][mb][half] *= f;
                            acc[nq][mb][2 + half] *= f;
                        }
                    }
                }
                const float base[2] = {top[nq][0] == -INFINITY ? 0.0f : top[nq][0], top[nq][1] == -INFINITY ? 0.0f : top[nq][1]};
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const float x = exp2_fast(s[nq][2 * o] - base[0]), y = exp2_fast(s[nq][2 * o + 1] - base[1]);
                    sum[nq][0] += x;
                    sum[nq][1] += y;
                    uint32_t l[L];
                    limbs(x, y, l);
#pragma unroll
                    for (int i = 0; i < L; ++i) wf[nq][o][i] = transposed(l[i]);
                }
            }
            if (edge) {   // a weight of 0 times a value that is not finite must be 0: such values are taken out and added where they are seen
                unsigned keys = 0;
#pragma unroll 1
                for (int e = lane; e < STEP * St::PIECES; e += 32) {
                    const uint4 x = *reinterpret_cast<const uint4*>(st + St::POOL + St::at(e / St::PIECES, e % St::PIECES));
                    if (not_finite<F32S>(x.x) || not_finite<F32S>(x.y) || not_finite<F32S>(x.z) || not_finite<F32S>(x.w)) keys |= 1u << (e / St::PIECES);
                }
                keys = __reduce_or_sync(0xffffffffu, keys);
                if (keys) {
#pragma unroll 1
                    for (unsigned left = keys; left; left &= left - 1) {
                        const int key = __ffs(left) - 1;
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const float x = __shfl_sync(0xffffffffu, key < 8 ? s[nq][half] : s[nq][2 + half], (key & 7) * 4 + tq);
#pragma unroll
                                for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                                    for (int o = 0; o < 2; ++o) {
                                        const int ch = 16 * mb + 8 * o + g;
                                        const unsigned char* at = st + St::POOL + St::at(key, ch * (int)sizeof(TS) / 16) + ch * (int)sizeof(TS) % 16;
                                        float v;
                                        if constexpr (F32S) v = *reinterpret_cast<const float*>(at);
                                        else v = bf16_to_f(*reinterpret_cast<const uint16_t*>(at));
                                        if (x > -INFINITY && !(fabsf(v) < INFINITY)) acc[nq][mb][2 * o + half] += v;
                                    }
                            }
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int e = lane; e < STEP * St::PIECES; e += 32) {
                        uint4* at = reinterpret_cast<uint4*>(st + St::POOL + St::at(e / St::PIECES, e % St::PIECES));
                        uint4 x = *at;
                        x.x = finite_only<F32S>(x.x);
                        x.y = finite_only<F32S>(x.y);
                        x.z = finite_only<F32S>(x.z);
                        x.w = finite_only<F32S>(x.w);
                        *at = x;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the next copy into this stage comes after
                    __syncwarp();
                }
            }
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                uint32_t vf[LS][4];      // channels x keys: (g, 2 tq), (g + 8, 2 tq), (g, 2 tq + 8), (g + 8, 2 tq + 8)
                if constexpr (F32S) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int ch = 16 * mb + 8 * (i & 1) + g, key = 8 * (i >> 1) + 2 * tq;
                        const unsigned char* v = st + St::POOL + (ch & 3) * 4;
                        uint32_t l[LS];
                        limbs_down(*reinterpret_cast<const float*>(v + St::at(key, ch / 4)), *reinterpret_cast<const float*>(v + St::at(key + 1, ch / 4)), l);
#pragma unroll
                        for (int y = 0; y < LS; ++y) vf[y][i] = l[y];
                    }
                } else {
                    ldmatrix4_trans(at_v + St::at((lane & 7) + 8 * (lane >> 4), 2 * mb + ((lane >> 3) & 1)), vf[0]);
                }
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) {
                    if constexpr (L == 3) {
                        float high[4] = {0.0f, 0.0f, 0.0f, 0.0f}, low[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_limbs(high, low, vf, wf[nq][0], wf[nq][1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[nq][mb][i] += high[i] + low[i];
                    } else {
                        mma16816(acc[nq][mb], vf[0], wf[nq][0][0], wf[nq][1][0]);
                    }
                }
            }
            __syncwarp();   // every lane has read the stage: the next copies may go into it
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (!ok) break;

        // the rows' sums over the lanes that share a column, then the read itself or this piece's end of it
        float* part = ends + ((int64_t)w * 2 + (u == it.begin ? 1 : 0)) * Ends<HS, MR>::FLOATS;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float l = sum[nq][half];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                const int row = 8 * nq + 2 * tq + half;
                if (row >= rows) continue;
                if (whole) {
                    const float inv = l > 0.0f ? 1.0f / l : l;   // a sum that is NaN stays NaN
                    const int m = it.tile * MR + row, i = m / a.group, h = it.head * a.group + (m - i * a.group);
                    const int64_t to = (int64_t)(it.q.start + i) * a.out_token_stride + (int64_t)h * a.out_head_stride + g;
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const float x = acc[nq][mb][2 * o + half] * inv;
                            if constexpr (L == 1) static_cast<uint16_t*>(a.out)[to + 16 * mb + 8 * o] = bf16_rn_hw(x);
                            else static_cast<float*>(a.out)[to + 16 * mb + 8 * o] = x;
                        }
                    if (a.lse && g == 0) a.lse[(int64_t)(it.q.start + i) * a.heads + h] = l == 0.0f ? -INFINITY : (top[nq][half] + log2f(l)) * LN2;
                } else {
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                        for (int o = 0; o < 2; ++o) part[row * HS + 16 * mb + 8 * o + g] = acc[nq][mb][2 * o + half];
                    if (g == 0) {
                        part[MR * HS + row] = top[nq][half];
                        part[MR * HS + MR + row] = l;
                    }
                }
            }
        if (!whole && u == it.begin && lane == 0) {
            cuts[w].start = it.q.start;
            cuts[w].head = it.head;
            cuts[w].tile = it.tile;
            cuts[w].rows = rows;
            cuts[w].workers = (int)split::last_worker<Pl>(it, per) - w + 1;
        }
        u = run.stop;
        if (u < end) split::next<Pl>(a, it);
    }
    if (!ok) {   // the copies in flight end before the warp does
        for (uint32_t back = 1; back <= STAGES && back <= filled; ++back) tcc::bar_wait(bar + (filled - back) % STAGES, ((filled - back) / STAGES) & 1);
        if (lane == 0 && a.status) atomicOr(a.status, AVA_PAGED_WAIT_RAN_OUT);
    }
    if (__any_sync(0xffffffffu, bad_page) && lane == 0 && a.status) atomicOr(a.status, AVA_PAGED_BAD_PAGE);
}

// Joins the ends of the stretches that were cut (read_join.cuh): one block per worker, idle unless a cut stretch begins in its
// piece.  A warp takes a row; stretches of many parts (a long sequence) have the block's warps share a row's parts.
constexpr int JOIN_WARPS = 8, SHARED_PARTS = 16;
template <int HS, int MR>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const ReadArgs a, const float* __restrict__ ends, const split::Cut* __restrict__ cuts) {
    pdl_enter();
    const int w = blockIdx.x;
    const split::Cut cut = cuts[w];
    const int n = cut.workers;
    if (n == 0) return;
    constexpr int PER = HS / 32;
    __shared__ float part_o[JOIN_WARPS][HS], part_m[JOIN_WARPS], part_l[JOIN_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m, l, o[PER];
    if (n <= SHARED_PARTS) {
        for (int row = warp; row < cut.rows; row += JOIN_WARPS) {
            join_parts<HS, MR>(ends, w, row, n, 0, 1, m, l, o);
            join_write<HS>(a, cut.start, cut.head, cut.tile * MR + row, m, l, o);
        }
        return;
    }
    for (int row = 0; row < cut.rows; ++row) {
        join_parts<HS, MR>(ends, w, row, n, warp, JOIN_WARPS, m, l, o);
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
            join_write<HS>(a, cut.start, cut.head, cut.tile * MR + row, m, l, o);
        }
        __syncthreads();
    }
}

// Warps of a block: as many as registers allow (16 columns of queries leave room for twelve, 32 for eight; 16 warps with three stages each were slower), and
// the ring's stages share what is left of 192 KB.
constexpr int most_warps(int stage_bytes, int nq) { return nq > 2 ? 8 : stage_bytes <= 4096 ? 12 : stage_bytes <= 8192 ? 8 : 6; }
constexpr int most_stages(int stage_bytes, int nq) { return 196608 / (most_warps(stage_bytes, nq) * stage_bytes); }

template <typename TS, int L, int HS, int NQ>
cudaError_t launch_one(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms) {
    constexpr int BYTES = Stage<TS, HS>::BYTES, WARPS = most_warps(BYTES, NQ), STAGES = most_stages(BYTES, NQ), MR = 8 * NQ;
    const int workers = sms * WARPS;
    split::Cut* cuts = static_cast<split::Cut*>(room);
    float* ends = reinterpret_cast<float*>(cuts + workers);
    // by TMA where the store is a tensor for it and 16 keys are one box or two
    Coming coming{a.s.page_size == 8 ? 8 : a.s.page_size % STEP == 0 ? STEP : 0, 0};
    CUtensorMap mk = {}, mv = {};
    PoolShape shape;
    if (coming.box && (!pool_shape(a.s, &shape) || !pool_map(&mk, a.s.k, a.s.dtype, shape, coming.box) || !pool_map(&mv, a.s.v, a.s.dtype, shape, coming.box))) coming.box = 0;
    coming.heads_inside = coming.box && shape.heads_inside;
    cudaError_t rc = launch_serving<read_kernel<TS, L, HS, NQ, WARPS, STAGES>>(device, dim3(sms), dim3(WARPS * 32), (size_t)WARPS * STAGES * BYTES + 1024, st, 1, mk, mv, a, coming, ends,
                                    cuts, workers);
    if (rc != cudaSuccess) return rc;
    return launch_serving<join_kernel<HS, MR>>(device, dim3(workers), dim3(JOIN_WARPS * 32), 0, st, 1, a, ends, cuts);
}

template <typename TS, int L, int HS>
cudaError_t launch_rows(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms) {
    // Rows per key head that the host expects: a tile of 8, 16 or 32 of them reads the store once (three limbs of 128
    // channels stay in registers for 16).
    const int64_t rows = (int64_t)a.max_fresh * a.group;
    if (rows <= 8) return launch_one<TS, L, HS, 1>(device, st, a, room, sms);
    if constexpr (HS < 128 || L == 1) {
        if (rows > 24) return launch_one<TS, L, HS, 4>(device, st, a, room, sms);
        if (rows > 16) return launch_one<TS, L, HS, 3>(device, st, a, room, sms);
    }
    return launch_one<TS, L, HS, 2>(device, st, a, room, sms);
}
template <int HS>
cudaError_t launch_size(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms) {
    if (a.bf16_q) return launch_rows<uint16_t, 1, HS>(device, st, a, room, sms);
    if (a.s.dtype == AVA_BF16) return launch_rows<uint16_t, 3, HS>(device, st, a, room, sms);
    return launch_rows<float, 3, HS>(device, st, a, room, sms);
}

}  // namespace

int64_t paged_read_workspace(int head_size, int sms) {
    // at most 16 workers on an SM, and at most 256 rows of their tiles (most_warps times 8, 16 or 32; k_pread_tc.cu: 256)
    return (int64_t)sms * 16 * (int64_t)sizeof(split::Cut) + (int64_t)sms * 256 * 2 * (head_size + 2) * 4;
}

cudaError_t launch_paged_read(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms) {
    bool taken = false;
    const cudaError_t rc = launch_paged_read_tc(device, st, a, room, sms, &taken);
    if (taken || rc != cudaSuccess) return rc;
    if (a.s.head_size == 32) return launch_size<32>(device, st, a, room, sms);
    if (a.s.head_size == 64) return launch_size<64>(device, st, a, room, sms);
    return launch_size<128>(device, st, a, room, sms);
}

}  // namespace ava
