// The read of new tokens over a bf16 store in pages when a request brings many rows per key head (prompt chunks, drafted
// runs with shared key heads): the same o = sum_j softmax_j(scale q . k_j) v_j on tcgen05 tensor cores.
//
// A block is a worker of read_split.cuh with tiles of 256 rows and units of KT keys; its piece of the line is walked
// stretch by stretch.  Per unit and 128-row tile: S = Q K^T into tensor memory (Q and K from shared memory), one thread per
// row turns its row of S into weights with a running maximum and sum, and writes them over S as the bf16 operand of
// O += P V (P from tensor memory, V from shared memory as it arrived, keys down: the multiply takes it that way).  O stays
// in tensor memory; it is rescaled only when a row's maximum has grown by more than 2^8, so almost never after the first
// units.  Two groups of 128 threads work on half a tile each: while one turns its scores into weights the tensor cores
// multiply for the other.
// Keys and values come by TMA, a box per page and 64 channels, a unit of both to a slot of one ring; a page outside the store,
// or past the stretch, is a coordinate past the tensor's last page, which TMA fills with zeros without reading.
// A weight of 0 times whatever lies in a hidden place must be 0.  So a warp goes over the units that some row sees only in
// part before they are multiplied: rows of V in front of the stretch or behind it (the rest of a page, left padding) become
// zeros, and so do values that are not finite (a later token's, which earlier rows do not see); the rows that do see
// those get them added behind the multiplies.
// With f32 queries Q and P are three bf16 limbs each (L 3): three products per step instead of one.
//
// P is written over its S.  Each group has two such places, so the scores of the next 64 keys are made while this step's are
// turned into weights; a place is taken again once the completion of its P V has been seen (multiplies into different
// accumulators are not ordered by their issue).  Each group has an issuing warp of its own that waits where it must; one
// warp polling for both took 1500 cycles a round of its own code.
// Measured (one B200): 4 chunks of up to 2048 tokens over 8192 keys, 32 heads on 8 key heads of 128, bf16: 555 us, 1.05
// PFLOP/s, 0.64 of the measured bf16 rate; what bounds it is the latency of the row threads' chain, of which a scheduler has
// two warps (it issues in 0.41 of the cycles; a unit of 64 keys of both groups: 1280 cycles of multiplies, about 1900 in all; a
// quarter of the exponentials as polynomials in f32 arithmetic made it 15 us slower, so it is not the exponential unit).
// 16 chunks of up to 1024 over 2048 keys, 12 heads of 64, f32 queries: 211 us, three products for each of the 38 GFLOP;
// bounded by the same chain, longer by the limbs.  In both the code
// a tile runs once costs about five cycles an instruction (it is not in the instruction caches by then), hence the small
// loops around queries and results and one piece of code for every wait: 213 KB of code and 250 us before, 120 KB and 211 us.
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

using namespace tcc;

constexpr int THREADS = 384;             // two groups of 128 rows, a warp per group that issues multiplies, the copies' warp, the sweeping one
constexpr uint32_t PLACES = 2;           // of scores and weights, per group
struct Plan {                            // of the line: a tile's queries and results take as long as some units (4: 225 and 587 us, 8: 215 and
                                         // 582 us for 16 x 1024 and 4 x 2048 new tokens)
    static constexpr int MR = 256, KT = 64, START = 8, SNAP = 4;
};
constexpr int MR = Plan::MR, KT = Plan::KT;
constexpr float GROWN = 8.0f;            // powers of two a maximum may grow by before the sums are rescaled

// Units of a run in which values that are not finite were taken out of V: their keys.  A run can have at most so many units
// that some row sees in part (the diagonal's and a window's other end); the sweeping warp is at most as many runs ahead of
// the rows as the ring has units.
struct Found {
    int count;
    int unit[15];
    uint64_t keys[15];
};
constexpr uint32_t RUNS = 16;
constexpr uint32_t ROWS_ROOM = 2048;     // bytes

template <int HS_, int L_>
struct Shape {
    static constexpr int HS = HS_, L = L_;
    static constexpr int HALVES = HS / 64;                           // 64-channel columns of 128 bytes a row
    static constexpr uint32_t Q_LIMB = 128 * HS * 2, Q_TILE = L * Q_LIMB, KV = KT * HS * 2;
    static constexpr uint32_t RING = HS == 64 ? (L == 1 ? 10 : 6) : 4;   // units in shared memory
    static constexpr uint32_t OFF_K = 2 * Q_TILE, OFF_V = OFF_K + RING * KV, OFF_BAR = OFF_V + RING * KV;
    static constexpr uint32_t OFF_FOUND = OFF_BAR + 768;             // Found[RUNS]
    static constexpr uint32_t OFF_ROWS = (OFF_FOUND + RUNS * (uint32_t)sizeof(Found) + 127) / 128 * 128;   // put_rows' room, ROWS_ROOM for each row warp
    static constexpr uint32_t BYTES = OFF_ROWS + 8 * ROWS_ROOM + 1024;   // the rest: alignment to 1024
    // Tensor memory of a group: places of scores and weights, the mix.  A place's scores are read a chunk at a time and the
    // weights go back over it: the first limb in its first half, the second in the second, the third outside.
    static __device__ __forceinline__ uint32_t weights_at(int l, int c) { return l == 2 ? 64 + c / 2 : c + CW / 2 * l; }   // of the chunk of keys from c on
    // Chunks of CW columns.  The tensor cores' f32 sums are cut, not rounded, at every addition (one sum over 2048 keys and
    // three limbs lost 2e-6 of the read, always towards 0): with f32 queries the mix of every FLUSH units is added up in
    // registers, and of the limbs the small ones go first.
    static constexpr int CW = L == 3 ? 16 : 32, FLUSH = L == 3 ? 2 : 0;
    static constexpr uint32_t PLACE = L == 3 ? 96 : 64, C_O = PLACES * PLACE, GROUP = 256;
    static_assert(C_O + HS <= GROUP, "tensor memory");   // (three limbs of 128 channels do not fit, nor do their queries: k_pread.cu takes them)
    static_assert(BYTES <= 232448, "shared memory");
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_half(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
// two f32 operations in one instruction
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void apart(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// the next limb of a pair: bf16 of it, and what that leaves over
__device__ __forceinline__ uint32_t limb(uint64_t& x) {
    float a, b;
    apart(x, a, b);
    const uint32_t p = pack_bf16(a, b);
    x = fma2(two(low_half(p), high_half(p)), two(-1.0f, -1.0f), x);
    return p;
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(bar)) : "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(bar)) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_read(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 16) tmem_ld16(taddr, r);
    else tmem_ld32(taddr, r);
}
template <int N>
__device__ __forceinline__ void tmem_write(uint32_t taddr, const uint32_t (&r)[N]) {
    if constexpr (N == 8) tmem_st8(taddr, r);
    else tmem_st16(taddr, r);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    tmem_st16(taddr, r);
    tmem_st16(taddr + 16, r + 16);
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// V as it lies, [key][64 channels] with the 128-byte swizzle, for a multiply that wants it [channel][key]: 64 channels
// adjacent, 8 keys to 1024 bytes; `group` bytes from one 64-channel column to the next
__device__ __forceinline__ uint64_t desc_keys_down(uint32_t at, uint32_t group) {
    uint64_t d = 0;
    d |= (uint64_t)((at & 0x3FFFFu) >> 4);
    d |= (uint64_t)(group >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

struct Bars {
    uint64_t full[10], empty[10], passed[10], q_ready[2], s_ready[2][2], p_ready[2][2], pv_done[2][2], o_free[2], drained[2];
    uint32_t tmem, failed;
};
static_assert(sizeof(Bars) <= 768, "barriers");

// A wait that ends: true when the phase is there, false when it ran out here or anywhere in the block.  The first look is made
// in place; the waiting itself is one piece of code for all (in every place it was a third of the kernel's code).
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, volatile uint32_t* failed) {
    const uint32_t addr = s32(bar);
#pragma unroll 1
    for (uint32_t i = 0; i < B_WAIT_LIMIT; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(addr), "r"(parity)
            : "memory");
        if (done) return true;
        if (i > 64) {
            if (*failed) return false;
            if (i > 1024) __nanosleep(32);
        }
    }
    *failed = 1;
    return false;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile uint32_t* failed) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(s32(bar)), "r"(parity)
        : "memory");
    return done ? true : wait_slow(bar, parity, failed);
}
// one lane of a whole warp
__device__ __forceinline__ bool elected() {
    uint32_t yes = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "@p mov.u32 %0, 1;\n\t}"
        : "+r"(yes));
    return yes != 0;
}
// The same for a whole warp.  (One lane asking for the others, or one lane's branch around waits and multiplies, made the
// chunk of 16 x 1024 rows 1.4 times slower: multiplies are issued fast only from code that the whole warp runs.)
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* failed) {
    return __all_sync(0xffffffffu, wait(bar, parity, failed));
}
// A warp's arrival: what its lanes have done is done.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(bar);
}

// A worker's run over one stretch: units [ta, tb) of the store's own KT-key units, and of them [a, b) for the rows of group w.
struct Run {
    long long stop;
    bool whole;
    int ta, tb, rows;
    int a, b;
    __device__ __forceinline__ int count() const { return max(b - a, 0); }
    int all_from, all_to;                // keys that every row of the tile sees
    // whether the sweeping warp goes over unit t: some row does not see all of it
    __device__ __forceinline__ bool swept(int t) const { return t * KT < all_from || t * KT + KT > all_to; }
};
__device__ __forceinline__ Run run_of(const ReadArgs& a, const split::Item& it, long long u, long long end, int w) {
    Run r;
    const split::Share s = split::share<Plan>(it, u, end);
    r.stop = s.stop;
    r.whole = s.whole;
    const bool none = it.s.lo >= it.s.hi;
    r.ta = none ? 0 : it.s.lo / KT + s.from;
    r.tb = none ? 0 : it.s.lo / KT + s.to;
    r.rows = min(it.q.f * a.group - it.tile * MR, MR);
    r.all_to = it.q.c + it.tile * MR / a.group + 1;
    r.all_from = a.window > 0 ? max(it.q.first, it.q.c + (it.tile * MR + r.rows - 1) / a.group + 1 - a.window) : it.q.first;
    r.a = r.b = r.ta;
    if (r.rows > 128 * w) {   // the keys that this group's rows see
        const int m0 = it.tile * MR + 128 * w, m1 = it.tile * MR + min(r.rows, 128 * w + 128) - 1;
        const int hi = it.q.c + m1 / a.group + 1, lo = a.window > 0 ? max(it.q.first, it.q.c + m0 / a.group + 1 - a.window) : it.q.first;
        if (lo < hi) {
            r.a = max(r.ta, lo / KT);
            r.b = min(r.tb, (hi + KT - 1) / KT);
        }
    }
    return r;
}

__device__ __forceinline__ void next_item(const ReadArgs& a, split::Item& it) { split::next<Plan>(a, it); }

// PIECES 16-byte pieces of a row per lane, as stores whose lanes lie next to one another: through the warp's shared memory.
// (A lane storing its own row touches 32 lines with every 16 bytes; the results of a tile took 4100 cycles of the block's
// load and store unit that way, 1000 this way, and its queries as many.)  at: where the lane's row begins, in bytes; rows: that are stored.
template <int PIECES>
__device__ __forceinline__ void put_rows(unsigned char* room, const uint32_t (&x)[4 * PIECES], unsigned char* base, int64_t at, int rows, bool wide, int element) {
    constexpr int ROW = 16 * PIECES, ROWS = (int)ROWS_ROOM / ROW;
    const int lane = threadIdx.x & 31;
    auto turned = [](int row, int piece) { return row * ROW + ((piece ^ (PIECES == 8 ? row & 7 : (row >> 1) & 3)) << 4); };
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += ROWS) {
        if (lane / ROWS * ROWS == r0) {
#pragma unroll
            for (int k = 0; k < PIECES; ++k) *reinterpret_cast<uint4*>(room + turned(lane % ROWS, k)) = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < ROWS * PIECES / 32; ++i) {
            const int row = (i * 32 + lane) / PIECES, piece = lane % PIECES;
            const uint4 y = *reinterpret_cast<const uint4*>(room + turned(row, piece));
            unsigned char* to = base + __shfl_sync(0xffffffffu, at, r0 + row) + piece * 16;
            if (r0 + row >= rows) continue;
            if (wide) {
                *reinterpret_cast<uint4*>(to) = y;
            } else {
                const unsigned char* from = room + turned(row, piece);
#pragma unroll 1
                for (int k = 0; k < 16; k += element) {
                    if (element == 4) *reinterpret_cast<uint32_t*>(to + k) = *reinterpret_cast<const uint32_t*>(from + k);
                    else *reinterpret_cast<uint16_t*>(to + k) = *reinterpret_cast<const uint16_t*>(from + k);
                }
            }
        }
        __syncwarp();
    }
}

// Adds what the sweeping warp has taken out of V to a row that sees it, in its results or in its end (the warp's own
// writes): an infinity or a NaN is what its mix then is.
template <int HS>
__device__ __noinline__ void add_found(const ReadArgs& a, int r, int head, const volatile Found* found, int low, int pos, int from, int to, float* end, int64_t out_at) {
    const int32_t* pages = a.table + (int64_t)r * a.max_pages;
    for (int f = 0; f < found->count; ++f) {
        const int t = found->unit[f];
        if (t < from || t >= to) continue;
        for (uint64_t keys = found->keys[f]; keys; keys &= keys - 1) {
            const int j = t * KT + __ffsll((long long)keys) - 1;
            if (j < low || j > pos) continue;
            const int page = pages[j / a.s.page_size];
            if (page < 0 || page >= a.s.n_pages) continue;
            const uint16_t* v = static_cast<const uint16_t*>(a.s.v) + page * a.s.page_stride + head * a.s.head_stride + (j % a.s.page_size) * a.s.place_stride;
#pragma unroll 1
            for (int c = 0; c < HS; ++c) {
                if ((v[c] & 0x7f80u) != 0x7f80u) continue;
                const float x = bf16_to_f(v[c]);
                if (end) end[c] += x;
                else if (a.bf16_q) static_cast<uint16_t*>(a.out)[out_at + c] = f_to_bf16(bf16_to_f(static_cast<uint16_t*>(a.out)[out_at + c]) + x);
                else static_cast<float*>(a.out)[out_at + c] += x;
            }
        }
    }
}

template <typename Sh>
__global__ void __launch_bounds__(THREADS, 1) read_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ReadArgs a,
                                                            const int heads_inside, const int box_rows, float* __restrict__ ends, split::Cut* __restrict__ cuts) {
    constexpr int HS = Sh::HS, L = Sh::L;
    constexpr uint32_t RING = Sh::RING;
    constexpr int CW = Sh::CW, FLUSH = Sh::FLUSH;
    extern __shared__ unsigned char raw[];
    unsigned char* smem = raw + ((1024u - (s32(raw) & 1023u)) & 1023u);
    const uint32_t at0 = s32(smem);
    Bars* bars = reinterpret_cast<Bars*>(smem + Sh::OFF_BAR);
    volatile uint32_t* failed = &bars->failed;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_enter();
    // this block's piece of the line (the sums lie where the copies will)
    bool bad_length = false;
    const split::Line line = split::line<Plan>(a, reinterpret_cast<long long*>(smem + Sh::OFF_K), &bad_length);
    if (bad_length && a.status && blockIdx.x == 0) atomicOr(a.status, AVA_PAGED_BAD_LENGTH);
    const int worker = blockIdx.x;
    const long long per = max((line.total() + gridDim.x - 1) / (long long)gridDim.x, 1ll);
    split::Item it = {};
    it.r = -1;
    long long u = 0, end = 0;
#pragma unroll 1
    for (int k = 1; k >= 0; --k) {           // where the piece ends, then where it begins
        end = u;
        const split::Item known = it;
        u = split::piece<Plan>(a, line, per, worker + k, &it, &known);
    }
    if (tid == 0) {
        cuts[worker].workers = 0;
        for (uint32_t i = 0; i < RING; ++i) {
            bar_init(&bars->full[i], 1);
            bar_init(&bars->empty[i], 3);     // each group has used it or passed it over, the sweeping warp has been there
            bar_init(&bars->passed[i], 1);
        }
        for (int w = 0; w < 2; ++w) {
            bar_init(&bars->q_ready[w], 4);   // a group's warps
            for (uint32_t i = 0; i < PLACES; ++i) {
                bar_init(&bars->s_ready[w][i], 1);
                bar_init(&bars->p_ready[w][i], 4);
                bar_init(&bars->pv_done[w][i], 1);
            }
            bar_init(&bars->o_free[w], 4);
            bar_init(&bars->drained[w], 1);
        }
        bars->failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_async();   // the sums were written where copies will be
    __syncwarp();
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&bars->tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = bars->tmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    bool ok = true;

    if (warp < 8) {
        // ---- one row per thread
        const int w = warp >> 2, row = tid & 127, q_row = w * 128 + row;   // row within the block's tile
        const uint32_t mine = tmem + w * Sh::GROUP + ((uint32_t)((warp & 3) * 32) << 16);
        const float scale2 = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * LOG2E;   // its sign is in the queries
        const bool out_wide = !((reinterpret_cast<uintptr_t>(a.out) & 15) || (a.out_token_stride % (L == 3 ? 4 : 8)) || (a.out_head_stride % (L == 3 ? 4 : 8)));
        uint32_t n_p = 0, runs = 0;      // units of this group so far: its barriers' phases; runs with units
        // A run's queries into the operand layout, the warp's 32 rows together, lanes next to one another reading a row.  They are
        // brought as soon as the scores of the run before are made, in front of its epilogue, so that the first scores of the
        // next run are ready behind it.  All of it in small loops: code that runs once a tile comes from beyond the instruction
        // caches, some five cycles an instruction, and a straight-line form took 7000 cycles a tile.
        constexpr int EL = L == 3 ? 4 : 2, CH = 16 / EL, PIECES = HS / CH;   // channels in 16 bytes, pieces of a row
        const bool q_wide = !((reinterpret_cast<uintptr_t>(a.q) & 15) || (a.q_token_stride % CH) || (a.q_head_stride % CH));
        // the scale's sign goes into the queries, so that the largest score is the largest product; a scale of 0 empties them
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u, keep = a.scale == 0.0f ? 0u : 0xffffffffu;
        auto bring = [&](const split::Item& of, const Run& run) {
            const int m = of.tile * MR + min(q_row, run.rows - 1), i = m / a.group, h = of.head * a.group + (m - i * a.group);
            const int64_t mine_from = ((int64_t)(of.q.start + i) * a.q_token_stride + (int64_t)h * a.q_head_stride) * EL;
            const int piece = lane % PIECES, r0 = (warp & 3) * 32;
            // 16 bytes of a row where they will be multiplied from; f32 ones in the first two limbs' places
            unsigned char* to = smem + w * Sh::Q_TILE + (piece / 8) * (L == 3 ? (int)Sh::Q_LIMB : 128 * 128);
            const unsigned char* q = static_cast<const unsigned char*>(a.q) + piece * 16;
#pragma unroll 1
            for (int k = 0; k < PIECES; ++k) {
                const int row = (k * 32 + lane) / PIECES;
                const unsigned char* from = q + __shfl_sync(0xffffffffu, mine_from, row);
                unsigned char* at = to + swz128(r0 + row, 8 * (piece % 8));
                if (q_wide) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s32(at)), "l"(from) : "memory");
                } else {
#pragma unroll 1
                    for (int b = 0; b < 16; b += EL) {
                        if (EL == 4) *reinterpret_cast<uint32_t*>(at + b) = *reinterpret_cast<const uint32_t*>(from + b);
                        else *reinterpret_cast<uint16_t*>(at + b) = *reinterpret_cast<const uint16_t*>(from + b);
                    }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if constexpr (L == 3) {
                unsigned char* limbs_at = smem + w * Sh::Q_TILE;
#pragma unroll 1
                for (int k = 0; k < PIECES; k += 2) {   // four rows at a time: all of them read, then their limbs written over them
                    uint4 x[2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) x[z] = *reinterpret_cast<const uint4*>(to + swz128(r0 + ((k + z) * 32 + lane) / PIECES, 8 * (piece % 8)));
                    __syncwarp();
                    uint64_t y[2][2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        y[z][0] = two(__uint_as_float(x[z].x), __uint_as_float(x[z].y));
                        y[z][1] = two(__uint_as_float(x[z].z), __uint_as_float(x[z].w));
                    }
#pragma unroll
                    for (int l = 0; l < L; ++l)
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            unsigned char* at = limbs_at + l * Sh::Q_LIMB + swz128(r0 + ((k + z) * 32 + lane) / PIECES, 8 * (piece / 2)) + (piece & 1) * 8;
                            const uint32_t p0 = (limb(y[z][0]) ^ sign) & keep, p1 = (limb(y[z][1]) ^ sign) & keep;
                            *reinterpret_cast<uint2*>(at) = make_uint2(p0, p1);
                        }
                }
            } else if (sign || !keep) {
#pragma unroll 1
                for (int k = 0; k < PIECES; ++k) {
                    uint4* at = reinterpret_cast<uint4*>(to + swz128(r0 + (k * 32 + lane) / PIECES, 8 * (piece % 8)));
                    const uint4 x = *at;
                    *at = make_uint4((x.x ^ sign) & keep, (x.y ^ sign) & keep, (x.z ^ sign) & keep, (x.w ^ sign) & keep);
                }
            }
            fence_async();
            warp_arrive(&bars->q_ready[w]);
        };
        // (the first time round there is no run yet, only the next one's queries: one place for them in the code)
        bool none_yet = true;
        Run run = {};
        run.stop = u;
        while (ok && (none_yet || u < end)) {
            const bool whole = run.whole;
            const int units = run.count();
            const bool live = q_row < run.rows;
            const int m = it.tile * MR + max(min(q_row, run.rows - 1), 0), i = m / a.group, h = it.head * a.group + (m - i * a.group);
            const int pos = it.q.c + i, low = a.window > 0 ? max(it.q.first, pos - a.window + 1) : it.q.first;
            float top = -INFINITY, sum = 0.0f;
            uint64_t acc[FLUSH ? HS / 2 : 1];    // the mix of the units that have been flushed
#pragma unroll
            for (int k = 0; k < (FLUSH ? HS / 2 : 1); ++k) acc[k] = 0ull;
            for (int n = 0; n < units && ok; ++n) {
                const int t = run.a + n;
                const uint32_t place = n_p % PLACES, at = mine + place * Sh::PLACE;
                ok = warp_wait(&bars->s_ready[w][place], (n_p / PLACES) & 1, failed);
                if (!ok) break;
                tc_after();
                const int from = low - t * KT, to = pos - t * KT;   // keys [from, to] of the unit are seen
                const bool edge = __any_sync(0xffffffffu, from > 0 || to < KT - 1);
                const uint64_t scales = two(scale2, scale2);
                uint64_t part[2];
                if constexpr (L == 1) {
                    // One pass with the maximum as it was, the weights kept in registers; only when that has grown by more than
                    // 2^GROWN (a tile's first unit, hardly ever after) a second one with the new maximum.  (Two passes over the
                    // scores, the maximum first: 579 us for 4 x 2048 new tokens, one 557.)
                    uint32_t p[KT / 2];
#pragma unroll 1
                    for (bool again = false;; again = true) {
                        const float base = top == -INFINITY ? 0.0f : top;
                        const uint64_t bases = two(-base, -base);
                        float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        part[0] = part[1] = 0ull;
#pragma unroll
                        for (int c = 0; c < KT; c += 32) {
                            uint32_t s[32];
                            tmem_ld32(at + c, s);
                            tmem_wait_ld();
                            if (edge) {
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (c + j < from || c + j > to) s[j] = 0xff800000u;
                            }
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                high[k & 3] = fmaxf(high[k & 3], fmaxf(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])));
                                float x, y;
                                apart(fma2(two(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), scales, bases), x, y);
                                x = exp2_fast(x);
                                y = exp2_fast(y);
                                part[k & 1] = add2(part[k & 1], two(x, y));
                                p[c / 2 + k] = pack_bf16(x, y);
                            }
                        }
                        if (again) break;
                        const float peak2 = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3])) * scale2;
                        const bool grown = peak2 > top + GROWN || (top == -INFINITY && peak2 > -INFINITY);
                        if (!__any_sync(0xffffffffu, grown)) break;
                        const float now = grown ? peak2 : top, f = grown ? (top == -INFINITY ? 0.0f : exp2_fast(top - now)) : 1.0f;
                        if (n > 0) {                 // once the unit before has been added up
                            ok = warp_wait(&bars->pv_done[w][(n_p - 1) % PLACES], ((n_p - 1) / PLACES) & 1, failed);
                            if (!ok) break;
                            tc_after();
#pragma unroll 1
                            for (int c = 0; c < HS; c += 32) {
                                uint32_t o[32];
                                tmem_ld32(mine + Sh::C_O + c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                                tmem_st32(mine + Sh::C_O + c, o);
                            }
                        }
                        sum *= f;
                        top = now;
                    }
                    if (!ok) break;
                    tmem_st16(at + Sh::weights_at(0, 0), p);
                    tmem_st16(at + Sh::weights_at(0, 32), p + 16);
                } else {
                    float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    // Two passes, some columns at a time in loops that are not unrolled: straight through, the code is larger than
                    // the instruction caches keep at hand, and three limbs of 64 weights are more than the registers hold.
#pragma unroll 1
                    for (int c = 0; c < KT; c += 32) {
                        uint32_t s[32];
                        tmem_read(at + c, s);
                        tmem_wait_ld();
                        if (edge) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (c + j < from || c + j > to) s[j] = 0xff800000u;
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) high[j & 3] = fmaxf(high[j & 3], __uint_as_float(s[j]));
                    }
                    const float peak2 = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3])) * scale2;
                    const bool grown = peak2 > top + GROWN || (top == -INFINITY && peak2 > -INFINITY);
                    const bool some = __any_sync(0xffffffffu, grown);
                    if (n > 0 && some) {             // once the unit before has been added up
                        ok = warp_wait(&bars->pv_done[w][(n_p - 1) % PLACES], ((n_p - 1) / PLACES) & 1, failed);
                        if (!ok) break;
                        tc_after();
                    }
                    if (some) {
                        const float now = grown ? peak2 : top, f = grown ? (top == -INFINITY ? 0.0f : exp2_fast(top - now)) : 1.0f;
                        if (n > 0) {
#pragma unroll 1
                            for (int c = 0; c < HS; c += 32) {
                                uint32_t o[32];
                                tmem_ld32(mine + Sh::C_O + c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                                tmem_st32(mine + Sh::C_O + c, o);
                            }
                            tmem_wait_st();          // it may be read again below
                        }
#pragma unroll
                        for (int k = 0; k < HS / 2; ++k) acc[k] = mul2(acc[k], two(f, f));
                        sum *= f;
                        top = now;
                    }
                    const float base = top == -INFINITY ? 0.0f : top;
                    const uint64_t bases = two(-base, -base);
                    part[0] = part[1] = 0ull;
#pragma unroll 1
                    for (int c = 0; c < KT; c += CW) {
                        uint32_t s[CW], p[L][CW / 2];
                        tmem_read(at + c, s);
                        tmem_wait_ld();
                        if (edge) {
#pragma unroll
                            for (int j = 0; j < CW; ++j)
                                if (c + j < from || c + j > to) s[j] = 0xff800000u;
                        }
#pragma unroll
                        for (int k = 0; k < CW / 2; ++k) {
                            float x, y;
                            apart(fma2(two(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1])), scales, bases), x, y);
                            x = exp2_fast(x);
                            y = exp2_fast(y);
                            uint64_t e = two(x, y);
                            part[k & 1] = add2(part[k & 1], e);
#pragma unroll
                            for (int l = 0; l < L; ++l) p[l][k] = limb(e);
                        }
#pragma unroll
                        for (int l = 0; l < L; ++l) tmem_write(at + Sh::weights_at(l, c), p[l]);
                    }
                    if (n > 0 && n % FLUSH == 0) {   // the mix so far joins acc; the next one starts anew
                        ok = warp_wait(&bars->pv_done[w][(n_p - 1) % PLACES], ((n_p - 1) / PLACES) & 1, failed);
                        if (!ok) break;
                        tc_after();
#pragma unroll
                        for (int c = 0; c < HS; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(mine + Sh::C_O + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k) acc[c / 2 + k] = add2(acc[c / 2 + k], two(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1])));
                        }
                    }
                }
                float x, y;
                apart(add2(part[0], part[1]), x, y);
                sum += x + y;
                tmem_wait_st();
                tc_before();
                warp_arrive(&bars->p_ready[w][place]);
                ++n_p;
            }
            if (!ok) break;
            split::Item then = it;
            Run then_run = run;
            if (run.stop < end) {
                if (!none_yet) next_item(a, then);
                then_run = run_of(a, then, run.stop, end, w);
                if (then_run.count() > 0) bring(then, then_run);
            }
            // ---- the read of the row, or this piece's end of it
            if (units > 0 && ok) ok = warp_wait(&bars->pv_done[w][(n_p - 1) % PLACES], ((n_p - 1) / PLACES) & 1, failed);
            if (!ok) break;
            tc_after();
            if (!none_yet) {
                const float inv = whole ? (sum > 0.0f ? 1.0f / sum : sum) : 1.0f;
                unsigned char* room = smem + Sh::OFF_ROWS + warp * ROWS_ROOM;
                float* end_of = ends + ((int64_t)worker * 2 + (u == it.begin ? 1 : 0)) * Ends<HS, MR>::FLOATS;
                const int64_t to = (int64_t)(it.q.start + i) * a.out_token_stride + (int64_t)h * a.out_head_stride;
#pragma unroll(FLUSH ? HS / 32 : 1)
                for (int c = 0; c < HS; c += 32) {
                    uint32_t o[32];
                    float x[32];
                    if (units > 0) {
                        tmem_ld32(mine + Sh::C_O + c, o);
                        tmem_wait_ld();
                        if constexpr (FLUSH > 0) {
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                float y, z;
                                apart(add2(acc[c / 2 + k], two(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1]))), y, z);
                                o[2 * k] = __float_as_uint(y);
                                o[2 * k + 1] = __float_as_uint(z);
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 32; ++k) x[k] = units > 0 ? __uint_as_float(o[k]) : 0.0f;
                    const int rows = run.rows - (q_row - lane);   // of this warp that are there
                    if (L == 3 || !whole) {
                        uint32_t y[32];
#pragma unroll
                        for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(x[k] * inv);
                        put_rows<8>(room, y, reinterpret_cast<unsigned char*>(whole ? a.out : end_of), 4 * (whole ? to + c : (int64_t)(q_row * HS + c)), rows, !whole || out_wide, 4);
                    } else {
                        uint32_t y[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) y[k] = pack_bf16(x[2 * k] * inv, x[2 * k + 1] * inv);
                        put_rows<4>(room, y, static_cast<unsigned char*>(a.out), 2 * (to + c), rows, out_wide, 2);
                    }
                }
                if (live) {
                    if (!whole) {
                        end_of[MR * HS + q_row] = top;
                        end_of[MR * HS + MR + q_row] = sum;
                    } else if (a.lse) {
                        a.lse[(int64_t)(it.q.start + i) * a.heads + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
                    }
                }
                if (!whole && u == it.begin && tid == 0) {
                    cuts[worker].start = it.q.start;
                    cuts[worker].head = it.head;
                    cuts[worker].tile = it.tile;
                    cuts[worker].rows = run.rows;
                    cuts[worker].workers = (int)split::last_worker<Plan>(it, per) - worker + 1;
                }
            }
            __syncwarp();                        // the row's results have been stored by all lanes
            if (units > 0 && live && (run.swept(run.a) || run.swept(run.b - 1))) {
                const volatile Found* found = reinterpret_cast<const Found*>(smem + Sh::OFF_FOUND) + runs % RUNS;
                if (found->count > 0) {          // values that are not finite have been taken out: the row gets those that it sees
                    float* row_end = ends + ((int64_t)worker * 2 + (u == it.begin ? 1 : 0)) * Ends<HS, MR>::FLOATS + q_row * HS;
                    add_found<HS>(a, it.r, it.head, found, low, pos, run.a, run.b, whole ? nullptr : row_end,
                                  (int64_t)(it.q.start + i) * a.out_token_stride + (int64_t)h * a.out_head_stride);
                }
            }
            if (run.ta < run.tb) ++runs;
            tc_before();
            if (units > 0) warp_arrive(&bars->o_free[w]);
            u = run.stop;
            it = then;
            run = then_run;
            none_yet = false;
        }
    } else if (warp < 10) {
        // ---- a group's multiplies: one lane issues
        constexpr uint32_t i_s = instr_desc(KT), i_o = instr_desc(HS) | (1u << 16);   // V with its keys down
        const int w = warp - 8;
        const uint32_t d = tmem + w * Sh::GROUP;
        uint32_t n_s = 0, n_p = 0, n_run = 0, base = 0;   // units scored, mixed; runs; units of the ring before this run
        while (u < end && ok) {
            const Run run = run_of(a, it, u, end, w);
            const int from = run.a, to = run.b;
            auto full = [&](int t) {             // unit t has landed
                const uint32_t seq = base + (uint32_t)(t - run.ta);
                ok = ok && warp_wait(&bars->full[seq % RING], (seq / RING) & 1, failed);
            };
            auto pass = [&](int t) {             // a unit that is the other group's alone
                full(t);
                if (ok && lane == 0) {
                    const uint32_t slot = (base + (uint32_t)(t - run.ta)) % RING;
                    bar_arrive(&bars->empty[slot]);
                }
            };
            // (a run without work for this group is passed over only when its rows are done with the one before: the sweeping
            // warp is then never further ahead of them than the ring)
            if (from >= to && n_run > 0) ok = ok && warp_wait(&bars->o_free[w], (n_run - 1) & 1, failed);
            for (int t = run.ta; t < min(from, run.tb) && ok; ++t) pass(t);
            if (from < to) ok = ok && warp_wait(&bars->q_ready[w], n_run & 1, failed);
            // a step: the mix of unit t, and as soon as that is done the scores of the unit that takes its place
#pragma unroll 1
            for (int t = from - (int)PLACES; t < to && ok; ++t) {
                const int ts = t + (int)PLACES;
                if (ts < to) full(ts);           // waited for before the weights are: nothing but the mix lies between them and the next scores
                if (t >= from) {
                    const uint32_t seq = base + (uint32_t)(t - run.ta), slot = seq % RING, place = n_p % PLACES;
                    const bool first = t == from, fresh_sum = FLUSH ? (t - from) % (FLUSH ? FLUSH : 1) == 0 : first;
                    if (run.swept(t)) ok = ok && warp_wait(&bars->passed[slot], (seq / RING) & 1, failed);
                    if (first && n_run > 0) ok = ok && warp_wait(&bars->o_free[w], (n_run - 1) & 1, failed);
                    ok = ok && warp_wait(&bars->p_ready[w][place], (n_p / PLACES) & 1, failed);
                    if (!ok) break;
                    if (elected()) {
                        tc_after();
                        const uint32_t at_v = at0 + Sh::OFF_V + slot * Sh::KV;
#pragma unroll
                        for (int l = L - 1; l >= 0; --l)
#pragma unroll
                            for (int c = 0; c < KT / 16; ++c)
                                mma_ts(d + Sh::C_O, d + place * Sh::PLACE + Sh::weights_at(l, 16 * c / CW * CW) + 16 * c % CW / 2, desc_keys_down(at_v + c * 2048, KT * 128),
                                       i_o, !fresh_sum || l < L - 1 || c > 0);
                        commit(&bars->pv_done[w][place]);
                        commit(&bars->empty[slot]);
                    }
                    __syncwarp();
                    ++n_p;
                }
                if (ts >= to) continue;
                const uint32_t place = n_s % PLACES, slot = (base + (uint32_t)(ts - run.ta)) % RING;
                if (n_s >= PLACES) ok = ok && warp_wait(&bars->pv_done[w][place], ((n_s - PLACES) / PLACES) & 1, failed);
                if (!ok) break;
                if (elected()) {
                    tc_after();
                    const unsigned char* q = smem + w * Sh::Q_TILE;
                    const unsigned char* k = smem + Sh::OFF_K + slot * Sh::KV;
#pragma unroll
                    for (int l = L - 1; l >= 0; --l)
#pragma unroll
                        for (int c = 0; c < HS / 16; ++c)
                            mma_ss(d + place * Sh::PLACE, operand_desc(q + l * Sh::Q_LIMB + (c / 4) * (128 * 128)) + 2u * (c & 3),
                                   operand_desc(k + (c / 4) * (KT * 128)) + 2u * (c & 3), i_s, l < L - 1 || c > 0);
                    commit(&bars->s_ready[w][place]);
                }
                __syncwarp();
                ++n_s;
            }
            for (int t = max(to, run.ta); t < run.tb && ok; ++t) pass(t);
            if (from < to) ++n_run;
            base += (uint32_t)(run.tb - run.ta);
            u = run.stop;
            if (u < end) next_item(a, it);
        }
        if (!ok) {   // the multiplies in flight end before the block does
            if (elected()) commit(&bars->drained[w]);
            __syncwarp();
            bar_wait(&bars->drained[w], 0);
        }
    } else if (warp == 10) {
        // ---- the copies: a lane per box
        uint32_t n = 0;
        bool bad_page = false;
        const int boxes = KT / box_rows * Sh::HALVES;
        while (u < end && ok) {
            const Run run = run_of(a, it, u, end, 0);
            const int32_t* pages = a.table + (int64_t)it.r * a.max_pages;
            for (int t = run.ta; t < run.tb && ok; ++t, ++n) {
                // a box is box_rows keys of one page (a unit's keys may lie within one page or run over several)
                int page = a.s.n_pages, place = 0;
                const int b = lane % (KT / box_rows), j = t * KT + b * box_rows;
                if (lane < boxes && j < it.s.hi && j + box_rows > it.s.lo) {
                    const int pi = j / a.s.page_size;
                    page = pages[pi];
                    place = j - pi * a.s.page_size;
                    if (page < 0 || page >= a.s.n_pages) {
                        bad_page = true;
                        page = a.s.n_pages;
                    }
                }
                const uint32_t slot = n % RING, turn = n / RING;
                if (turn > 0) ok = warp_wait(&bars->empty[slot], (turn - 1) & 1, failed);
                if (!ok) break;
                if (lane == 0) bar_expect(&bars->full[slot], 2 * Sh::KV);
                __syncwarp();
                if (lane < boxes) {   // at most 16: boxes of 8 keys and more
                    const int half = lane / (KT / box_rows), x = heads_inside ? it.head : place, y = heads_inside ? place : it.head;
                    const uint32_t to = at0 + slot * Sh::KV + half * (KT * 128) + b * box_rows * 128;
                    tma_box(to + Sh::OFF_K, &map_k, half * 64, x, y, page, &bars->full[slot]);
                    tma_box(to + Sh::OFF_V, &map_v, half * 64, x, y, page, &bars->full[slot]);
                }
                __syncwarp();
            }
            u = run.stop;
            if (u < end) next_item(a, it);
        }
        if (__any_sync(0xffffffffu, bad_page) && lane == 0 && a.status) atomicOr(a.status, AVA_PAGED_BAD_PAGE);
        if (!ok) {   // the copies in flight end before the block does
            for (uint32_t back = 1; back <= RING && back <= n; ++back) bar_wait(&bars->full[(n - back) % RING], ((n - back) / RING) & 1);
        }
    } else {
        // ---- the sweeping warp
        uint32_t n = 0, runs = 0;
        while (u < end && ok) {
            const Run run = run_of(a, it, u, end, 0);
            volatile Found* found = reinterpret_cast<Found*>(smem + Sh::OFF_FOUND) + runs % RUNS;
            int count = 0;
            for (int t = run.ta; t < run.tb && ok; ++t, ++n) {
                const uint32_t slot = n % RING;
                ok = warp_wait(&bars->full[slot], (n / RING) & 1, failed);
                if (!ok) break;
                if (run.swept(t)) {
                    unsigned char* v = smem + Sh::OFF_V + slot * Sh::KV;
                    const int clear_to = it.s.lo - t * KT, clear_from = it.s.hi - t * KT;   // rows in front of the stretch, and behind it
                    uint64_t keys = 0;
                    for (int e = lane; e < KT * (HS / 8); e += 32) {
                        const int key = e / (HS / 8), c = e % (HS / 8);
                        uint4* at = reinterpret_cast<uint4*>(v + (c / 8) * (KT * 128) + swz128(key, (c & 7) * 8));
                        if (key < clear_to || key >= clear_from) {
                            *at = make_uint4(0, 0, 0, 0);
                            continue;
                        }
                        uint4 x = *at;
                        uint32_t* y = reinterpret_cast<uint32_t*>(&x);
                        bool any = false;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {   // an exponent of all ones, in either half
                            const uint32_t m = ((y[k] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((y[k] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
                            any |= m != 0;
                            y[k] &= ~m;
                        }
                        if (any) {
                            *at = x;
                            keys |= 1ull << key;
                        }
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) keys |= __shfl_xor_sync(0xffffffffu, keys, o);
                    if (keys && count < 15) {
                        if (lane == 0) {
                            found->unit[count] = t;
                            found->keys[count] = keys;
                        }
                        ++count;
                    }
                    fence_async();
                }
                __threadfence_block();
                if (lane == 0) found->count = count;
                warp_arrive(&bars->passed[slot]);
                if (lane == 0) bar_arrive(&bars->empty[slot]);
            }
            if (run.ta < run.tb) ++runs;
            u = run.stop;
            if (u < end) next_item(a, it);
        }
    }
    if (!ok && lane == 0 && a.status) atomicOr(a.status, AVA_PAGED_WAIT_RAN_OUT);
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins the ends of the stretches that were cut (read_join.cuh): a block per worker and eight rows, a warp per row.
template <int HS>
__global__ void __launch_bounds__(256) join_rows_kernel(const ReadArgs a, const float* __restrict__ ends, const split::Cut* __restrict__ cuts) {
    pdl_enter();
    const split::Cut cut = cuts[blockIdx.x];
    const int row = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (cut.workers == 0 || row >= cut.rows) return;
    float m, l, o[HS / 32];
    join_parts<HS, MR>(ends, blockIdx.x, row, cut.workers, 0, 1, m, l, o);
    join_write<HS>(a, cut.start, cut.head, cut.tile * MR + row, m, l, o);
}

template <int HS, int L>
cudaError_t launch_one(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms, const PoolShape& pool, bool* taken) {
    using Sh = Shape<HS, L>;
    const int box_rows = a.s.page_size < KT ? a.s.page_size : KT;
    if (box_rows < 8 || KT % box_rows || a.s.page_size % box_rows) return cudaSuccess;
    CUtensorMap mk, mv;
    if (!pool_map(&mk, a.s.k, AVA_BF16, pool, box_rows) || !pool_map(&mv, a.s.v, AVA_BF16, pool, box_rows)) return cudaSuccess;
    *taken = true;
    split::Cut* cuts = static_cast<split::Cut*>(room);
    float* ends = reinterpret_cast<float*>(cuts + sms);
    cudaError_t rc = launch_serving<read_tc_kernel<Sh>>(device, dim3(sms), dim3(THREADS), Sh::BYTES, st, 1, mk, mv, a, pool.heads_inside ? 1 : 0, box_rows, ends, cuts);
    if (rc != cudaSuccess) return rc;
    return launch_serving<join_rows_kernel<HS>>(device, dim3(sms, MR / 8), dim3(256), 0, st, 1, a, ends, cuts);
}

}  // namespace

cudaError_t launch_paged_read_tc(int device, cudaStream_t st, const ReadArgs& a, void* room, int sms, bool* taken) {
    *taken = false;
    PoolShape pool;
    // Few rows per key head stay with the warp kernel, whose tiles of 8 to 32 rows read the store once.  Measured at 32 requests
    // of up to 4096 keys, 8 key heads (warp kernel / this one): 24 rows 90 / 102 us and 32 rows 144 / 104 us at 128 channels,
    // 32 rows 83 / 85 us and 48 rows 115 / 84 us at 64; f32 queries 32 rows 134 / 136 us, 48 rows 193 / 136 us.
    const int64_t few = a.s.head_size == 128 ? 24 : 32;
    if (a.s.dtype != AVA_BF16 || (a.s.head_size != 64 && !(a.s.head_size == 128 && a.bf16_q)) || (int64_t)a.max_fresh * a.group <= few || !pool_shape(a.s, &pool))
        return cudaSuccess;
    if (a.s.head_size == 64) return a.bf16_q ? launch_one<64, 1>(device, st, a, room, sms, pool, taken) : launch_one<64, 3>(device, st, a, room, sms, pool, taken);
    return launch_one<128, 1>(device, st, a, room, sms, pool, taken);
}

}  // namespace ava
