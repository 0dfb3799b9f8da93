// The lists of a serving step (block tables, slot maps) from the requests' lengths, and new keys and values into their pages.
//
// The lists.  With need = ceil((cached + fresh) / page) and owned pages per request, every request gives
// g = max(owned - need, 0) pages (trim) or takes t = max(need - owned, 0).  Exclusive sums of g, t and fresh over the
// requests say where each request's pages lie on the stack and where its tokens lie in the packed step: given page i of
// request r goes to place F + G(r) + i of the stack of height F, taken page i comes from place F + sum(g) - 1 - T(r) - i.
// The sums run in one block (a few kilobytes of lengths, one sum over the block for all three); the slots of a larger
// step's tokens, which are the bulk of the bytes, are written by as many blocks as there are tokens.
#include <cuda_runtime.h>

#include "ava_math.h"
#include "kernels.cuh"
#include "serving.cuh"

namespace ava {

namespace {

constexpr int PLAN_THREADS = 1024, TOKEN_THREADS = 256, PER_THREAD = 4, TOKENS_PER_BLOCK = TOKEN_THREADS * PER_THREAD;

// the last index i of 0 .. n - 1 with a[i] <= x (a ascending, a[0] <= x)
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The places of four tokens from t on; start[r - r0] is the first token of request r, for r = r0 .. r0 + n (total for the
// last of them), in shared memory or not.
__device__ __forceinline__ void put_tokens(const PlanArgs& a, int t, int total, const int* start, int r0, int n, bool wide, uint32_t& bad) {
    int64_t slot[PER_THREAD];
    int pos[PER_THREAD], row[PER_THREAD];
    int i = t < total ? last_not_above(start, n, t) : 0, cached = 0, from = 0, to = -1;
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) {
        slot[k] = -1;
        pos[k] = row[k] = -1;
        if (t + k < total) {
            if (t + k >= to) {   // this token's request: the next one that is not empty
                while (to >= 0 && start[i + 1] <= t + k) ++i;
                from = start[i];
                to = start[i + 1];
                cached = a.cached[r0 + i];
            }
            row[k] = r0 + i;
            pos[k] = cached + (t + k - from);
            const int p = pos[k] / a.page_size;   // below the request's need, which the table has places for
            const int page = a.table[(int64_t)row[k] * a.max_pages + p];
            if (page < 0 || page >= a.n_pages) bad |= AVA_PAGED_BAD_PAGE;
            else slot[k] = (int64_t)page * a.page_size + (pos[k] - p * a.page_size);
        }
    }
    if (wide && t + PER_THREAD <= a.max_tokens) {
        *reinterpret_cast<longlong2*>(a.slot + t) = make_longlong2(slot[0], slot[1]);
        *reinterpret_cast<longlong2*>(a.slot + t + 2) = make_longlong2(slot[2], slot[3]);
        if (a.pos) *reinterpret_cast<int4*>(a.pos + t) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        if (a.row) *reinterpret_cast<int4*>(a.row + t) = make_int4(row[0], row[1], row[2], row[3]);
    } else {
#pragma unroll
        for (int k = 0; k < PER_THREAD; ++k)
            if (t + k < a.max_tokens) {
                a.slot[t + k] = slot[k];
                if (a.pos) a.pos[t + k] = pos[k];
                if (a.row) a.row[t + k] = row[k];
            }
    }
}
__device__ __forceinline__ bool wide_tokens(const PlanArgs& a) {
    return !((reinterpret_cast<uintptr_t>(a.slot) | reinterpret_cast<uintptr_t>(a.pos) | reinterpret_cast<uintptr_t>(a.row)) & 15);
}

// What one request gives, takes and adds.
struct Share {
    int need, give, take, fresh, own;
};
__device__ __forceinline__ Share share(const PlanArgs& a, int r) {
    Share s;
    s.fresh = a.fresh[r];
    s.own = a.owned[r];
    s.need = (int)(((long long)a.cached[r] + s.fresh + a.page_size - 1) / a.page_size);
    s.take = max(s.need - s.own, 0);
    s.give = a.trim ? max(s.own - s.need, 0) : 0;
    return s;
}

// Each thread has the requests [tid * per, tid * per + per): one sum over the block says where the pages and tokens of all
// of them lie, whether the step can be granted included.  The pages are then moved by all threads, page by page.
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const PlanArgs a, const int tokens_here) {
    pdl_enter();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the tokens' kernel gets its blocks in place
    __shared__ long long warp_sum[3][33];
    __shared__ int s_off[PLAN_THREADS + 1], s_start[PLAN_THREADS + 1], s_own[PLAN_THREADS];
    __shared__ uint32_t s_bad;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rows = a.rows, per = (rows + PLAN_THREADS - 1) / PLAN_THREADS;
    const int r0 = min(tid * per, rows), r1 = min(r0 + per, rows);
    if (tid == 0) s_bad = 0;
    const int F = a.free_count[0];
    uint32_t bad = 0;
    long long sum[3] = {0, 0, 0};   // given, taken, new tokens
    Share only{};                   // the thread's one request, when it has no more
    for (int r = r0; r < r1; ++r) {
        const int c = a.cached[r], n = a.fresh[r], o = a.owned[r];
        const long long tokens = (long long)c + n;
        if (c < 0 || n < 0 || o < 0 || o > a.max_pages || tokens > 0x7fffffffll) {
            bad |= AVA_PAGED_BAD_LENGTH;
            continue;
        }
        const int need = (int)(((unsigned)tokens + (unsigned)a.page_size - 1u) / (unsigned)a.page_size);
        if (need > a.max_pages) bad |= AVA_PAGED_NO_TABLE;
        only.need = need;
        only.own = o;
        only.fresh = n;
        only.take = max(need - o, 0);
        only.give = a.trim ? max(o - need, 0) : 0;
        sum[0] += only.give;
        sum[1] += only.take;
        sum[2] += n;
    }
    long long inc[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        inc[i] = sum[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, inc[i], o);
            if (lane >= o) inc[i] += y;
        }
        if (lane == 31) warp_sum[i][warp] = inc[i];
    }
    bad = __reduce_or_sync(0xffffffffu, bad);
    __syncthreads();
    if (bad && lane == 0) atomicOr(&s_bad, bad);
    if (warp < 3) {
        const long long y = warp_sum[warp][lane];
        long long s = y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long z = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += z;
        }
        warp_sum[warp][lane] = s - y;
        if (lane == 31) warp_sum[warp][32] = s;
    }
    __syncthreads();
    const long long given = warp_sum[0][32], taken = warp_sum[1][32], tokens = warp_sum[2][32];
    uint32_t refused = s_bad;
    if (F < 0 || F > a.n_pages || given > (long long)(a.n_pages - F)) refused |= AVA_PAGED_BAD_LENGTH;
    else if (taken > F + given) refused |= AVA_PAGED_NO_PAGES;
    if (tokens > a.max_tokens) refused |= AVA_PAGED_NO_TOKENS;
    const int total = refused ? 0 : (int)tokens, top = F + (int)given;
    bad = 0;
    __syncthreads();

    if (refused) {
        for (int r = r0; r < r1; ++r) {
            a.owned_out[r] = a.owned[r];
            a.q_start[r] = 0;
        }
    } else {
        const int first_given = (int)(warp_sum[0][warp] + inc[0] - sum[0]), first_taken = (int)(warp_sum[1][warp] + inc[1] - sum[1]);
        int first_token = (int)(warp_sum[2][warp] + inc[2] - sum[2]);
        s_start[tid] = first_token;
        if (tid == 0) s_start[PLAN_THREADS] = total;
        // page k of those that change hands belongs to the thread whose sum is the last not above k, and there to the
        // request that the walk over the thread's requests ends at
        if (given > 0) {
            s_off[tid] = first_given;
            __syncthreads();
            for (int k = tid; k < (int)given; k += PLAN_THREADS) {
                const int who = last_not_above(s_off, PLAN_THREADS, k);
                int i = k - s_off[who], r = who * per;
                Share s = share(a, r);
                while (i >= s.give) {
                    i -= s.give;
                    s = share(a, ++r);
                }
                const int page = a.table[(int64_t)r * a.max_pages + s.need + i];
                if (page < 0 || page >= a.n_pages) bad |= AVA_PAGED_BAD_PAGE;
                a.free_list[F + k] = page;
            }
            __syncthreads();   // what is given may be taken in the same step
        }
        s_off[tid] = first_taken;
        s_own[tid] = only.own;
        __syncthreads();
        constexpr int AT_ONCE = 4;
        for (int k0 = tid; k0 < (int)taken; k0 += AT_ONCE * PLAN_THREADS) {
            int page[AT_ONCE];
            int64_t to[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int k = k0 + j * PLAN_THREADS;
                to[j] = -1;
                if (k < (int)taken) {
                    page[j] = a.free_list[top - 1 - k];
                    const int who = last_not_above(s_off, PLAN_THREADS, k);
                    int i = k - s_off[who], r = who * per, own = s_own[who];
                    if (per > 1) {
                        Share s = share(a, r);
                        while (i >= s.take) {
                            i -= s.take;
                            s = share(a, ++r);
                        }
                        own = s.own;
                    }
                    to[j] = (int64_t)r * a.max_pages + own + i;
                }
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
                if (to[j] >= 0) {
                    if (page[j] < 0 || page[j] >= a.n_pages) bad |= AVA_PAGED_BAD_PAGE;
                    a.table[to[j]] = page[j];
                }
        }
        __syncthreads();       // the counts may be written over their inputs
        for (int r = r0; r < r1; ++r) {
            const Share s = per == 1 ? only : share(a, r);
            a.q_start[r] = first_token;
            a.owned_out[r] = a.trim ? s.need : max(s.need, s.own);
            first_token += s.fresh;
        }
    }
    if (tid == 0) {
        a.q_start[rows] = total;
        a.free_count_out[0] = refused ? F : top - (int)taken;
    }
    __syncthreads();
    // a small step's tokens too, in the same launch
    if (tokens_here)
        for (int t = tid * PER_THREAD; t < a.max_tokens; t += PLAN_THREADS * PER_THREAD)
            put_tokens(a, t, total, per == 1 ? s_start : a.q_start, 0, per == 1 ? PLAN_THREADS : rows, wide_tokens(a), bad);
    bad = __reduce_or_sync(0xffffffffu, bad);
    if (bad && lane == 0) atomicOr(&s_bad, bad);
    __syncthreads();
    if (tid == 0 && a.status) a.status[0] = refused | s_bad;
}

// The tokens of a larger step.  A block's tokens run over a stretch of requests whose first tokens it brings into shared
// memory once (searching them in L2 cost ten dependent reads a token).
__global__ void __launch_bounds__(TOKEN_THREADS) plan_tokens_kernel(const PlanArgs a) {
    constexpr int KEPT = 1536;
    __shared__ int s_start[KEPT + 1];
    __shared__ int s_range[2];
    pdl_enter();
    const int total = a.q_start[a.rows], t0 = blockIdx.x * TOKENS_PER_BLOCK, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (warp < 2 && t0 < total) {   // the requests of the block's first and last token, by 32-way search
        const int t = warp == 0 ? t0 : min(t0 + TOKENS_PER_BLOCK, total) - 1;
        int lo = 0, n = a.rows;
        while (n > 1) {
            const int step = (n + 31) / 32, at = lo + lane * step;
            const unsigned below = __ballot_sync(0xffffffffu, lane * step < n && a.q_start[at] <= t);
            const int k = 31 - __clz(below);
            n = min(step, n - k * step);
            lo += k * step;
        }
        if (lane == 0) s_range[warp] = lo;
    }
    __syncthreads();
    const int r0 = t0 < total ? s_range[0] : 0, n = t0 < total ? s_range[1] - r0 + 1 : 0;
    const bool kept = n <= KEPT;
    if (kept)
        for (int i = tid; i <= n; i += TOKEN_THREADS) s_start[i] = a.q_start[r0 + i];
    __syncthreads();
    uint32_t bad = 0;
    const int t = t0 + tid * PER_THREAD;
    if (t < a.max_tokens) put_tokens(a, t, total, kept ? s_start : a.q_start + r0, r0, n, wide_tokens(a), bad);
    if (bad && a.status) atomicOr(a.status, bad);
}

// ---- append.  A thread moves eight channels of both pools, four times over tokens a grid apart, all loads before the first
// store; channels, strides or pointers that are not whole 16-byte pieces take the form that moves one channel at a time.
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) { return f_to_bf16(lo) | ((uint32_t)f_to_bf16(hi) << 16); }

// where a channel of a token goes in the pools, -1: nowhere
__device__ __forceinline__ int64_t place_of(const AppendArgs& a, int64_t slot, int head, int channel, bool first) {
    if (slot < 0) return -1;
    const int64_t places = (int64_t)a.s.n_pages * a.s.page_size;
    if (slot >= places) {
        if (first && a.status) atomicOr(a.status, AVA_PAGED_BAD_PAGE);
        return -1;
    }
    const int64_t page = places <= 0x7fffffffll ? (int64_t)((uint32_t)slot / (uint32_t)a.s.page_size) : slot / a.s.page_size;
    return page * a.s.page_stride + head * a.s.head_stride + (slot - page * a.s.page_size) * a.s.place_stride + channel;
}

template <bool BF16_IN, bool BF16_OUT>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
    pdl_enter();
    constexpr int TIMES = 4, IN = BF16_IN ? 1 : 2, OUT = BF16_OUT ? 1 : 2;   // 16-byte pieces of eight channels
    const uint32_t per_head = a.s.head_size / 8, per_token = a.s.kv_heads * per_head;
    const uint32_t n = (uint32_t)a.tokens * per_token, step = gridDim.x * 256;
    uint4 x[TIMES][2][IN];
    int64_t to[TIMES];
#pragma unroll
    for (int i = 0; i < TIMES; ++i) {
        const uint32_t id = blockIdx.x * 256 + threadIdx.x + i * step;
        to[i] = -1;
        if (id < n) {
            const uint32_t t = id / per_token, piece = id - t * per_token, h = piece / per_head, c = 8 * (piece - h * per_head);
            const int64_t from = (int64_t)t * a.token_stride + (int64_t)h * a.head_stride + c;
            const int64_t slot = a.slot[t];
#pragma unroll
            for (int k = 0; k < IN; ++k) {
                x[i][0][k] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(a.k) + from * (BF16_IN ? 2 : 4)) + k);
                x[i][1][k] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(a.v) + from * (BF16_IN ? 2 : 4)) + k);
            }
            to[i] = place_of(a, slot, (int)h, (int)c, piece == 0);
        }
    }
#pragma unroll
    for (int i = 0; i < TIMES; ++i) {
        if (to[i] < 0) continue;
#pragma unroll
        for (int pool = 0; pool < 2; ++pool) {
            uint4* out = reinterpret_cast<uint4*>(static_cast<unsigned char*>(pool ? a.s.v : a.s.k) + to[i] * (BF16_OUT ? 2 : 4));
            const uint4(&y)[IN] = x[i][pool];
            if constexpr (!BF16_IN && BF16_OUT) {
                const uint4 u = y[0], v = y[IN - 1];
                out[0] = make_uint4(two_bf16(__uint_as_float(u.x), __uint_as_float(u.y)), two_bf16(__uint_as_float(u.z), __uint_as_float(u.w)),
                                    two_bf16(__uint_as_float(v.x), __uint_as_float(v.y)), two_bf16(__uint_as_float(v.z), __uint_as_float(v.w)));
            } else {
#pragma unroll
                for (int k = 0; k < OUT; ++k) out[k] = y[k];
            }
        }
    }
}

template <typename Tin, typename Tout>
__device__ __forceinline__ Tout converted(Tin x) {
    if constexpr (sizeof(Tin) == 4 && sizeof(Tout) == 2) return f_to_bf16(x);
    else return x;
}
template <typename Tin, typename Tout>
__global__ void __launch_bounds__(256) append_any_kernel(const AppendArgs a) {
    pdl_enter();
    const int hs = a.s.head_size, width = a.s.kv_heads * hs;
    const int64_t n = (int64_t)a.tokens * width;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / width;
        const int c = (int)(i - t * width), h = c / hs, x = c - h * hs;
        const int64_t to = place_of(a, a.slot[t], h, x, c == 0), from = t * a.token_stride + h * a.head_stride + x;
        if (to < 0) continue;
        static_cast<Tout*>(a.s.k)[to] = converted<Tin, Tout>(static_cast<const Tin*>(a.k)[from]);
        static_cast<Tout*>(a.s.v)[to] = converted<Tin, Tout>(static_cast<const Tin*>(a.v)[from]);
    }
}

}  // namespace

cudaError_t launch_paged_plan(int device, cudaStream_t st, const PlanArgs& a) {
    const bool one = a.max_tokens <= PER_THREAD * PLAN_THREADS;   // one round of the one block
    cudaError_t rc = launch_serving<plan_kernel>(device, dim3(1), dim3(PLAN_THREADS), 0, st, 1, a, one ? 1 : 0);
    if (rc != cudaSuccess || one) return rc;
    return launch_serving<plan_tokens_kernel>(device, dim3((a.max_tokens + TOKENS_PER_BLOCK - 1) / TOKENS_PER_BLOCK), dim3(TOKEN_THREADS), 0, st, 1, a);
}

cudaError_t launch_paged_append(int device, cudaStream_t st, const AppendArgs& a) {
    const int in = a.bf16_in ? 2 : 4, out = a.s.dtype == AVA_BF16 ? 2 : 4;
    const uintptr_t pointers = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.s.k) | reinterpret_cast<uintptr_t>(a.s.v);
    const int64_t bytes = a.token_stride * in | a.head_stride * in | a.s.page_stride * out | a.s.head_stride * out | a.s.place_stride * out;
    const int64_t n = (int64_t)a.tokens * a.s.kv_heads * a.s.head_size;
    if (!((pointers | (uintptr_t)bytes) & 15) && a.s.head_size % 8 == 0 && n / 8 < 0x40000000ll) {
        // few tokens are spread over the SMs first (a piece per thread); many go four to a thread
        const int64_t threads = n / 8 <= 148 * 1024 ? n / 8 : (n / 8 + 3) / 4;
        const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
        if (a.bf16_in) return launch_serving<append_kernel<true, true>>(device, grid, block, 0, st, 1, a);
        if (out == 2) return launch_serving<append_kernel<false, true>>(device, grid, block, 0, st, 1, a);
        return launch_serving<append_kernel<false, false>>(device, grid, block, 0, st, 1, a);
    }
    const dim3 grid((unsigned)((n + 255) / 256 < 148 * 64 ? (n + 255) / 256 : 148 * 64)), block(256);
    if (a.bf16_in) return launch_serving<append_any_kernel<uint16_t, uint16_t>>(device, grid, block, 0, st, 1, a);
    if (out == 2) return launch_serving<append_any_kernel<float, uint16_t>>(device, grid, block, 0, st, 1, a);
    return launch_serving<append_any_kernel<float, float>>(device, grid, block, 0, st, 1, a);
}

}  // namespace ava
