// The lists of a serving step (block tables, slot maps) from the requests' lengths, and new keys and values into their pages.
//
// The lists.  With need = ceil((cached + fresh) / page) and owned pages per request, every request gives
// g = max(owned - need, 0) pages (trim) or takes t = max(need - owned, 0).  Exclusive sums of g, t and fresh over the
// requests say where each request's pages lie on the stack and where its tokens lie in the packed step: given page i of
// request r goes to place F + G(r) + i of the stack of height F, taken page i comes from place F + sum(g) - 1 - T(r) - i.
// The sums run in one block (a few kilobytes of lengths); the slots of the tokens, which are the bulk of the bytes, are
// written by as many blocks as there are tokens, each finding its requests by search in the first-token sums.
#include <cuda_runtime.h>

#include "ava_math.h"
#include "kernels.cuh"
#include "serving.cuh"

namespace ava {

namespace {

constexpr int PLAN_THREADS = 1024, TOKEN_THREADS = 256, TOKENS_PER_BLOCK = 1024;

// Exclusive sums of two counts over the block's threads; every thread calls it.  tot gets the block's sums.
__device__ __forceinline__ void block_sums(int (&x)[2], int (&tot)[2], int (*warp_tot)[2]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        inc[c] = x[c];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc[c], o);
            if (lane >= o) inc[c] += y;
        }
        if (lane == 31) warp_tot[warp][c] = inc[c];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            int y = warp_tot[lane][c], s = y;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int z = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += z;
            }
            warp_tot[lane][c] = s - y;
            if (lane == 31) warp_tot[32][c] = s;
        }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        x[c] = warp_tot[warp][c] + inc[c] - x[c];
        tot[c] = warp_tot[32][c];
    }
    __syncthreads();
}

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

__device__ __forceinline__ void put_token(const PlanArgs& a, int t, int total, int r, int start, uint32_t& bad) {
    int64_t slot = -1;
    int pos = -1, row = -1;
    if (t < total) {
        pos = a.cached[r] + (t - start);
        row = r;
        const int p = pos / a.page_size;
        const int page = a.table[(int64_t)r * a.max_pages + p];   // p < need(r) <= max_pages: checked before the tokens are counted in
        if (page < 0 || page >= a.n_pages) bad |= AVA_PAGED_BAD_PAGE;
        else slot = (int64_t)page * a.page_size + (pos - p * a.page_size);
    }
    a.slot[t] = slot;
    if (a.pos) a.pos[t] = pos;
    if (a.row) a.row[t] = row;
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const PlanArgs a, const int tokens_here) {
    pdl_enter();
    __shared__ int warp_tot[33][2];
    __shared__ int s_off[PLAN_THREADS + 1], s_row[PLAN_THREADS];   // offsets (and what else a row needs) of the rows of a chunk
    __shared__ unsigned long long s_fresh, s_give, s_take;
    __shared__ uint32_t s_bad;
    const int tid = threadIdx.x, rows = a.rows;
    if (tid == 0) {
        s_fresh = s_give = s_take = 0ull;
        s_bad = 0;
    }
    const int F = a.free_count[0];
    __syncthreads();

    // the whole step first: whether it can be granted
    {
        unsigned long long f = 0, g = 0, t = 0;
        uint32_t bad = 0;
        for (int r = tid; r < rows; r += PLAN_THREADS) {
            const int c = a.cached[r], n = a.fresh[r], o = a.owned[r];
            const long long tokens = (long long)c + n;
            if (c < 0 || n < 0 || o < 0 || o > a.max_pages || tokens > 0x7fffffffll) {
                bad |= AVA_PAGED_BAD_LENGTH;
                continue;
            }
            const long long need = (tokens + a.page_size - 1) / a.page_size;
            if (need > a.max_pages) bad |= AVA_PAGED_NO_TABLE;
            f += (unsigned long long)n;
            if (need > o) t += (unsigned long long)(need - o);
            else if (a.trim) g += (unsigned long long)(o - need);
        }
        if (f) atomicAdd(&s_fresh, f);
        if (g) atomicAdd(&s_give, g);
        if (t) atomicAdd(&s_take, t);
        if (bad) atomicOr(&s_bad, bad);
    }
    __syncthreads();
    if (tid == 0) {
        uint32_t bad = s_bad;
        if (F < 0 || F > a.n_pages || s_give > (unsigned long long)(a.n_pages - F)) bad |= AVA_PAGED_BAD_LENGTH;
        else if (s_take > (unsigned long long)F + s_give) bad |= AVA_PAGED_NO_PAGES;
        if (s_fresh > (unsigned long long)a.max_tokens) bad |= AVA_PAGED_NO_TOKENS;
        s_bad = bad;
    }
    __syncthreads();
    const uint32_t refused = s_bad;
    const int total = refused ? 0 : (int)s_fresh, top = F + (int)s_give;
    if (refused) {
        for (int r = tid; r < rows; r += PLAN_THREADS) {
            a.owned_out[r] = a.owned[r];
            a.q_start[r] = 0;
        }
        if (tid == 0) {
            a.q_start[rows] = 0;
            a.free_count_out[0] = F;
        }
    }
    uint32_t bad = 0;
    // given pages onto the stack, all of them before any is taken
    if (!refused && s_give) {
        int carry = 0;
        for (int r0 = 0; r0 < rows; r0 += PLAN_THREADS) {
            const int r = r0 + tid;
            int need = 0, give = 0;
            if (r < rows) {
                need = (int)(((long long)a.cached[r] + a.fresh[r] + a.page_size - 1) / a.page_size);
                give = max(a.owned[r] - need, 0);
            }
            int x[2] = {give, 0}, tot[2];
            block_sums(x, tot, warp_tot);
            s_off[tid] = x[0];
            s_row[tid] = need;
            __syncthreads();
            for (int k = tid; k < tot[0]; k += PLAN_THREADS) {
                const int i = last_not_above(s_off, PLAN_THREADS, k);
                const int page = a.table[(int64_t)(r0 + i) * a.max_pages + s_row[i] + (k - s_off[i])];
                if (page < 0 || page >= a.n_pages) bad |= AVA_PAGED_BAD_PAGE;
                a.free_list[F + carry + k] = page;
            }
            carry += tot[0];
            __syncthreads();
        }
    }
    // pages off the stack, the counts, the first tokens
    if (!refused) {
        int taken = 0, tokens = 0;
        for (int r0 = 0; r0 < rows; r0 += PLAN_THREADS) {
            const int r = r0 + tid;
            int take = 0, fresh = 0, own = 0, now = 0;
            if (r < rows) {
                fresh = a.fresh[r];
                own = a.owned[r];
                const int need = (int)(((long long)a.cached[r] + fresh + a.page_size - 1) / a.page_size);
                take = max(need - own, 0);
                now = a.trim ? need : max(need, own);
            }
            int x[2] = {take, fresh}, tot[2];
            block_sums(x, tot, warp_tot);
            if (r < rows) {
                a.q_start[r] = tokens + x[1];
                a.owned_out[r] = now;
            }
            s_off[tid] = x[0];
            s_row[tid] = own;
            __syncthreads();
            for (int k = tid; k < tot[0]; k += PLAN_THREADS) {
                const int i = last_not_above(s_off, PLAN_THREADS, k);
                const int page = a.free_list[top - 1 - taken - k];
                if (page < 0 || page >= a.n_pages) bad |= AVA_PAGED_BAD_PAGE;
                a.table[(int64_t)(r0 + i) * a.max_pages + s_row[i] + (k - s_off[i])] = page;
            }
            taken += tot[0];
            tokens += tot[1];
            __syncthreads();
        }
        if (tid == 0) {
            a.q_start[rows] = tokens;
            a.free_count_out[0] = top - taken;
        }
    }
    if (bad) atomicOr(&s_bad, bad);
    __syncthreads();
    // a small step's tokens too, in the same launch
    if (tokens_here) {
        bad = 0;
        for (int t = tid; t < a.max_tokens; t += PLAN_THREADS) {
            const int r = t < total ? last_not_above(a.q_start, rows, t) : 0;
            put_token(a, t, total, r, t < total ? a.q_start[r] : 0, bad);
        }
        if (bad) atomicOr(&s_bad, bad);
        __syncthreads();
    }
    if (tid == 0 && a.status) a.status[0] = s_bad;
}

__global__ void __launch_bounds__(TOKEN_THREADS) plan_tokens_kernel(const PlanArgs a) {
    pdl_enter();
    const int total = a.q_start[a.rows];
    uint32_t bad = 0;
    for (int i = threadIdx.x; i < TOKENS_PER_BLOCK; i += TOKEN_THREADS) {
        const int t = blockIdx.x * TOKENS_PER_BLOCK + i;
        if (t >= a.max_tokens) break;
        const int r = t < total ? last_not_above(a.q_start, a.rows, t) : 0;
        put_token(a, t, total, r, t < total ? a.q_start[r] : 0, bad);
    }
    if (bad && a.status) atomicOr(a.status, bad);
}

// ---- append: one channel of both pools per thread
template <typename Tin, typename Tout>
struct Convert;
template <>
struct Convert<float, float> {
    static __device__ float go(float x) { return x; }
};
template <>
struct Convert<float, uint16_t> {
    static __device__ uint16_t go(float x) { return f_to_bf16(x); }
};
template <>
struct Convert<uint16_t, uint16_t> {
    static __device__ uint16_t go(uint16_t x) { return x; }
};

template <typename Tin, typename Tout>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
    pdl_enter();
    const int hs = a.s.head_size, width = a.s.kv_heads * hs;
    const int64_t n = (int64_t)a.tokens * width;
    const int64_t places = (int64_t)a.s.n_pages * a.s.page_size;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / width;
        const int c = (int)(i - t * width), h = c / hs, x = c - h * hs;
        const int64_t slot = a.slot[t];
        if (slot < 0) continue;
        if (slot >= places) {
            if (c == 0 && a.status) atomicOr(a.status, AVA_PAGED_BAD_PAGE);
            continue;
        }
        const int64_t page = slot / a.s.page_size, place = slot - page * a.s.page_size;
        const int64_t from = t * a.token_stride + h * a.head_stride + x;
        const int64_t to = page * a.s.page_stride + h * a.s.head_stride + place * a.s.place_stride + x;
        static_cast<Tout*>(a.s.k)[to] = Convert<Tin, Tout>::go(static_cast<const Tin*>(a.k)[from]);
        static_cast<Tout*>(a.s.v)[to] = Convert<Tin, Tout>::go(static_cast<const Tin*>(a.v)[from]);
    }
}

}  // namespace

cudaError_t launch_paged_plan(cudaStream_t st, const PlanArgs& a) {
    const bool one = a.max_tokens <= 4 * PLAN_THREADS;
    cudaError_t rc = launch_serving(plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, st, 1, a, one ? 1 : 0);
    if (rc != cudaSuccess || one) return rc;
    return launch_serving(plan_tokens_kernel, dim3((a.max_tokens + TOKENS_PER_BLOCK - 1) / TOKENS_PER_BLOCK), dim3(TOKEN_THREADS), 0, st, 1, a);
}

cudaError_t launch_paged_append(cudaStream_t st, const AppendArgs& a) {
    const int64_t n = (int64_t)a.tokens * a.s.kv_heads * a.s.head_size;
    const dim3 grid((unsigned)((n + 255) / 256 < 148 * 64 ? (n + 255) / 256 : 148 * 64)), block(256);
    if (a.bf16_in) return launch_serving(append_kernel<uint16_t, uint16_t>, grid, block, 0, st, 1, a);
    if (a.s.dtype == AVA_BF16) return launch_serving(append_kernel<float, uint16_t>, grid, block, 0, st, 1, a);
    return launch_serving(append_kernel<float, float>, grid, block, 0, st, 1, a);
}

}  // namespace ava
