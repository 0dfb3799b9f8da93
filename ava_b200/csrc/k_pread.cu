// The read of new tokens over a store in pages: o = sum_j softmax_j(scale q . k_j) v_j.
//
// The plain form: one warp per (token, head), a key at a time with the running maximum and sum.
#include <cuda_runtime.h>

#include "ava_math.h"
#include "kernels.cuh"
#include "serving.cuh"

namespace ava {

namespace {

__device__ __forceinline__ float load_elem(const void* p, int64_t i, bool bf16) {
    return bf16 ? bf16_to_f(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}

template <int PER>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int t = (int)(item / a.heads), h = (int)(item % a.heads);
    if (blockIdx.x == 0)
        for (int r = threadIdx.x; r < a.rows; r += 256)
            if ((a.q_start[r] < 0 || a.q_start[r + 1] < a.q_start[r] || a.q_start[r + 1] > a.max_tokens) && a.status) atomicOr(a.status, AVA_PAGED_BAD_LENGTH);
    if (t >= a.max_tokens || t >= a.q_start[a.rows]) return;
    int lo = 0, hi = a.rows;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int r = lo;
    if (t >= a.q_start[r + 1]) return;   // the sums are not ascending
    const int64_t pos64 = (int64_t)a.cached[r] + (t - a.q_start[r]);
    const int64_t room = (int64_t)a.max_pages * a.s.page_size;
    if (a.cached[r] < 0 || t < a.q_start[r] || pos64 >= room) {
        if (a.status && lane == 0) atomicOr(a.status, AVA_PAGED_BAD_LENGTH);
        return;
    }
    const int pos = (int)pos64, kvh = h / a.group;
    int j0 = a.first ? max(a.first[r], 0) : 0;
    if (a.window > 0) j0 = max(j0, pos - a.window + 1);
    float q[PER], o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        q[i] = load_elem(a.q, (int64_t)t * a.q_token_stride + (int64_t)h * a.q_head_stride + lane + 32 * i, a.bf16_q);
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = j0; j <= pos; ++j) {
        const int page = a.table[(int64_t)r * a.max_pages + j / a.s.page_size];
        if (page < 0 || page >= a.s.n_pages) {
            if (a.status && lane == 0) atomicOr(a.status, AVA_PAGED_BAD_PAGE);
            continue;
        }
        const int64_t at = page * a.s.page_stride + kvh * a.s.head_stride + (j % a.s.page_size) * a.s.place_stride;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) x = fmaf(q[i], load_elem(a.s.k, at + lane + 32 * i, a.s.dtype == AVA_BF16), x);
#pragma unroll
        for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        x *= a.scale;
        const float mn = fmaxf(m, x), old = m == -INFINITY ? 0.0f : expf(m - mn), e = x == -INFINITY ? 0.0f : expf(x - mn);
        l = l * old + e;
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = fmaf(e, load_elem(a.s.v, at + lane + 32 * i, a.s.dtype == AVA_BF16), o[i] * old);
        m = mn;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int64_t to = (int64_t)t * a.out_token_stride + (int64_t)h * a.out_head_stride + lane;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (a.bf16_q) static_cast<uint16_t*>(a.out)[to + 32 * i] = f_to_bf16(o[i] * inv);
        else static_cast<float*>(a.out)[to + 32 * i] = o[i] * inv;
    }
    if (a.lse && lane == 0) a.lse[(int64_t)t * a.heads + h] = l > 0.0f ? m + logf(l) : -INFINITY;
}

}  // namespace

cudaError_t launch_paged_read(cudaStream_t st, const ReadArgs& a) {
    const dim3 grid((unsigned)(((int64_t)a.max_tokens * a.heads + 7) / 8)), block(256);
    if (a.s.head_size == 32) return launch_serving(read_kernel<1>, grid, block, 0, st, 1, a);
    if (a.s.head_size == 64) return launch_serving(read_kernel<2>, grid, block, 0, st, 1, a);
    return launch_serving(read_kernel<4>, grid, block, 0, st, 1, a);
}

}  // namespace ava
