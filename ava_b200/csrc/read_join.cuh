// What the two kernels that read over pages share behind read_split.cuh: the ends of cut stretches in the workspace, and
// joining them.
#pragma once
#include <cuda_runtime.h>

#include "bf16_hw.cuh"
#include "read_split.cuh"
#include "serving.cuh"

namespace ava {

constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Workspace of one worker's piece: the two ends that may be cut (0: goes on from the worker before, 1: goes on in the
// next), each MR rows of HS sums, then the rows' maxima (of scores times log2 e) and sums.
template <int HS, int MR>
struct Ends {
    static constexpr int FLOATS = MR * (HS + 2);
};

// Joining the ends of a stretch that was cut.  With the parts' maxima m_i (of scores times log2 e), sums l_i and mixes o_i:
//   m = max m_i, out = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i.
// A warp takes a row: the parts' maxima and sums a lane each, then all lanes the parts' mixes, whose loads depend on nothing
// but their weights, the first parts' not even on those.

// the parts k = k0, k0 + step, ... < n of a row: their common maximum, sum and mix
template <int HS, int MR>
__device__ __forceinline__ void join_parts(const float* ends, int w, int row, int n, int k0, int step, float& m, float& l, float (&o)[HS / 32]) {
    constexpr int PER = HS / 32, EARLY = 4;
    const int lane = threadIdx.x & 31;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = 0.0f;
    for (int b = k0; b < n; b += 32 * step) {
        const int mine = b + lane * step;
        auto part_of = [&](int k) { return ends + ((int64_t)(w + k) * 2 + (k == 0 ? 1 : 0)) * Ends<HS, MR>::FLOATS; };
        const int count = min(32, (n - b + step - 1) / step);
        float early[EARLY][PER];   // the first parts' mixes, asked for before the weights are known
#pragma unroll
        for (int k = 0; k < EARLY; ++k)
#pragma unroll
            for (int i = 0; i < PER; ++i) early[k][i] = k < count ? part_of(b + k * step)[row * HS + lane + 32 * i] : 0.0f;
        const float mk = mine < n ? part_of(mine)[MR * HS + row] : -INFINITY, lk = mine < n ? part_of(mine)[MR * HS + MR + row] : 0.0f;
        float now = mk;
#pragma unroll
        for (int x = 16; x; x >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, x));
        now = fmaxf(now, m);
        const float before = m == -INFINITY ? 0.0f : exp2_fast(m - now), weight = mk == -INFINITY ? 0.0f : exp2_fast(mk - now);
        float s = lk * weight;
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        l = l * before + s;
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] *= before;
#pragma unroll
        for (int k = 0; k < EARLY; ++k) {
            const float wk = __shfl_sync(0xffffffffu, weight, k);
#pragma unroll
            for (int i = 0; i < PER; ++i) o[i] = fmaf(early[k][i], wk, o[i]);
        }
#pragma unroll 4
        for (int k = EARLY; k < count; ++k) {
            const float wk = __shfl_sync(0xffffffffu, weight, k);
            const float* part = part_of(b + k * step) + row * HS + lane;
#pragma unroll
            for (int i = 0; i < PER; ++i) o[i] = fmaf(part[32 * i], wk, o[i]);
        }
        m = now;
    }
}
template <int HS>
__device__ __forceinline__ void join_write(const ReadArgs& a, int start, int head, int m_row, float m, float l, const float (&o)[HS / 32]) {
    const int lane = threadIdx.x & 31;
    const float inv = l > 0.0f ? 1.0f / l : l;
    const int i = m_row / a.group, h = head * a.group + (m_row - i * a.group);
    const int64_t to = (int64_t)(start + i) * a.out_token_stride + (int64_t)h * a.out_head_stride + lane;
#pragma unroll
    for (int c = 0; c < HS / 32; ++c) {
        if (a.bf16_q) static_cast<uint16_t*>(a.out)[to + 32 * c] = bf16_rn_hw(o[c] * inv);
        else static_cast<float*>(a.out)[to + 32 * c] = o[c] * inv;
    }
    if (a.lse && lane == 0) a.lse[(int64_t)(start + i) * a.heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

}  // namespace ava
