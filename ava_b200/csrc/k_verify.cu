// Drafted tokens against the target's probabilities (the form that keeps the target's own distribution).
//
// A draft d drawn from q is kept with probability min(1, p(d) / q(d)); the first refused place is redrawn from
// max(p - q, 0), whose mass is what the kept drafts leave over, so every token is distributed as p.  All of it is decided
// by comparisons: u q(d) < p(d) per draft (a handful of gathered values), then one running sum over the vocabulary for
// the token behind the kept ones.  The bytes are that one row of p and, after a refusal, of q.
//
// A cluster of blocks per request (distributed shared memory joins them; no workspace): each block sums a contiguous part
// of the vocabulary in f64, tile by tile of 128 * m tokens per warp, the parts' sums say in which part the drawn place
// lies, the tiles' sums in which tile, and one warp walks that tile again.  f64 throughout: a running sum over 10^4 and
// more tokens decides between neighbours, and 24 bits would move the border by more than a neighbour's width.
// Greedy: the blocks of the cluster take the places in turn, each the largest of its row.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "kernels.cuh"
#include "serving.cuh"

namespace ava {

namespace {

namespace cg = cooperative_groups;

constexpr int V_THREADS = 256, V_WARPS = V_THREADS / 32, V_TILES = 32, V_PARTS = 8;

struct Row {
    const float *p, *q;   // q nullptr: p alone
    int without;          // a token that does not count (a certain draft that was refused), or -1
};

__device__ __forceinline__ double weight(float p, float q) {
    const double x = p > 0.0f ? (double)p : 0.0;
    const double y = q > 0.0f ? (double)q : 0.0;
    return fmax(x - y, 0.0);
}

// p and q of tokens j .. j + 3 (those at or beyond hi read as 0)
__device__ __forceinline__ void load4(const Row& w, int j, int hi, bool wide, float (&p)[4], float (&q)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = q[i] = 0.0f;
    if (wide && j + 4 <= hi) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(w.p + j));
        p[0] = u.x; p[1] = u.y; p[2] = u.z; p[3] = u.w;
        if (w.q) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(w.q + j));
            q[0] = v.x; q[1] = v.y; q[2] = v.z; q[3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j + i < hi) {
                p[i] = __ldg(w.p + j + i);
                if (w.q) q[i] = __ldg(w.q + j + i);
            }
    }
}
__device__ __forceinline__ void weights4(const Row& w, int j, const float (&p)[4], const float (&q)[4], double (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = j + i == w.without ? 0.0 : weight(p[i], q[i]);
}

// The block's part [lo, hi) in tiles of 128 * m tokens: their sums.  A warp walks its V_TILES / V_WARPS tiles together, so
// that their loads are in flight at once (one tile after the other waited for memory tile by tile: 63 us for 256 requests
// of 32768 tokens; 512 threads of 128 registers, one block to an SM and so wave after wave: 37 us).
__device__ __forceinline__ void tile_sums(const Row& w, int lo, int hi, int m, bool wide, double* sums) {
    constexpr int MINE = V_TILES / V_WARPS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double s[MINE];
#pragma unroll
    for (int k = 0; k < MINE; ++k) s[k] = 0.0;
#pragma unroll 1
    for (int b = 0; b < m; ++b) {
        float p[MINE][4], q[MINE][4];
#pragma unroll
        for (int k = 0; k < MINE; ++k) load4(w, lo + ((warp * MINE + k) * m + b) * 128 + lane * 4, hi, wide, p[k], q[k]);
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            double x[4];
            weights4(w, lo + ((warp * MINE + k) * m + b) * 128 + lane * 4, p[k], q[k], x);
            s[k] += (x[0] + x[1]) + (x[2] + x[3]);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int k = 0; k < MINE; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < MINE; ++k) sums[warp * MINE + k] = s[k];
}

__global__ void __launch_bounds__(V_THREADS, 4) verify_kernel(const VerifyArgs a) {
    pdl_enter();
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int r = blockIdx.x / parts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ double sums[V_TILES];
    __shared__ double totals[2][V_PARTS];   // of every block's part, written by that block; once more after a fall back
    __shared__ int s_kept, s_pick;
    __shared__ float best_x[V_WARPS];
    __shared__ int best_i[V_WARPS];

    const int start = a.q_start[r], end = a.q_start[r + 1], n = end - start - 1;
    uint32_t* out = a.out + (int64_t)r * a.max_out;
    // every block of the cluster takes the same way out: nobody is left waiting
    const bool bad = start < 0 || end < start || end > a.max_tokens || n >= a.max_out;
    if (bad || n < 0) {
        if (part == 0) {
            for (int i = tid; i < a.max_out; i += V_THREADS) out[i] = AVA_NO_TOKEN;
            if (tid == 0) {
                a.n_out[r] = 0;
                if (bad && a.status) atomicOr(a.status, AVA_PAGED_BAD_LENGTH);
            }
        }
        return;
    }
    const uint32_t* draft = a.tok + start + 1;

    if (!a.uniform) {
        for (int i = part; i <= n; i += parts) {
            const float* p = a.p + (int64_t)(start + i) * a.p_stride;
            float bx = -INFINITY;
            int bi = a.vocab;
            for (int j = tid; j < a.vocab; j += V_THREADS) {
                const float x = p[j];
                if (x > bx || (x == bx && j < bi)) {
                    bx = x;
                    bi = j;
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const float x = __shfl_xor_sync(0xffffffffu, bx, o);
                const int k = __shfl_xor_sync(0xffffffffu, bi, o);
                if (x > bx || (x == bx && k < bi)) {
                    bx = x;
                    bi = k;
                }
            }
            if (lane == 0) {
                best_x[warp] = bx;
                best_i[warp] = bi;
            }
            __syncthreads();
            if (tid == 0) {
                for (int k = 1; k < V_WARPS; ++k)
                    if (best_x[k] > bx || (best_x[k] == bx && best_i[k] < bi)) {
                        bx = best_x[k];
                        bi = best_i[k];
                    }
                out[i] = bi < a.vocab ? (uint32_t)bi : 0u;   // nothing but NaN: the first token, as the host's sampler takes it
            }
            __syncthreads();
        }
        cluster.sync();
        if (part == 0 && warp == 0) {
            int kept = n;
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int i = i0 + lane;
                const bool off = i < n && out[i] != draft[i];
                if (i < n && draft[i] >= (uint32_t)a.vocab && a.status) atomicOr(a.status, AVA_PAGED_BAD_TOKEN);
                const unsigned who = __ballot_sync(0xffffffffu, off);
                if (who && kept == n) kept = i0 + __ffs(who) - 1;
            }
            for (int i = kept + 1 + lane; i < a.max_out; i += 32) out[i] = AVA_NO_TOKEN;
            if (lane == 0) a.n_out[r] = kept + 1;
        }
        return;
    }

    if (warp == 0) {   // the kept drafts: every block finds them for itself
        int kept = n;
        for (int i0 = 0; i0 < n && kept == n; i0 += 32) {
            const int i = i0 + lane;
            bool no = false;
            if (i < n) {
                const uint32_t d = draft[i];
                if (d >= (uint32_t)a.vocab) {
                    no = true;
                    if (part == 0 && a.status) atomicOr(a.status, AVA_PAGED_BAD_TOKEN);
                } else {
                    const float pd = a.p[(int64_t)(start + i) * a.p_stride + d];
                    const float qd = a.q ? a.q[(int64_t)(start + i) * a.q_stride + d] : 1.0f;
                    no = !(a.uniform[start + i] * (qd > 0.0f ? (double)qd : 0.0) < (double)pd);
                }
            }
            const unsigned who = __ballot_sync(0xffffffffu, no);
            if (who) kept = i0 + __ffs(who) - 1;
        }
        if (lane == 0) {
            s_kept = kept;
            s_pick = -1;
        }
    }
    __syncthreads();
    const int kept = s_kept;
    const double u = a.uniform[end - 1];
    Row w;
    w.p = a.p + (int64_t)(start + kept) * a.p_stride;
    w.q = kept < n && a.q ? a.q + (int64_t)(start + kept) * a.q_stride : nullptr;
    w.without = kept < n && !a.q && draft[kept] < (uint32_t)a.vocab ? (int)draft[kept] : -1;
    // parts of whole groups of four tokens, tiles of 128 * m
    const int span = ((a.vocab + parts - 1) / parts + 3) & ~3;
    const int lo = min(part * span, a.vocab), hi = min(lo + span, a.vocab), m = (span + 128 * V_TILES - 1) / (128 * V_TILES);

    double whole = 0.0, before = 0.0;
    int mine = -1;
    for (int attempt = 0; attempt < 2; ++attempt) {
        const bool wide = !((reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.q)) & 15);
        tile_sums(w, lo, hi, m, wide, sums);
        __syncthreads();
        if (warp == 0) {
            double s = sums[lane];
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane < parts) *cluster.map_shared_rank(&totals[attempt][part], lane) = s;
        }
        cluster.sync();   // after it a block reads its own memory only, so the others may leave
        whole = 0.0;
        for (int k = 0; k < parts; ++k) whole += totals[attempt][k];
        // the part the drawn place lies in: the first whose running sum exceeds u * whole, else the last with any mass
        const double target = u * whole;
        double run = 0.0;
        bool found = false;
        mine = -1;
        for (int k = 0; k < parts && !found; ++k) {
            const double s = totals[attempt][k];
            if (s > 0.0) {          // a part without mass is never it, whatever the number drawn (below 0 too)
                mine = k;
                before = run;
                run += s;
                found = run > target;
            }
        }
        if ((whole > 0.0 && whole < INFINITY) || (!w.q && w.without < 0)) break;
        w.q = nullptr;    // no mass in the difference: the target's own
        w.without = -1;
    }
    const bool mass = whole > 0.0 && whole < INFINITY;
    if (part != (mass ? mine : 0)) return;
    const double target = u * whole;
    if (mass && warp == 0) {
        // the tile, then the token: by running sums over lanes, in token order
        const double own = sums[lane];
        double inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, before + inc > target && own > 0.0);
        const unsigned some = __ballot_sync(0xffffffffu, own > 0.0);
        const int tile = over ? __ffs(over) - 1 : 31 - __clz(some);
        double at = __shfl_sync(0xffffffffu, before + (inc - own), tile);
        const bool wide = !((reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.q)) & 15);
        int pick = -1, last = -1;
        for (int b = 0; b < m && pick < 0; ++b) {
            const int j = lo + tile * 128 * m + b * 128 + lane * 4;
            float p[4], q[4];
            double x[4];
            load4(w, j, hi, wide, p, q);
            weights4(w, j, p, q, x);
            const double four = ((x[0] + x[1]) + x[2]) + x[3];
            double sum = four;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += y;
            }
            double run = at + (sum - four);
            int first = -1, some_here = -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                run += x[i];
                if (x[i] > 0.0) {
                    some_here = j + i;
                    if (first < 0 && run > target) first = j + i;
                }
            }
            const unsigned hit = __ballot_sync(0xffffffffu, first >= 0), any = __ballot_sync(0xffffffffu, some_here >= 0);
            if (any) last = __shfl_sync(0xffffffffu, some_here, 31 - __clz(any));
            if (hit) pick = __shfl_sync(0xffffffffu, first, __ffs(hit) - 1);
            at += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) s_pick = pick >= 0 ? pick : last;   // rounding put the border behind the tile: its last token with mass
    }
    __syncthreads();
    for (int i = tid; i < a.max_out; i += V_THREADS) out[i] = i < kept ? draft[i] : i == kept && s_pick >= 0 ? (uint32_t)s_pick : AVA_NO_TOKEN;
    if (tid == 0) {
        a.n_out[r] = kept + 1;
        if (!mass && a.status) atomicOr(a.status, AVA_PAGED_NO_MASS);
    }
}

}  // namespace

cudaError_t launch_verify(int device, cudaStream_t st, const VerifyArgs& a) {
    // blocks per request: enough to have about four on every SM (one request's row is then read by eight SMs), one for
    // the larger batches, whose requests fill the GPU by themselves
    int cluster = V_PARTS;
    while (cluster > 1 && (int64_t)a.rows * cluster > 4 * 148) cluster >>= 1;
    return launch_serving<verify_kernel>(device, dim3(a.rows * cluster), dim3(V_THREADS), 0, st, cluster, a);
}

}  // namespace ava
