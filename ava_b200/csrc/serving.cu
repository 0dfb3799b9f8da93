// Entry points of the serving operators (include/ava_engine.h, "serving from pages"): argument checks, the device of the
// call, the launch.  Nothing is allocated or waited for, and nothing is shared between threads but the error text's own
// thread-local string.
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <string>
#include <utility>

#include "../../include/ava_engine.h"
#include "serving.cuh"

namespace {

using namespace ava;

thread_local std::string g_serving_error;

int fail(int code, const char* call, const char* why) noexcept {
    try {
        g_serving_error = std::string(call) + ": " + why;
    } catch (...) {   // no memory for the text: the code says it
    }
    return code;
}

// Devices of this process (their number does not change once there are any).
int device_count() {
    static std::atomic<int> known{0};
    int n = known.load(std::memory_order_relaxed);
    if (n > 0) return n;
    if (cudaGetDeviceCount(&n) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    known.store(n, std::memory_order_relaxed);
    return n;
}

// The call's device for as long as it lives; the thread's own comes back.
struct OnDevice {
    int before = -1;
    bool ok = false;
    explicit OnDevice(int device) {
        if (device < 0 || device >= device_count()) return;
        if (cudaGetDevice(&before) != cudaSuccess) return;
        ok = before == device || cudaSetDevice(device) == cudaSuccess;
        if (before == device) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

constexpr const char* NO_DEVICE = "no such CUDA device (this library has no CPU path)";

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int launched(cudaError_t rc, const char* call) {
    if (rc == cudaSuccess) return AVA_OK;
    cudaGetLastError();
    return fail(AVA_ERR_CUDA, call, cudaGetErrorString(rc));
}

int sm_count(int device) {
    int n = 0;
    return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess ? n : 0;
}

// Indexes of requests, tokens and pages are 32 bits in the kernels, with room for a block's stride behind the last.
constexpr int32_t MOST_ROWS = 1 << 24, MOST_TOKENS = 1 << 30, MOST_PAGES = 1 << 30;

// Whether an array that is written has no element twice: extents and strides of its dimensions but the innermost, which
// holds `inner` adjacent elements.  Sorted by stride each must reach over all inside it (a broadcast has stride 0).
template <int N>
bool distinct(int64_t inner, int64_t (&n)[N], int64_t (&stride)[N]) {
    for (int i = 1; i < N; ++i)
        for (int j = i; j > 0 && stride[j] < stride[j - 1]; --j) {
            std::swap(stride[j], stride[j - 1]);
            std::swap(n[j], n[j - 1]);
        }
    __int128 reach = inner;
    for (int i = 0; i < N; ++i) {
        if (n[i] <= 1) continue;
        if (stride[i] < reach) return false;
        reach += static_cast<__int128>(n[i] - 1) * stride[i];
    }
    return true;
}

// What append and attend need of a store; nullptr: fine.
const char* store_fault(const ava_paged_store* s) {
    if (!s || !s->k || !s->v) return "a store without its pools";
    if (s->dtype != AVA_F32 && s->dtype != AVA_BF16) return "the store's dtype is AVA_F32 or AVA_BF16";
    if (s->n_pages <= 0 || s->kv_heads <= 0 || s->page_size <= 0 || s->head_size <= 0) return "the store's sizes must be positive";
    if (s->page_stride < 0 || s->head_stride < 0 || s->place_stride < s->head_size) return "the store's strides: not negative, places at least a head apart";
    if (static_cast<int64_t>(s->kv_heads) * s->head_size > 1 << 30) return "the store's heads: at most 2^30 channels a token";
    const uintptr_t el = s->dtype == AVA_BF16 ? 2 : 4;
    if (!aligned(s->k, el) || !aligned(s->v, el)) return "the store's pools must be aligned to their elements";
    return nullptr;
}

}  // namespace

extern "C" {

const char* ava_serving_last_error(void) { return g_serving_error.c_str(); }

int ava_paged_plan(int device, void* stream, const int32_t* cached, const int32_t* fresh, int32_t rows, int32_t page_size, int32_t n_pages,
                   int32_t* table, int32_t max_pages, const int32_t* owned, int32_t* owned_out, int32_t* free_list, const int32_t* free_count,
                   int32_t* free_count_out, int32_t trim, int32_t* q_start, int64_t* slot, int32_t* pos, int32_t* row, int32_t max_tokens,
                   uint32_t* status) {
    static const char* const call = "ava_paged_plan";
    if (!cached || !fresh || !table || !owned || !owned_out || !free_list || !free_count || !free_count_out || !q_start || (!slot && max_tokens > 0))
        return fail(AVA_ERR_ARG, call, "null pointer");
    if (rows <= 0 || page_size <= 0 || n_pages <= 0 || max_pages <= 0 || max_tokens < 0) return fail(AVA_ERR_ARG, call, "sizes must be positive");
    const void* words[] = {cached, fresh, table, owned, owned_out, free_list, free_count, free_count_out, q_start, pos, row, status};
    for (const void* w : words)
        if (!aligned(w, 4)) return fail(AVA_ERR_ARG, call, "the lists must be 4-byte aligned");
    if (!aligned(slot, 8)) return fail(AVA_ERR_ARG, call, "slot must be 8-byte aligned");
    if (rows > MOST_ROWS || max_tokens > MOST_TOKENS || n_pages > MOST_PAGES) return fail(AVA_NOT_APPLICABLE, call, "at most 2^24 requests, 2^30 tokens and 2^30 pages");
    OnDevice dev(device);
    if (!dev.ok) return fail(AVA_ERR_CUDA, call, NO_DEVICE);
    PlanArgs a{};
    a.cached = cached; a.fresh = fresh; a.owned = owned; a.free_count = free_count;
    a.table = table; a.owned_out = owned_out; a.free_list = free_list; a.free_count_out = free_count_out; a.q_start = q_start;
    a.slot = slot; a.pos = pos; a.row = row; a.status = status;
    a.rows = rows; a.page_size = page_size; a.n_pages = n_pages; a.max_pages = max_pages; a.max_tokens = max_tokens; a.trim = trim != 0;
    return launched(launch_paged_plan(device, static_cast<cudaStream_t>(stream), a), call);
}

int ava_paged_append(int device, void* stream, const ava_paged_store* store, const void* k, const void* v, int32_t dtype, int64_t token_stride,
                     int64_t head_stride, const int64_t* slot, int32_t tokens, uint32_t* status) {
    static const char* const call = "ava_paged_append";
    if (const char* why = store_fault(store)) return fail(AVA_ERR_ARG, call, why);
    if (tokens < 0) return fail(AVA_ERR_ARG, call, "tokens must not be negative");
    if (tokens > 0 && (!k || !v || !slot)) return fail(AVA_ERR_ARG, call, "null pointer");
    if (dtype != AVA_F32 && dtype != AVA_BF16) return fail(AVA_ERR_ARG, call, "dtype is AVA_F32 or AVA_BF16");
    if (token_stride < 0 || head_stride < 0) return fail(AVA_ERR_ARG, call, "strides must not be negative");
    int64_t extents[] = {store->n_pages, store->kv_heads, store->page_size}, strides[] = {store->page_stride, store->head_stride, store->place_stride};
    if (!distinct(store->head_size, extents, strides)) return fail(AVA_ERR_ARG, call, "a store that is written must not overlap itself");
    const uintptr_t el = dtype == AVA_BF16 ? 2 : 4;
    if (!aligned(k, el) || !aligned(v, el)) return fail(AVA_ERR_ARG, call, "k and v must be aligned to their elements");
    if (!aligned(slot, 8) || !aligned(status, 4)) return fail(AVA_ERR_ARG, call, "slot must be 8-byte and status 4-byte aligned");
    if (dtype == AVA_BF16 && store->dtype == AVA_F32) return fail(AVA_NOT_APPLICABLE, call, "bf16 rows into an f32 store");
    OnDevice dev(device);
    if (!dev.ok) return fail(AVA_ERR_CUDA, call, NO_DEVICE);
    if (tokens == 0) return AVA_OK;
    AppendArgs a{};
    a.s = *store; a.k = k; a.v = v; a.token_stride = token_stride; a.head_stride = head_stride; a.slot = slot; a.status = status;
    a.tokens = tokens; a.bf16_in = dtype == AVA_BF16;
    return launched(launch_paged_append(device, static_cast<cudaStream_t>(stream), a), call);
}

int64_t ava_paged_attend_workspace(int device, int32_t head_size) {
    static const char* const call = "ava_paged_attend_workspace";
    if (head_size != 32 && head_size != 64 && head_size != 128) return fail(AVA_NOT_APPLICABLE, call, "head sizes 32, 64 and 128"), -1;
    OnDevice dev(device);
    if (!dev.ok) return fail(AVA_ERR_CUDA, call, NO_DEVICE), -1;
    const int sms = sm_count(device);
    if (sms <= 0) return fail(AVA_ERR_CUDA, call, NO_DEVICE), -1;
    return paged_read_workspace(head_size, sms);
}

int ava_paged_attend(int device, void* stream, const ava_paged_store* store, const void* q, int32_t dtype, int64_t q_token_stride,
                     int64_t q_head_stride, int32_t heads, const int32_t* table, int32_t max_pages, const int32_t* cached, const int32_t* first,
                     const int32_t* q_start, int32_t rows, int32_t max_tokens, int32_t max_fresh, float scale, int32_t window, void* out,
                     int64_t out_token_stride, int64_t out_head_stride, float* lse, void* workspace, int64_t workspace_bytes, uint32_t* status) {
    static const char* const call = "ava_paged_attend";
    if (const char* why = store_fault(store)) return fail(AVA_ERR_ARG, call, why);
    if (!table || !cached || !q_start || (max_tokens > 0 && (!q || !out))) return fail(AVA_ERR_ARG, call, "null pointer");
    if (rows <= 0 || max_pages <= 0 || max_tokens < 0 || max_fresh < 0 || heads <= 0 || window < 0) return fail(AVA_ERR_ARG, call, "sizes must be positive");
    if (heads % store->kv_heads) return fail(AVA_ERR_ARG, call, "heads must be a multiple of the store's");
    if (dtype != AVA_F32 && dtype != AVA_BF16) return fail(AVA_ERR_ARG, call, "dtype is AVA_F32 or AVA_BF16");
    if (q_token_stride < 0 || q_head_stride < 0 || out_token_stride < 0 || out_head_stride < store->head_size)
        return fail(AVA_ERR_ARG, call, "strides must not be negative, and out's heads at least a head apart");
    if (!(scale == scale) || scale > 3.0e38f || scale < -3.0e38f) return fail(AVA_ERR_ARG, call, "scale must be finite");
    const uintptr_t el = dtype == AVA_BF16 ? 2 : 4;
    if (!aligned(q, el) || !aligned(out, el)) return fail(AVA_ERR_ARG, call, "q and out must be aligned to their elements");
    const void* words[] = {table, cached, first, q_start, lse, status};
    for (const void* w : words)
        if (!aligned(w, 4)) return fail(AVA_ERR_ARG, call, "lists, lse and status must be 4-byte aligned");
    if (store->head_size != 32 && store->head_size != 64 && store->head_size != 128) return fail(AVA_NOT_APPLICABLE, call, "head sizes 32, 64 and 128");
    int64_t extents[] = {max_tokens, heads}, strides[] = {out_token_stride, out_head_stride};
    if (!distinct(store->head_size, extents, strides)) return fail(AVA_ERR_ARG, call, "out must not overlap itself");
    // the store is read in pieces of 16 bytes
    const int64_t piece = store->dtype == AVA_BF16 ? 8 : 4;
    if (!aligned(store->k, 16) || !aligned(store->v, 16) || store->page_stride % piece || store->head_stride % piece || store->place_stride % piece)
        return fail(AVA_ERR_ARG, call, "the store's pools and strides must be multiples of 16 bytes");
    if (dtype == AVA_BF16 && store->dtype == AVA_F32) return fail(AVA_NOT_APPLICABLE, call, "bf16 queries over an f32 store");
    if (rows > MOST_ROWS || static_cast<int64_t>(max_tokens) * heads > MOST_TOKENS) return fail(AVA_NOT_APPLICABLE, call, "at most 2^24 requests and 2^30 tokens times heads");
    OnDevice dev(device);
    if (!dev.ok) return fail(AVA_ERR_CUDA, call, NO_DEVICE);
    const int sms = sm_count(device);
    if (sms <= 0) return fail(AVA_ERR_CUDA, call, NO_DEVICE);
    if (!workspace || workspace_bytes < paged_read_workspace(store->head_size, sms) || !aligned(workspace, 16)) return fail(AVA_ERR_ARG, call, "workspace: too small, missing or not 16-byte aligned");
    if (max_tokens == 0) return AVA_OK;
    ReadArgs a{};
    a.s = *store; a.q = q; a.out = out; a.lse = lse;
    a.q_token_stride = q_token_stride; a.q_head_stride = q_head_stride; a.out_token_stride = out_token_stride; a.out_head_stride = out_head_stride;
    a.table = table; a.cached = cached; a.first = first; a.q_start = q_start; a.status = status; a.scale = scale;
    a.heads = heads; a.group = heads / store->kv_heads; a.max_pages = max_pages; a.rows = rows; a.max_tokens = max_tokens; a.max_fresh = max_fresh;
    a.window = window; a.bf16_q = dtype == AVA_BF16;
    return launched(launch_paged_read(device, static_cast<cudaStream_t>(stream), a, workspace, sms), call);
}

int ava_verify_drafts(int device, void* stream, const float* p, int64_t p_stride, const float* q, int64_t q_stride, const uint32_t* tok,
                      const int32_t* q_start, int32_t rows, int32_t max_tokens, int32_t vocab, const double* uniform, int32_t max_out, uint32_t* out,
                      int32_t* n_out, uint32_t* status) {
    static const char* const call = "ava_verify_drafts";
    if (!q_start || !out || !n_out || (max_tokens > 0 && (!p || !tok))) return fail(AVA_ERR_ARG, call, "null pointer");
    if (rows <= 0 || max_tokens < 0 || vocab <= 0 || max_out <= 0) return fail(AVA_ERR_ARG, call, "sizes must be positive");
    if (p_stride < vocab || (q && q_stride < vocab)) return fail(AVA_ERR_ARG, call, "rows of probabilities must be at least a vocabulary apart");
    if (q && !uniform) return fail(AVA_ERR_ARG, call, "greedy drafts have no probabilities: q must be NULL when uniform is");
    const void* words[] = {p, q, tok, q_start, out, n_out, status};
    for (const void* w : words)
        if (!aligned(w, 4)) return fail(AVA_ERR_ARG, call, "arrays must be 4-byte aligned");
    if (!aligned(uniform, 8)) return fail(AVA_ERR_ARG, call, "uniform must be 8-byte aligned");
    if (vocab > (1 << 30) || rows > MOST_ROWS) return fail(AVA_NOT_APPLICABLE, call, "a vocabulary of at most 2^30 tokens and 2^24 requests");
    OnDevice dev(device);
    if (!dev.ok) return fail(AVA_ERR_CUDA, call, NO_DEVICE);
    VerifyArgs a{};
    a.p = p; a.q = q; a.p_stride = p_stride; a.q_stride = q_stride; a.tok = tok; a.q_start = q_start; a.uniform = uniform; a.out = out; a.n_out = n_out;
    a.status = status; a.rows = rows; a.max_tokens = max_tokens; a.vocab = vocab; a.max_out = max_out;
    return launched(launch_verify(device, static_cast<cudaStream_t>(stream), a), call);
}

}  // extern "C"
