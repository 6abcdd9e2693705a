// C ABI of the operators beside the KDA forward: argument validation in front of the launches.
#include <float.h>

#include <array>
#include <initializer_list>

#include "fkda_internal.h"

namespace {

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Strides (elements) of a bf16 tensor that is read in tiles, dimensions outermost first: those longer than one step by positive
// multiples of 16 bytes; the others are never stepped, but a tensor map wants something valid for them too.
bool tile_strides(int64_t* stride, std::initializer_list<int64_t> sizes) {
    int i = 0;
    for (const int64_t n : sizes) {
        if (n <= 1) stride[i] = 8;
        if (stride[i] <= 0 || stride[i] % 8 != 0 || stride[i] >= (int64_t)1 << 39) return false;
        ++i;
    }
    return true;
}
// The same for a tensor that is only written, in 16-byte pieces.
bool row_strides(const int64_t* stride, std::initializer_list<int64_t> sizes) {
    int i = 0;
    for (const int64_t n : sizes) {
        if (n > 1 && (stride[i] <= 0 || stride[i] % 8 != 0)) return false;
        ++i;
    }
    return true;
}
// Kernels multiply scores, masked ones of minus infinity among them, by scale times log2(e), which therefore is neither 0 (where a smaller
// number would be flushed to) nor infinite.
bool softmax_scale(float x) { return x >= FLT_MIN && x <= FLT_MAX / 2; }
bool in_range(int64_t x, int64_t lo, int64_t hi) { return lo <= x && x <= hi; }
constexpr int64_t kMost = 0x7fffffff;

template <typename Launch>
int enqueue(const Launch& launch) {
    int launches = 0;
    const int rc = launch(&launches);
    if (rc == FKDA_OK) fkda::set_last_launch_count(launches);
    return rc;
}

int check(fkda_linear_params* p) {
    if (!in_range(p->B, 1, kMost) || !in_range(p->T, 0, kMost - 64) || !in_range(p->H, 1, 65535) || !in_range(p->Hk, 1, p->H) || p->H % p->Hk != 0 ||
        !in_range(p->N, 1, kMost))
        return FKDA_ERR_BAD_SHAPE;
    if (p->cu_seqlens != nullptr && p->B != 1) return FKDA_ERR_VARLEN_BATCH;
    if (p->cu_seqlens == nullptr && p->N != p->B) return FKDA_ERR_BAD_SHAPE;
    if (p->state_dtype != FKDA_STATE_BF16 && p->state_dtype != FKDA_STATE_FP32) return FKDA_ERR_BAD_STATE_DTYPE;
    if (p->T > 0 && (!p->q || !p->k || !p->v || !p->g || !p->out)) return FKDA_ERR_NULL_POINTER;
    if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->out, 16) || !aligned(p->g, 4) || !aligned(p->initial_state, 16) ||
        !aligned(p->final_state, 16) || !aligned(p->cu_seqlens, 8))
        return FKDA_ERR_ALIGNMENT;
    if (!tile_strides(p->q_stride, {p->B, p->T, p->Hk}) || !tile_strides(p->k_stride, {p->B, p->T, p->Hk}) || !tile_strides(p->v_stride, {p->B, p->T, p->H}) ||
        !tile_strides(p->out_stride, {p->B, p->T, p->H}))
        return FKDA_ERR_ALIGNMENT;
    return FKDA_OK;
}

int check(fkda_latent_params* p) {
    if (!in_range(p->B, 1, kMost) || !in_range(p->T, 0, kMost - 256) || !in_range(p->Tk, 0, kMost - 256) || !in_range(p->H, 1, 65535) || !in_range(p->N, 1, kMost))
        return FKDA_ERR_BAD_SHAPE;
    if ((p->cu_seqlens != nullptr) != (p->cu_seqlens_k != nullptr)) return FKDA_ERR_NULL_POINTER;
    if (p->cu_seqlens != nullptr && p->B != 1) return FKDA_ERR_VARLEN_BATCH;
    if (p->cu_seqlens == nullptr && p->N != p->B) return FKDA_ERR_BAD_SHAPE;
    if (!softmax_scale(p->scale)) return FKDA_ERR_BAD_SCALE;
    if (p->T > 0 && (!p->q || !p->out)) return FKDA_ERR_NULL_POINTER;
    if (p->Tk > 0 && (!p->k || !p->k_rope || !p->v)) return FKDA_ERR_NULL_POINTER;
    if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->k_rope, 16) || !aligned(p->v, 16) || !aligned(p->out, 16) || !aligned(p->lse, 4) ||
        !aligned(p->cu_seqlens, 8) || !aligned(p->cu_seqlens_k, 8))
        return FKDA_ERR_ALIGNMENT;
    if (!tile_strides(p->q_stride, {p->B, p->T, p->H}) || !tile_strides(p->k_stride, {p->B, p->Tk, p->H}) || !tile_strides(p->v_stride, {p->B, p->Tk, p->H}) ||
        !tile_strides(p->k_rope_stride, {p->B, p->Tk}) || !row_strides(p->out_stride, {p->B, p->T, p->H}))
        return FKDA_ERR_ALIGNMENT;
    return FKDA_OK;
}

int check(fkda_latent_decode_params* p) {
    if (!in_range(p->B, 0, kMost) || !in_range(p->Tq, 0, kMost) || !in_range(p->H, 1, 65535) || !in_range(p->Tq * p->H, 0, kMost - 64) ||
        !in_range(p->pages, 0, kMost) || !in_range(p->page_size, 16, 1 << 20) || p->page_size % 16 != 0 || !in_range(p->max_pages, 0, kMost) ||
        p->max_pages * p->page_size > kMost - 64)
        return FKDA_ERR_BAD_SHAPE;
    if (!softmax_scale(p->scale)) return FKDA_ERR_BAD_SCALE;
    if (p->B * p->Tq == 0) return FKDA_OK;
    if (!p->q || !p->cache_lens || !p->out || (p->max_pages > 0 && (!p->block_table || !p->cache)) || (p->max_pages > 0 && p->pages < 1)) return FKDA_ERR_NULL_POINTER;
    if (!aligned(p->q, 16) || !aligned(p->cache, 16) || !aligned(p->out, 16) || !aligned(p->lse, 4) || !aligned(p->block_table, 4) || !aligned(p->cache_lens, 4))
        return FKDA_ERR_ALIGNMENT;
    if (!tile_strides(p->q_stride, {p->B, p->Tq * p->H}) || !tile_strides(p->cache_stride, {p->pages, p->page_size}) ||
        !row_strides(p->out_stride, {p->B, p->Tq * p->H}))
        return FKDA_ERR_ALIGNMENT;
    return FKDA_OK;
}

template <typename Params>
int workspace_missing(const Params& p, size_t need) {
    return need > 0 && (p.workspace == nullptr || p.workspace_bytes < need || !aligned(p.workspace, 256)) ? FKDA_ERR_WORKSPACE : FKDA_OK;
}

thread_local int g_starve_ms = 0;
constexpr int kMaxDevices = 64;
// What this thread was last told of the waits that gave up on each device: one thread's question takes no answer from another.
thread_local std::array<uint32_t, 3> g_seen[kMaxDevices] = {};

}  // namespace

int fkda::starve_next() {
    const int ms = g_starve_ms;
    g_starve_ms = 0;
    return ms;
}

extern "C" {

size_t fkda_linear_workspace_bytes(const fkda_linear_params* p) {
    if (p == nullptr || p->B <= 0 || p->T < 0 || p->H <= 0 || p->N <= 0) return 0;
    return fkda::linear_workspace(*p);
}

int fkda_linear_attention_fwd(const fkda_linear_params* given, void* stream) {
    fkda::set_last_launch_count(0);
    if (given == nullptr) return FKDA_ERR_NULL_POINTER;
    fkda_linear_params p = *given;
    int rc = check(&p);
    if (rc == FKDA_OK) rc = workspace_missing(p, fkda_linear_workspace_bytes(&p));
    if (rc != FKDA_OK) return rc;
    if (p.T == 0 && p.final_state == nullptr) return FKDA_OK;
    return enqueue([&](int* n) { return fkda::launch_linear(p, static_cast<cudaStream_t>(stream), n); });
}

int fkda_latent_attention_fwd(const fkda_latent_params* given, void* stream) {
    fkda::set_last_launch_count(0);
    if (given == nullptr) return FKDA_ERR_NULL_POINTER;
    fkda_latent_params p = *given;
    const int rc = check(&p);
    if (rc != FKDA_OK || p.T == 0) return rc;
    return enqueue([&](int* n) { return fkda::launch_latent_prompt(p, static_cast<cudaStream_t>(stream), n); });
}

size_t fkda_latent_decode_workspace_bytes(const fkda_latent_decode_params* p) {
    if (p == nullptr || p->B <= 0 || p->Tq <= 0 || p->H <= 0) return 0;
    return fkda::latent_decode_workspace(*p);
}

int fkda_latent_attention_decode(const fkda_latent_decode_params* given, void* stream) {
    fkda::set_last_launch_count(0);
    if (given == nullptr) return FKDA_ERR_NULL_POINTER;
    fkda_latent_decode_params p = *given;
    int rc = check(&p);
    if (rc != FKDA_OK || p.B * p.Tq == 0) return rc;
    rc = workspace_missing(p, fkda_latent_decode_workspace_bytes(&p));
    if (rc != FKDA_OK) return rc;
    return enqueue([&](int* n) { return fkda::launch_latent_decode(p, static_cast<cudaStream_t>(stream), n); });
}

int fkda_operator_test_starve(int32_t wait_ms) {
    if (!in_range(wait_ms, 1, 1000)) return FKDA_ERR_BAD_SHAPE;
    g_starve_ms = wait_ms;
    return FKDA_OK;
}

int fkda_operator_status(void* stream_v) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return FKDA_ERR_LAUNCH;
    std::array<uint32_t, 3> times{};
    if (fkda::linear_gave_up(stream, &times[0]) != FKDA_OK || fkda::prompt_gave_up(stream, &times[1]) != FKDA_OK ||
        fkda::decode_gave_up(stream, &times[2]) != FKDA_OK)
        return FKDA_ERR_LAUNCH;
    const bool same = times == g_seen[dev];
    g_seen[dev] = times;
    return same ? FKDA_OK : FKDA_ERR_DEVICE_STATUS;
}

}  // extern "C"
