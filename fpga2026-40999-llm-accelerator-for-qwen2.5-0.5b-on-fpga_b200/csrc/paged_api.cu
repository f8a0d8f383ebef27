// C entry points of the paged KV cache: argument checks, then one launcher.
#include <initializer_list>

#include "paged.cuh"

using namespace qb;

namespace qb {

int paged_check(const qwen_b200_paged_kv *kv) {
    if (!kv || !kv->k || !kv->v || !kv->table || !kv->lengths) return QWEN_B200_EINVAL;
    if (kv->format != QWEN_B200_KV8 && kv->format != QWEN_B200_KV_BF16) return QWEN_B200_EINVAL;
    if (kv->head_dim != 64 && kv->head_dim != 128) return QWEN_B200_EINVAL;
    const uint32_t t = kv->page_tokens;
    if (t < 16 || t > 256 || (t & (t - 1))) return QWEN_B200_EINVAL;
    if (!kv->layers || !kv->pages || !kv->kv_heads || !kv->seqs || !kv->max_pages) return QWEN_B200_EINVAL;
    if (kv->pages >= 1u << 31 || kv->seqs > 65536 || kv->layers > 65536 || kv->kv_heads > 16384)
        return QWEN_B200_EINVAL;
    if ((uint64_t)kv->max_pages * t > 1ull << 30) return QWEN_B200_EINVAL;
    uintptr_t align = (uintptr_t)kv->k | (uintptr_t)kv->v;
    if (kv->format == QWEN_B200_KV8) {
        if (!kv->kscales || !kv->vscales) return QWEN_B200_EINVAL;
        align |= (uintptr_t)kv->kscales | (uintptr_t)kv->vscales;
    }
    if ((align & 15) || (((uintptr_t)kv->table | (uintptr_t)kv->lengths | (uintptr_t)kv->refs) & 3))
        return QWEN_B200_EINVAL;
    // pages of one layer and layers of one page apart: one of the two strides
    // spans the other's whole range
    const uint64_t block = (uint64_t)kv->kv_heads * t;
    if ((kv->layer_stride | kv->page_stride) & 15) return QWEN_B200_EINVAL;
    if (kv->layer_stride > 1ull << 40 || kv->page_stride > 1ull << 31) return QWEN_B200_EINVAL;  // (a tensor map's stride is below 2^40 bytes)
    if (kv->pages > 1 && kv->page_stride < block) return QWEN_B200_EINVAL;
    if (kv->layers > 1 && kv->layer_stride < block) return QWEN_B200_EINVAL;
    const unsigned __int128 pspan = (unsigned __int128)(kv->pages - 1) * kv->page_stride + block;
    const unsigned __int128 lspan = (unsigned __int128)(kv->layers - 1) * kv->layer_stride + block;
    if (kv->layers > 1 && kv->pages > 1 && kv->layer_stride < pspan && kv->page_stride < lspan)
        return QWEN_B200_EINVAL;
    if (pspan + lspan > ((unsigned __int128)1 << 54)) return QWEN_B200_EINVAL;  // byte offsets in 64 bits
    return QWEN_B200_OK;
}

// Every device pointer of a call (NULL: not given) has to be the current device's.
static int check_pointers(std::initializer_list<const void *> pointers) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return QWEN_B200_EDEVICE;
    }
    for (const void *p : pointers) {
        cudaPointerAttributes a;
        if (!p) continue;
        if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
            cudaGetLastError();
            return QWEN_B200_EDEVICE;
        }
        if (a.type != cudaMemoryTypeManaged && (a.type != cudaMemoryTypeDevice || a.device != dev)) return QWEN_B200_EINVAL;
    }
    return QWEN_B200_OK;
}
static int paged_check_device(const qwen_b200_paged_kv &kv, std::initializer_list<const void *> more) {
    const bool scales = kv.format == QWEN_B200_KV8;
    if (int rc = check_pointers({kv.k, kv.v, scales ? kv.kscales : nullptr, scales ? kv.vscales : nullptr, kv.table,
                                 kv.lengths}))
        return rc;
    return check_pointers(more);
}

// Lists of 32-bit indexes and counts in device memory.
static bool words_aligned(std::initializer_list<const uint32_t *> lists) {
    uintptr_t bits = 0;
    for (const uint32_t *p : lists) bits |= (uintptr_t)p;
    return (bits & 3) == 0;
}

PagedView paged_view(const qwen_b200_paged_kv &kv, uint32_t layer) {
    const uint64_t row = (uint64_t)layer * kv.layer_stride, bytes = paged_row_bytes(kv);
    PagedView c;
    c.k = (const uint8_t *)kv.k + row * bytes;
    c.v = (const uint8_t *)kv.v + row * bytes;
    c.ks = kv.format == QWEN_B200_KV8 ? kv.kscales + row : nullptr;
    c.vs = kv.format == QWEN_B200_KV8 ? kv.vscales + row : nullptr;
    c.table = kv.table;
    c.lengths = kv.lengths;
    c.page_rows = kv.page_stride;
    c.pages = kv.pages;
    c.seqs = kv.seqs;
    c.max_pages = kv.max_pages;
    c.hkv = kv.kv_heads;
    c.tshift = __builtin_ctz(kv.page_tokens);
    return c;
}

int paged_sms() {
    static int sms[64];  // written with the same value by every thread that finds 0
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = __atomic_load_n(&sms[dev], __ATOMIC_RELAXED);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        __atomic_store_n(&sms[dev], n, __ATOMIC_RELAXED);
    }
    return n;
}

static int attn_check(const qwen_b200_paged_kv *kv, uint32_t layer, const uint16_t *q, uint64_t q_stride,
                      uint32_t q_heads, uint32_t rows, float scale, uint16_t *ctx, uint64_t ctx_stride, void *ws) {
    if (int rc = paged_check(kv)) return rc;
    if (!q || !ctx || !ws || !rows || layer >= kv->layers) return QWEN_B200_EINVAL;
    if (!q_heads || q_heads % kv->kv_heads || q_heads > 65536) return QWEN_B200_EINVAL;
    const uint64_t width = (uint64_t)q_heads * kv->head_dim;
    if (q_stride < width || ctx_stride < width || ((q_stride | ctx_stride) & 7)) return QWEN_B200_EINVAL;
    if (q_stride > 1ull << 40 || ctx_stride > 1ull << 40) return QWEN_B200_EINVAL;
    if (((uintptr_t)q | (uintptr_t)ctx | (uintptr_t)ws) & 15) return QWEN_B200_EINVAL;
    if (!(fabsf(scale) <= 2.0e38f)) return QWEN_B200_EINVAL;  // log2(e) scale is finite
    return QWEN_B200_OK;
}

static PagedAttnArgs attn_args(const qwen_b200_paged_kv &kv, uint32_t layer, const uint16_t *q, uint64_t q_stride,
                               uint32_t q_heads, const uint32_t *seqs, uint32_t window, uint32_t sinks, float scale,
                               uint16_t *ctx, uint64_t ctx_stride) {
    PagedAttnArgs a;
    a.c = paged_view(kv, layer);
    a.q = q;
    a.q_stride = q_stride;
    a.ctx_stride = ctx_stride;
    a.ctx = ctx;
    a.seqs = seqs;
    a.starts = nullptr;
    a.qh = q_heads;
    a.window = window;
    a.sinks = sinks;
    a.scale = scale;
    a.format = kv.format;
    a.dim = kv.head_dim;
    return a;
}

// Checks shared by the page management calls.
static int pages_check(const qwen_b200_paged_kv *kv, std::initializer_list<const uint32_t *> lists, uint32_t n,
                       uint32_t *status, void *ws, size_t ws_bytes) {
    if (int rc = paged_check(kv)) return rc;
    if (!words_aligned(lists) || n >= 1u << 31) return QWEN_B200_EINVAL;
    if (!kv->refs || !status || ((uintptr_t)status & 3) || !ws || ((uintptr_t)ws & 15)) return QWEN_B200_EINVAL;
    if (ws_bytes < pages_ws(kv->pages)) return QWEN_B200_EINVAL;
    for (const uint32_t *p : lists)
        if (int rc = check_pointers({p})) return rc;
    return paged_check_device(*kv, {kv->refs, status, ws});
}

}  // namespace qb

extern "C" {

int qwen_b200_op_paged_append(const qwen_b200_paged_kv *kv, uint32_t layer, const uint16_t *k, const uint16_t *v,
                              uint64_t row_stride, uint32_t rows, const uint32_t *seqs, const uint32_t *positions,
                              void *stream) {
    if (int rc = paged_check(kv)) return rc;
    if (!k || !v || !rows || !seqs || !positions || layer >= kv->layers || rows >= 1u << 31) return QWEN_B200_EINVAL;
    if (row_stride < (uint64_t)kv->kv_heads * kv->head_dim || (row_stride & 7) || row_stride > 1ull << 40)
        return QWEN_B200_EINVAL;
    if ((((uintptr_t)k | (uintptr_t)v) & 15) || !words_aligned({seqs, positions})) return QWEN_B200_EINVAL;
    if (int rc = paged_check_device(*kv, {k, v, seqs, positions})) return rc;
    return launch_paged_append(*kv, layer, k, v, row_stride, rows, seqs, positions, (cudaStream_t)stream);
}

size_t qwen_b200_paged_decode_workspace(const qwen_b200_paged_kv *kv, uint32_t q_heads, uint32_t rows) {
    if (paged_check(kv) || !q_heads || q_heads % kv->kv_heads) return 0;
    return paged_decode_ws(kv->kv_heads, q_heads, kv->head_dim, rows);
}

int qwen_b200_op_paged_decode(const qwen_b200_paged_kv *kv, uint32_t layer, const uint16_t *q, uint64_t q_stride,
                              uint32_t q_heads, uint32_t rows, const uint32_t *seqs, uint32_t window, uint32_t sinks,
                              float scale, uint16_t *ctx, uint64_t ctx_stride, void *workspace,
                              size_t workspace_bytes, void *stream) {
    if (int rc = attn_check(kv, layer, q, q_stride, q_heads, rows, scale, ctx, ctx_stride, workspace)) return rc;
    if (rows > 65536 || !words_aligned({seqs})) return QWEN_B200_EINVAL;
    if (int rc = paged_check_device(*kv, {q, seqs, ctx, workspace})) return rc;
    if (workspace_bytes < paged_decode_ws(kv->kv_heads, q_heads, kv->head_dim, rows)) return QWEN_B200_EINVAL;
    PagedAttnArgs a = attn_args(*kv, layer, q, q_stride, q_heads, seqs, window, sinks, scale, ctx, ctx_stride);
    a.rows = rows;
    a.n = rows;
    return launch_paged_decode(a, workspace, (cudaStream_t)stream);
}

size_t qwen_b200_paged_prefill_workspace(const qwen_b200_paged_kv *kv, uint32_t q_heads, uint32_t n, uint32_t rows) {
    if (paged_check(kv) || !q_heads || q_heads % kv->kv_heads) return 0;
    return paged_prefill_ws(kv->kv_heads, q_heads, kv->head_dim, n, rows);
}

int qwen_b200_op_paged_prefill(const qwen_b200_paged_kv *kv, uint32_t layer, const uint16_t *q, uint64_t q_stride,
                               uint32_t q_heads, uint32_t n, const uint32_t *seqs, const uint32_t *starts,
                               uint32_t rows, uint32_t window, uint32_t sinks, float scale, uint16_t *ctx,
                               uint64_t ctx_stride, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = attn_check(kv, layer, q, q_stride, q_heads, rows, scale, ctx, ctx_stride, workspace)) return rc;
    if (!starts || !n || n > 65536 || rows > 1u << 24 || !words_aligned({seqs, starts})) return QWEN_B200_EINVAL;
    if ((uint64_t)rows * (q_heads / kv->kv_heads) >= 1ull << 31) return QWEN_B200_EINVAL;
    PagedAttnArgs a = attn_args(*kv, layer, q, q_stride, q_heads, seqs, window, sinks, scale, ctx, ctx_stride);
    a.rows = rows;
    a.n = n;
    a.starts = starts;
    if (!paged_prefill_fits(a)) return QWEN_B200_EINVAL;
    if (int rc = paged_check_device(*kv, {q, seqs, starts, ctx, workspace})) return rc;
    if (workspace_bytes < paged_prefill_ws(kv->kv_heads, q_heads, kv->head_dim, n, rows)) return QWEN_B200_EINVAL;
    return launch_paged_prefill(a, workspace, (cudaStream_t)stream);
}

size_t qwen_b200_pages_workspace(const qwen_b200_paged_kv *kv) {
    return paged_check(kv) ? 0 : pages_ws(kv->pages);
}

int qwen_b200_op_pages_reserve(const qwen_b200_paged_kv *kv, const uint32_t *seqs, const uint32_t *tokens, uint32_t n,
                               uint32_t *status, void *workspace, size_t workspace_bytes, void *stream) {
    if (!seqs || !tokens || !n) return QWEN_B200_EINVAL;
    if (int rc = pages_check(kv, {seqs, tokens}, n, status, workspace, workspace_bytes)) return rc;
    return launch_pages_reserve(*kv, seqs, tokens, n, status, workspace, (cudaStream_t)stream);
}

int qwen_b200_op_pages_fork(const qwen_b200_paged_kv *kv, const uint32_t *parents, const uint32_t *children,
                            const uint32_t *prefix, uint32_t n, uint32_t *status, void *workspace,
                            size_t workspace_bytes, void *stream) {
    if (!parents || !children || !prefix || !n) return QWEN_B200_EINVAL;
    if (int rc = pages_check(kv, {parents, children, prefix}, n, status, workspace, workspace_bytes)) return rc;
    return launch_pages_fork(*kv, parents, children, prefix, n, status, workspace, (cudaStream_t)stream);
}

int qwen_b200_op_pages_free(const qwen_b200_paged_kv *kv, const uint32_t *seqs, uint32_t n, uint32_t *status,
                            void *workspace, size_t workspace_bytes, void *stream) {
    if (!seqs || !n) return QWEN_B200_EINVAL;
    if (int rc = pages_check(kv, {seqs}, n, status, workspace, workspace_bytes)) return rc;
    return launch_pages_free(*kv, seqs, n, status, (cudaStream_t)stream);
}

int qwen_b200_op_pages_compact(const qwen_b200_paged_kv *kv, uint32_t *status, void *workspace,
                               size_t workspace_bytes, void *stream) {
    if (int rc = pages_check(kv, {}, 0, status, workspace, workspace_bytes)) return rc;
    return launch_pages_compact(*kv, status, workspace, (cudaStream_t)stream);
}

int qwen_b200_op_pages_copy(const qwen_b200_paged_kv *kv, const uint32_t *src, const uint32_t *dst, uint32_t n,
                            void *stream) {
    if (int rc = paged_check(kv)) return rc;
    if (!src || !dst || !n || n >= 1u << 31 || !words_aligned({src, dst})) return QWEN_B200_EINVAL;
    if (int rc = paged_check_device(*kv, {src, dst})) return rc;
    return launch_pages_copy(*kv, src, dst, n, (cudaStream_t)stream);
}

}  // extern "C"
