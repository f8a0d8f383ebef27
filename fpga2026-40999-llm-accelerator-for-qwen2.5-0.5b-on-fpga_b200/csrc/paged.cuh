// The paged KV cache as the kernels see it (one layer), and what the host
// side of its entry points shares. Every index that comes from device memory
// is checked here before it is used, so no table, length or sequence list can
// take an access out of the pool.
#pragma once
#include "common.cuh"
#include "qwen_b200.h"

namespace qb {

constexpr uint32_t PG_NO_PAGE = 0xffffffffu;

struct PagedView {
    const uint8_t *k, *v;   // the layer's first row
    const float *ks, *vs;   // its scales (KV8)
    const uint32_t *table;  // [seqs][max_pages]
    const uint32_t *lengths;
    uint64_t page_rows;     // rows from one page to the next
    uint32_t pages, seqs, max_pages, hkv;
    int tshift;             // log2(page_tokens)
};

// Tokens of a sequence, cut to what its table row can name; 0 for no sequence.
__device__ __forceinline__ int paged_length(const PagedView &c, uint32_t seq) {
    if (seq >= c.seqs) return 0;
    return (int)min(c.lengths[seq], c.max_pages << c.tshift);
}
// First pool row of (page, head); the caller has checked page < c.pages.
__device__ __forceinline__ uint64_t paged_row(const PagedView &c, uint32_t page, uint32_t head) {
    return (uint64_t)page * c.page_rows + ((uint64_t)head << c.tshift);
}

// Keys visible to the token at `pos` (its own included) under a window and
// first tokens: [0, first) and [low, pos].
struct KeySpan {
    int first, low;
};
__host__ __device__ __forceinline__ KeySpan key_span(int pos, uint32_t window, uint32_t sinks) {
    const int low = window && (uint32_t)pos >= window ? pos + 1 - (int)window : 0;
    return {(int)(sinks < (uint32_t)low ? sinks : (uint32_t)low), low};
}

// n / d and n % d, by 32-bit division where both fit; a 64-bit one is several
// hundred instructions, kept out of line (the kernels' loops share the
// instruction cache with everything that is inlined around them).
static __device__ __noinline__ unsigned long long div64_wide(unsigned long long n, unsigned long long d) { return n / d; }
__device__ __forceinline__ void div64(unsigned long long n, unsigned long long d, unsigned long long &q,
                                      unsigned long long &r) {
    if (((n | d) >> 32) == 0) {
        q = (uint32_t)n / (uint32_t)d;
        r = (uint32_t)n - (uint32_t)q * (uint32_t)d;
    } else {
        q = div64_wide(n, d);
        r = n - q * d;
    }
}

// An equal split of `total` units over g CTAs, each with at least `least` of
// them: CTA c takes units [start(c), start(c + 1)).
struct UnitSplit {
    unsigned long long q, r;
    uint32_t g;
    UnitSplit() = default;
    __device__ __forceinline__ UnitSplit(unsigned long long total, uint32_t max_ctas, uint32_t least) {
        unsigned long long want, rest;
        div64(total + least - 1, least, want, rest);
        g = (uint32_t)min((unsigned long long)max_ctas, max(want, 1ull));
        div64(total, g, q, r);
    }
    __device__ __forceinline__ unsigned long long start(uint32_t c) const {
        return c * q + min((unsigned long long)c, r);
    }
    __device__ __forceinline__ uint32_t cta_of(unsigned long long u) const {
        const unsigned long long edge = r * (q + 1);
        unsigned long long c, rest;
        div64(u < edge ? u : u - edge, u < edge ? q + 1 : q, c, rest);
        return (uint32_t)(u < edge ? c : r + c);
    }
};

// Host side: 0, or the status of a descriptor that cannot be used.
int paged_check(const qwen_b200_paged_kv *kv);
PagedView paged_view(const qwen_b200_paged_kv &kv, uint32_t layer);
inline uint32_t paged_row_bytes(const qwen_b200_paged_kv &kv) {
    return kv.format == QWEN_B200_KV8 ? kv.head_dim : 2 * kv.head_dim;
}
// SMs of the current device, looked up once per device.
int paged_sms();

struct PagedAttnArgs {
    PagedView c;
    const uint16_t *q;
    uint64_t q_stride, ctx_stride;
    uint16_t *ctx;
    const uint32_t *seqs, *starts;  // starts: prefill only
    uint32_t qh, rows, n;           // rows of q; n sequences (prefill)
    uint32_t window, sinks;
    float scale;
    uint32_t format, dim;
};
size_t paged_decode_ws(uint32_t kv_heads, uint32_t q_heads, uint32_t dim, uint32_t rows);
int launch_paged_decode(const PagedAttnArgs &a, void *ws, cudaStream_t st);
size_t paged_prefill_ws(uint32_t kv_heads, uint32_t q_heads, uint32_t dim, uint32_t n, uint32_t rows);
// Whether the blocks of a KV head that such a call can have are counted in 32 bits.
bool paged_prefill_fits(const PagedAttnArgs &a);
int launch_paged_prefill(const PagedAttnArgs &a, void *ws, cudaStream_t st);
int launch_paged_append(const qwen_b200_paged_kv &kv, uint32_t layer, const uint16_t *k, const uint16_t *v,
                        uint64_t row_stride, uint32_t rows, const uint32_t *seqs, const uint32_t *positions,
                        cudaStream_t st);
size_t pages_ws(uint32_t pages);
int launch_pages_reserve(const qwen_b200_paged_kv &kv, const uint32_t *seqs, const uint32_t *tokens, uint32_t n,
                         uint32_t *status, void *ws, cudaStream_t st);
int launch_pages_fork(const qwen_b200_paged_kv &kv, const uint32_t *parents, const uint32_t *children,
                      const uint32_t *prefix, uint32_t n, uint32_t *status, void *ws, cudaStream_t st);
int launch_pages_free(const qwen_b200_paged_kv &kv, const uint32_t *seqs, uint32_t n, uint32_t *status,
                      cudaStream_t st);
int launch_pages_compact(const qwen_b200_paged_kv &kv, uint32_t *status, void *ws, cudaStream_t st);
int launch_pages_copy(const qwen_b200_paged_kv &kv, const uint32_t *src, const uint32_t *dst, uint32_t n,
                      cudaStream_t st);

}  // namespace qb
