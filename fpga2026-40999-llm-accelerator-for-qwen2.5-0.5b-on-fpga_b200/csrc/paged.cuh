// The paged KV cache as the kernels see it (one layer), and what the host
// side of its entry points shares. Every index that comes from device memory
// is checked here before it is used, so no table, length or sequence list can
// take an access out of the pool.
#pragma once
#include <initializer_list>

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
// Whether every pointer (NULL: not given) is the current device's memory, and whether lists of 32-bit words are aligned.
int check_pointers(std::initializer_list<const void *> pointers);
bool words_aligned(std::initializer_list<const void *> lists);

struct PagedAttnArgs {
    PagedView c;
    const uint16_t *q;
    uint64_t q_stride, ctx_stride;
    uint16_t *ctx;
    const uint32_t *seqs, *starts;  // starts: prefill and shared decode
    uint32_t qh, rows, n;           // rows of q; n sequences (prefill) or groups (shared decode)
    uint32_t window, sinks;
    float scale;
    uint32_t format, dim;
    const uint32_t *prefix = nullptr;  // shared decode: tokens that a group's sequences share,
    uint32_t long_keys = 0;            // how many of them go to the tiles whatever the work,
    uint64_t tile_work = 0;            // and from how many rows * tokens on all do
};
// A group of sequences that share their first tokens: its rows of q, and how many tokens of its first row's sequence
// the tile kernel takes for all of them (0: none, each row takes its whole context).
struct SharedGroup {
    uint32_t row0, rows, seq;
    int keys;
};
// Whether a group is worth the tile kernel: rows * keys * KV heads * dims from 3 * 2^24 on. Its launch and the join of its
// pieces take some 12 us whatever the size, and the row kernel finds shared pages in L2. Row by row and with tiles, us of a
// captured call with L2 flushed, 64 own keys a row: 14 heads on 2 of 64 dims KV8, 64 rows on 2048 keys (2^24) 18 and 31,
// 4096 (2^25) 27 and 33, 6144 (3 * 2^24) 33 and 35, 8192 (2^26) 41 and 35, 256 rows on 4096 (2^27) 70 and 43; 32 heads on 8
// of 128 dims bf16, 32 rows on 512 keys (2^24) 21 and 29, 1024 (2^25) 27 and 31, 1536 (3 * 2^24) 33 and 33, 2048 (2^26) 39
// and 33, 64 rows on 4096 (2^28) 104 and 45, 2 rows on 32768 (2^26) 68 and 64; of 64 dims bf16 64 rows on 1024 (2^25) 25 and
// 27, of 128 KV8 32 rows on 1024 (2^25) 25 and 29.
constexpr uint64_t SHARED_WORK = 3ull << 24;
// From three items (row, KV head, block of 8 heads) an SM on the row kernel takes fewer warps for each, which a long context
// keeps busy after all others are done: there every prefix of SHARED_LONG keys and two or more rows goes to the tiles. That
// is for groups that are long beside the others. Without and with it, us as above, 14 heads on 2 of 64 dims KV8: 228 rows on
// 512 keys and 2 on 2048 25 and 25, on 4096 37 and 31, on 32000 190 and 43; 32 heads on 8 of 128 dims bf16, 128 rows in 4
// groups on some 6000 keys, two of them of 4 rows 227 and 80, one of 12 rows 150 and 78. Where all groups are long it gains
// if they have rows enough for their tiles: 16 groups of 16 rows on 2048 KV8 41 and 37, 32 of 4 rows of 128 dims bf16 107
// and 94, 32 of 4 rows of 32 heads on 1 of 64 dims 41 and 35, of 32 heads on 2 41 and 43, 64 rows of 64 heads on 1 on 2048
// 41 and 33, on 4096 70 and 41, and loses if not: 32 groups of 8 rows on 2048 41 and 47, 64 of 4 41 and 68, on 4096 72 and
// 110, 32 of 2 rows of 128 dims bf16 72 and 92, KV8 on 4096 115 and 195. A group cannot tell the two apart by itself. From
// 1024 keys on 32 groups of 4 rows of 128 dims 66 and 68, 16 of 4 41 and 49.
constexpr uint32_t SHARED_LONG = 2048;
inline bool shared_few_warps(uint64_t items, int sms) { return items >= 3 * (uint64_t)sms; }
__host__ __device__ __forceinline__ bool shared_worth(const PagedAttnArgs &a, uint32_t rows, uint64_t keys) {
    return rows >= 2 && (keys >= a.long_keys || rows * keys >= a.tile_work);
}
__device__ __forceinline__ SharedGroup shared_group(const PagedAttnArgs &a, uint32_t g) {
    SharedGroup s;
    s.row0 = min(a.starts[g], a.rows);
    s.rows = min(max(a.starts[g + 1], s.row0), a.rows) - s.row0;
    s.seq = s.rows == 0 ? QWEN_B200_NO_SEQ : a.seqs ? a.seqs[s.row0] : s.row0;
    s.keys = min((int)min(a.prefix[g], 0x7fffffffu), paged_length(a.c, s.seq));
    if (!shared_worth(a, s.rows, (uint32_t)s.keys)) s.keys = 0;
    return s;
}
// The group that a row belongs to; false for none. starts is not decreasing.
__device__ __forceinline__ bool shared_find(const PagedAttnArgs &a, uint32_t row, uint32_t &g) {
    uint32_t lo = 0, hi = a.n;  // the last start at or before the row
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (a.starts[mid] <= row) lo = mid; else hi = mid - 1;
    }
    g = lo;
    return lo < a.n && a.starts[lo] <= row && row < a.starts[lo + 1];
}
// What the tile kernel leaves for the row kernel. Units (tile, KV head, block of 128 keys) are numbered group by group,
// KV head by KV head, and split evenly over `ctas`; a tile's list of blocks is in pieces of the CTAs that have some of it
// (two a CTA at most: [m tile][l tile][o dim / 4][tile][4]), or whole, then by flattened row of a KV head:
// [hkv][rows * group] (m, l), [hkv][dim / 4][rows * group][4] o. (A thread of the tile kernel has a row: with four dims of
// all rows side by side its stores are whole lines; [row][dim] took 3 us more.)
constexpr uint32_t SHARED_BLOCK = 128, SHARED_LEAST = 1, SHARED_MAX_CTAS = 192;  // keys of a block, blocks of a CTA at least, CTAs
struct SharedParts {
    unsigned long long *base;  // [n + 1] units of one KV head in the groups before
    float *pieces, *ml, *o;
    uint32_t tile, ctas;
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
size_t paged_shared_ws(uint32_t q_heads, uint32_t dim, uint32_t n, uint32_t rows);
bool paged_shared_fits(const PagedAttnArgs &a);
int launch_paged_shared(const PagedAttnArgs &a, void *ws, cudaStream_t st);
// Its two halves: the shared tokens by tiles of query rows, then each row's own tokens joined with those.
size_t paged_shared_pieces_bytes(uint32_t dim);
int launch_shared_tiles(const PagedAttnArgs &a, SharedParts &parts, unsigned *err, cudaStream_t st);
int launch_shared_rows(const PagedAttnArgs &a, const SharedParts &parts, bool tiles, cudaStream_t st);

struct RotaryView {
    const float *table;
    uint32_t positions, rotated, pairs;
};
struct AppendRotary {
    const uint16_t *q, *k, *v;
    uint16_t *q_out;
    uint64_t q_stride, q_out_stride, kv_stride;
    uint32_t q_heads, rows;
    const uint32_t *seqs, *positions;
};
int launch_rotary(const RotaryView &t, const uint16_t *x, uint64_t x_stride, uint32_t heads, uint32_t dim, uint32_t rows,
                  const uint32_t *positions, uint16_t *out, uint64_t out_stride, cudaStream_t st);
int launch_paged_append_rotary(const qwen_b200_paged_kv &kv, uint32_t layer, const RotaryView &t, const AppendRotary &a,
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
