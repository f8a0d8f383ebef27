// Attention of one token per sequence where groups of sequences share their
// first tokens: the shared keys by tiles of query rows (paged_prefill.cu), then
// each row's own keys joined with those (paged_decode.cu). A group that is not
// worth the tiles has each row read its whole context, shared pages from L2.
//
// Mathematics, per (row, query head), P the group's prefix, over keys j < len:
//   x_j = log2(e) scale q.k_j,  p_j = 2^(x_j - m),  ctx = sum p_j v_j / sum p_j
// where key j < P is the first sequence's and key j >= P the row's own. Sums over
// disjoint keys join exactly: (m, l, o) and (m', l', o') give l 2^(m - M) + l' 2^(m' - M)
// and the like for o, M = max(m, m').
#include "kernels.h"
#include "paged.cuh"

namespace qb {

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t paged_shared_ws(uint32_t q_heads, uint32_t dim, uint32_t n, uint32_t rows) {
    const size_t heads = (size_t)rows * q_heads;
    return 256 + up256(((size_t)n + 1) * 8) + paged_shared_pieces_bytes(dim) + up256(heads * 8) + heads * dim * 4;
}

// The tile kernel's blocks and the row kernel's keys are counted in 32 bits.
bool paged_shared_fits(const PagedAttnArgs &a) {
    const uint64_t group = a.qh / a.c.hkv, items = a.c.hkv * ((group + 7) / 8);
    if (a.rows * group >= 1ull << 31 || a.rows * items * 8 >= 1ull << 31) return false;
    return paged_prefill_fits(a) && a.rows * items * ((((uint64_t)a.c.max_pages << a.c.tshift) >> 4) + 3) < 1ull << 32;
}

int launch_paged_shared(const PagedAttnArgs &args, void *ws, cudaStream_t st) {
    const int sms = paged_sms();
    if (sms <= 0) return -3;
    PagedAttnArgs a = args;
    a.long_keys = shared_few_warps((uint64_t)a.rows * a.c.hkv * ((a.qh / a.c.hkv + 7) / 8), sms) ? SHARED_LONG : 0xffffffffu;
    const size_t heads = (size_t)a.rows * a.qh;
    char *p = (char *)ws + 256;
    SharedParts parts = {};
    parts.base = reinterpret_cast<unsigned long long *>(p);
    p += up256(((size_t)a.n + 1) * 8);
    parts.pieces = reinterpret_cast<float *>(p);
    p += paged_shared_pieces_bytes(a.dim);
    parts.ml = reinterpret_cast<float *>(p);
    parts.o = reinterpret_cast<float *>(p + up256(heads * 8));
    a.tile_work = (SHARED_WORK / a.dim + a.c.hkv - 1) / a.c.hkv;
    // The host knows no prefix, but no group is worth the tile kernel where all rows with the widest table are not.
    const bool tiles = shared_worth(a, a.rows, (uint64_t)a.c.max_pages << a.c.tshift);
    PdlChain chain;
    if (tiles)
        if (int rc = launch_shared_tiles(a, parts, (unsigned *)ws, st)) return rc;
    return launch_shared_rows(a, parts, tiles, st);
}

}  // namespace qb
