// Writing into and managing the pages of the paged KV cache.
//
// Append: one pass over the new rows. Page management: the tables, lengths
// and reference counts are planned by one CTA (a few KB to a few hundred KB of
// metadata, bound by latency; one CTA needs no grid-wide barrier between
// checking a call and changing anything), which leaves a list of page copies
// for a grid-wide copy kernel (bound by HBM) launched right behind it.
#include "kernels.h"
#include "paged.cuh"

namespace qb {

// ---------------------------------------------------------------- append
// K and V rows of new tokens -> pages. DIM / 8 threads hold one (row, head) of
// K or V (blockIdx.y): a 16-byte load of 8 bf16 values each, the row's largest
// magnitude over the threads by shuffles, one 16-byte (bf16) or 8-byte (codes)
// store. A thread takes ROWS rows at a time, so that as many chains of
// sequence -> length -> page -> row are in flight. Bound by HBM for prompts
// (11k rows x 8 heads of 128 bf16: 14.2 us, 6.4 TB/s) and by that chain for single tokens.
// KV8: scale = amax / 127, code = clamp(rne(x / scale), +-127), every step one
// IEEE fp32 operation, the same bits as kv8_append_kernel.
constexpr int PA_THREADS = 256, PA_ROWS = 4;
template <bool KV8, int DIM>
__global__ void __launch_bounds__(PA_THREADS)
    paged_append_kernel(PagedView c, const uint16_t *__restrict__ k, const uint16_t *__restrict__ v,
                        uint64_t row_stride, uint32_t rows, const uint32_t *__restrict__ seqs,
                        const uint32_t *__restrict__ positions) {
    constexpr int TPR = DIM / 8, RPB = PA_THREADS / TPR;  // threads of a row, rows of a block at a time
    const int part = threadIdx.x % TPR;
    const bool is_v = blockIdx.y >= c.hkv;
    const uint32_t head = is_v ? blockIdx.y - c.hkv : blockIdx.y;
    const uint16_t *src = (is_v ? v : k) + head * DIM + 8 * part;
    uint32_t seq[PA_ROWS], pos[PA_ROWS], page[PA_ROWS];
    uint4 w[PA_ROWS];
    const uint64_t first = (uint64_t)blockIdx.x * (RPB * PA_ROWS) + threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < PA_ROWS; ++i) {
        const uint64_t r = first + i * RPB;
        seq[i] = pos[i] = 0xffffffffu;
        w[i] = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            seq[i] = seqs[r];
            pos[i] = positions[r];
            w[i] = *reinterpret_cast<const uint4 *>(src + r * row_stride);
        }
    }
#pragma unroll
    for (int i = 0; i < PA_ROWS; ++i) {
        page[i] = PG_NO_PAGE;
        if (pos[i] < (uint32_t)paged_length(c, seq[i])) page[i] = c.table[(uint64_t)seq[i] * c.max_pages + (pos[i] >> c.tshift)];
    }
    uint8_t *pool = const_cast<uint8_t *>(is_v ? c.v : c.k);
#pragma unroll
    for (int i = 0; i < PA_ROWS; ++i) {
        const bool live = page[i] < c.pages;
        const uint64_t dst = live ? paged_row(c, page[i], head) + (pos[i] & ((1u << c.tshift) - 1)) : 0;
        if constexpr (!KV8) {
            if (live) *reinterpret_cast<uint4 *>(pool + (dst * DIM + 8 * part) * 2) = w[i];
        } else {
            const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            float x[8], amax = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = bflo(ww[j]);
                x[2 * j + 1] = bfhi(ww[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
#pragma unroll
            for (int o = TPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if (!live) continue;  // (a row's threads agree, and the shuffles stay within it)
            const float s = __fdiv_rn(amax, 127.0f);
            uint32_t b[2] = {0u, 0u};
            if (s > 0.f) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int code = (int)fminf(fmaxf(rintf(__fdiv_rn(x[j], s)), -127.f), 127.f);
                    b[j >> 2] |= ((uint32_t)code & 0xffu) << (8 * (j & 3));
                }
            }
            *reinterpret_cast<uint2 *>(pool + dst * DIM + 8 * part) = make_uint2(b[0], b[1]);
            if (part == 0) const_cast<float *>(is_v ? c.vs : c.ks)[dst] = s;
        }
    }
}

int launch_paged_append(const qwen_b200_paged_kv &kv, uint32_t layer, const uint16_t *k, const uint16_t *v,
                        uint64_t row_stride, uint32_t rows, const uint32_t *seqs, const uint32_t *positions,
                        cudaStream_t st) {
    const PagedView c = paged_view(kv, layer);
    const uint32_t per = PA_THREADS / (kv.head_dim / 8) * PA_ROWS;
    const dim3 grid((rows + per - 1) / per, 2 * kv.kv_heads);
    auto *kernel = kv.format == QWEN_B200_KV8
                       ? (kv.head_dim == 64 ? paged_append_kernel<true, 64> : paged_append_kernel<true, 128>)
                       : (kv.head_dim == 64 ? paged_append_kernel<false, 64> : paged_append_kernel<false, 128>);
    kernel<<<grid, PA_THREADS, 0, st>>>(c, k, v, row_stride, rows, seqs, positions);
    return QB_LAUNCH_CHECK();
}

// ---------------------------------------------------------------- plans
constexpr int PP_THREADS = 1024;

struct PagesState {
    uint32_t *table, *lengths, *refs, *status;
    uint32_t pages, seqs, max_pages;
    int tshift;
    uint32_t *count;   // copies in `list`
    uint32_t *spare;   // [pages] free page ids, lowest first
    uint32_t *remap;   // [pages] new id of a page that moves
    uint4 *list;       // [pages] (src, dst, tokens, -)
};

size_t pages_ws(uint32_t pages) { return 256 + 24 * (((size_t)pages + 3) & ~(size_t)3); }

static PagesState pages_state(const qwen_b200_paged_kv &kv, uint32_t *status, void *ws) {
    PagesState s;
    s.table = kv.table;
    s.lengths = kv.lengths;
    s.refs = kv.refs;
    s.status = status;
    s.pages = kv.pages;
    s.seqs = kv.seqs;
    s.max_pages = kv.max_pages;
    s.tshift = __builtin_ctz(kv.page_tokens);
    const size_t p4 = ((size_t)kv.pages + 3) & ~(size_t)3;
    s.count = (uint32_t *)ws;
    s.spare = (uint32_t *)ws + 64;
    s.remap = s.spare + p4;
    s.list = reinterpret_cast<uint4 *>(s.remap + p4);
    return s;
}

// Exclusive prefix sum over the CTA; every thread also gets the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *warp_sums, uint32_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the sums of an earlier call have been read
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    uint32_t s = warp_sums[lane], t = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += y;
    }
    total = __shfl_sync(0xffffffffu, t, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, t - s, warp);
    return before + x - v;
}

struct PlanShared {
    uint32_t warp_sums[32];
    uint32_t seen[65536 / 32];  // one bit per sequence: named in this call
    unsigned long long need;    // pages that the call wants
    uint32_t bad;
};

__device__ __forceinline__ void plan_begin(const PagesState &s, PlanShared &sh) {
    for (uint32_t i = threadIdx.x; i < (s.seqs + 31) / 32; i += PP_THREADS) sh.seen[i] = 0;
    if (threadIdx.x == 0) {
        sh.bad = 0;
        sh.need = 0;
    }
    __syncthreads();
}
// Marks sequence q as named; false where it is out of range or was named before.
__device__ __forceinline__ bool plan_name(const PagesState &s, PlanShared &sh, uint32_t q) {
    return q < s.seqs && !(atomicOr(&sh.seen[q >> 5], 1u << (q & 31)) & (1u << (q & 31)));
}
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, int tshift) {
    return (uint32_t)(((uint64_t)tokens + (1u << tshift) - 1) >> tshift);
}

// The free pages, lowest first: the first `want` ids into s.spare; returns
// how many there are. Reads past L1 (atomics of this call change refs in L2).
__device__ uint32_t free_pages(const PagesState &s, PlanShared &sh, uint32_t want) {
    uint32_t found = 0;
    for (uint32_t base = 0; base < s.pages; base += 4 * PP_THREADS) {
        const uint32_t p = base + 4 * threadIdx.x;
        bool f[4];
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = p + i < s.pages && __ldcg(&s.refs[p + i]) == 0;
            n += f[i];
        }
        uint32_t total, rank = found + block_scan(n, sh.warp_sums, total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (f[i]) {
                if (rank < want) s.spare[rank] = p + i;
                ++rank;
            }
        found += total;
    }
    __syncthreads();  // s.spare is written
    return found;
}

__device__ __forceinline__ void plan_status(const PagesState &s, uint32_t code, uint32_t free_now) {
    if (threadIdx.x == 0) {
        s.status[0] = code;
        s.status[1] = free_now;
    }
}

__global__ void __launch_bounds__(PP_THREADS, 1)
    pages_reserve_kernel(PagesState s, const uint32_t *__restrict__ seqs, const uint32_t *__restrict__ tokens,
                         uint32_t n) {
    __shared__ PlanShared sh;
    const int lane = threadIdx.x & 31;
    plan_begin(s, sh);
    const uint64_t cap = (uint64_t)s.max_pages << s.tshift;
    // 64 bits: a sequence may want 2^26 pages, and there are up to 65536 of them
    unsigned long long want = 0;
    for (uint32_t i = threadIdx.x; i < n; i += PP_THREADS) {
        const uint32_t q = seqs[i];
        const bool ok = plan_name(s, sh, q);
        const uint64_t len = ok ? s.lengths[q] : 0, next = len + tokens[i];
        if (!ok || len > cap || next > cap)
            sh.bad = 1;
        else
            want += pages_of((uint32_t)next, s.tshift) - pages_of((uint32_t)len, s.tshift);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) want += __shfl_xor_sync(0xffffffffu, want, o);
    if (lane == 0 && want) atomicAdd(&sh.need, want);
    __syncthreads();
    const unsigned long long need = sh.need;
    const uint32_t have = free_pages(s, sh, (uint32_t)min(need, (unsigned long long)s.pages));
    if (sh.bad || need > have) {
        plan_status(s, sh.bad ? QWEN_B200_PAGES_BAD : QWEN_B200_PAGES_FULL, have);
        return;
    }
    uint32_t taken = 0;  // (need <= have: the sums below fit 32 bits)
    for (uint32_t base = 0; base < n; base += PP_THREADS) {
        const uint32_t i = base + threadIdx.x;
        uint32_t q = 0, held = 0, mine = 0;
        if (i < n) {
            q = seqs[i];
            const uint32_t len = s.lengths[q], next = len + tokens[i];
            held = pages_of(len, s.tshift);
            mine = pages_of(next, s.tshift) - held;
            s.lengths[q] = next;
        }
        uint32_t total;
        const uint32_t at = taken + block_scan(mine, sh.warp_sums, total);
        taken += total;
        // a warp fills each of its sequences' new entries together
        for (uint32_t todo = __ballot_sync(0xffffffffu, mine > 0); todo; todo &= todo - 1) {
            const int l = __ffs(todo) - 1;
            const uint32_t q2 = __shfl_sync(0xffffffffu, q, l), h2 = __shfl_sync(0xffffffffu, held, l),
                           m2 = __shfl_sync(0xffffffffu, mine, l), a2 = __shfl_sync(0xffffffffu, at, l);
            for (uint32_t j = lane; j < m2; j += 32) {
                const uint32_t page = s.spare[a2 + j];
                s.table[(uint64_t)q2 * s.max_pages + h2 + j] = page;
                s.refs[page] = 1;
            }
        }
    }
    plan_status(s, QWEN_B200_PAGES_OK, have - (uint32_t)need);
}

__global__ void __launch_bounds__(PP_THREADS, 1)
    pages_free_kernel(PagesState s, const uint32_t *__restrict__ seqs, uint32_t n) {
    __shared__ PlanShared sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    plan_begin(s, sh);
    bool bad = false;
    for (uint32_t i = threadIdx.x; i < n; i += PP_THREADS) {
        const uint32_t q = seqs[i];
        bad |= !plan_name(s, sh, q) || s.lengths[q] > (uint64_t)s.max_pages << s.tshift;
    }
    bad = __syncthreads_or(bad);
    // f(page) for every page that the sequences hold, a warp for each of them; whether one was true
    auto any_page = [&](auto f) {
        bool any = false;
        for (uint32_t i = warp; i < n; i += PP_THREADS / 32) {
            const uint32_t q = seqs[i], held = pages_of(s.lengths[q], s.tshift);
            for (uint32_t j = lane; j < held; j += 32) any |= f(s.table[(uint64_t)q * s.max_pages + j]);
        }
        return __syncthreads_or(any) != 0;
    };
    if (!bad) {
        bad = any_page([&](uint32_t page) { return page >= s.pages || atomicSub(&s.refs[page], 1u) == 0; });
        if (bad)  // an id that is no page, or more holders than counted: what was taken goes back
            any_page([&](uint32_t page) { return page < s.pages && (atomicAdd(&s.refs[page], 1u), false); });
        else
            for (uint32_t i = threadIdx.x; i < n; i += PP_THREADS) s.lengths[seqs[i]] = 0;
    }
    __syncthreads();
    const uint32_t have = free_pages(s, sh, 0);
    plan_status(s, bad ? QWEN_B200_PAGES_BAD : QWEN_B200_PAGES_OK, have);
}

__global__ void __launch_bounds__(PP_THREADS, 1)
    pages_fork_kernel(PagesState s, const uint32_t *__restrict__ parents, const uint32_t *__restrict__ children,
                      const uint32_t *__restrict__ prefix, uint32_t n) {
    __shared__ PlanShared sh;
    pdl_trigger();  // the copy kernel waits for this one to end
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    plan_begin(s, sh);
    const uint32_t mask = (1u << s.tshift) - 1;
    uint32_t need = 0;
    for (uint32_t base = 0; base < n; base += PP_THREADS) {
        const uint32_t i = base + threadIdx.x;
        uint32_t mine = 0;
        if (i < n) {
            const uint32_t p = parents[i], c = children[i], len = prefix[i];
            if (p >= s.seqs || !plan_name(s, sh, c) || s.lengths[c] != 0 || len > s.lengths[p] ||
                len > (uint64_t)s.max_pages << s.tshift)
                sh.bad = 1;
            else
                mine = (len & mask) != 0;
        }
        uint32_t total;
        block_scan(mine, sh.warp_sums, total);
        need += total;
    }
    __syncthreads();
    if (!sh.bad) {  // every id of the prefixes, before anything changes; a page that counts as free may be handed out
        for (uint32_t i = warp; i < n; i += PP_THREADS / 32) {
            const uint32_t p = parents[i], held = pages_of(prefix[i], s.tshift);
            for (uint32_t j = lane; j < held; j += 32) {
                const uint32_t page = s.table[(uint64_t)p * s.max_pages + j];
                if (page >= s.pages || s.refs[page] == 0) sh.bad = 1;
            }
        }
    }
    const uint32_t have = free_pages(s, sh, need);
    if (sh.bad || need > have) {
        if (threadIdx.x == 0) *s.count = 0;
        plan_status(s, sh.bad ? QWEN_B200_PAGES_BAD : QWEN_B200_PAGES_FULL, have);
        return;
    }
    // fresh pages for the partial tails (no prefix reads another child's row:
    // a child's length was 0, so as a parent it lends no page)
    uint32_t taken = 0;
    for (uint32_t base = 0; base < n; base += PP_THREADS) {
        const uint32_t i = base + threadIdx.x;
        const uint32_t len = i < n ? prefix[i] : 0, mine = (len & mask) != 0;
        uint32_t total;
        const uint32_t at = taken + block_scan(mine, sh.warp_sums, total);
        taken += total;
        if (mine) {
            const uint32_t page = s.spare[at], full = len >> s.tshift;
            s.list[at] = make_uint4(s.table[(uint64_t)parents[i] * s.max_pages + full], page, len & mask, 0);
            s.table[(uint64_t)children[i] * s.max_pages + full] = page;
            s.refs[page] = 1;
        }
        if (i < n) s.lengths[children[i]] = len;
    }
    for (uint32_t i = warp; i < n; i += PP_THREADS / 32) {
        const uint32_t full = prefix[i] >> s.tshift;
        const uint64_t from = (uint64_t)parents[i] * s.max_pages, to = (uint64_t)children[i] * s.max_pages;
        for (uint32_t j = lane; j < full; j += 32) {
            const uint32_t page = s.table[from + j];
            s.table[to + j] = page;
            atomicAdd(&s.refs[page], 1u);
        }
    }
    if (threadIdx.x == 0) *s.count = need;
    plan_status(s, QWEN_B200_PAGES_OK, have - need);
}

// Plan of a compaction: with L pages in use, free pages below L (holes) and
// used pages at or above it (movers) are equally many and are paired in
// ascending order. A mover is never a hole, so the copies are independent.
__global__ void __launch_bounds__(PP_THREADS, 1) pages_compact_kernel(PagesState s) {
    __shared__ PlanShared sh;
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) sh.bad = 0;
    __syncthreads();
    // Every sequence's length and pages, before anything changes: a page that a table names and refs counts as free
    // would be overwritten by one that moves. A warp has 32 sequences' lengths at a time, and four of them in flight.
    const uint64_t cap = (uint64_t)s.max_pages << s.tshift;
    bool bad = false;
    for (uint32_t base = warp; base < s.seqs; base += PP_THREADS) {
        const uint32_t mine = base + 32 * lane, len = mine < s.seqs ? s.lengths[mine] : 0;
        bad |= len > cap;
        const uint32_t held = len > cap ? 0 : pages_of(len, s.tshift);
        for (int k = 0; k < 32 && base + 32 * k < s.seqs; k += 4) {
            uint32_t h[4], most = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = __shfl_sync(0xffffffffu, held, k + i);
                most = max(most, h[i]);
            }
            for (uint32_t j = lane; j < most; j += 32) {
                uint32_t page[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    page[i] = j < h[i] ? s.table[(uint64_t)(base + 32 * (k + i)) * s.max_pages + j] : PG_NO_PAGE;
#pragma unroll
                for (int i = 0; i < 4; ++i) bad |= j < h[i] && (page[i] >= s.pages || s.refs[page[i]] == 0);
            }
        }
    }
    if (bad) sh.bad = 1;  // (read behind the scans' barriers)
    uint32_t live = 0;
    for (uint32_t base = 0; base < s.pages; base += 4 * PP_THREADS) {
        uint32_t mine = 0, total;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t p = base + 4 * threadIdx.x + i;
            mine += p < s.pages && s.refs[p] != 0;
        }
        block_scan(mine, sh.warp_sums, total);
        live += total;
    }
    if (sh.bad) {
        if (threadIdx.x == 0) *s.count = 0;
        plan_status(s, QWEN_B200_PAGES_BAD, s.pages - live);
        return;
    }
    uint32_t holes = 0, movers = 0;
    for (uint32_t base = 0; base < s.pages; base += 4 * PP_THREADS) {
        const uint32_t p = base + 4 * threadIdx.x;
        bool hit[4];
        uint32_t h = 0, m = 0, total;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const bool used = p + i < s.pages && s.refs[p + i] != 0;
            hit[i] = p + i < s.pages && (p + i < live ? !used : used);
            if (hit[i]) (p + i < live ? h : m) += 1;
        }
        uint32_t hr = holes + block_scan(h, sh.warp_sums, total);
        holes += total;
        uint32_t mr = movers + block_scan(m, sh.warp_sums, total);
        movers += total;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (p + i < s.pages) s.remap[p + i] = p + i;
            if (!hit[i]) continue;
            if (p + i < live)
                s.spare[hr++] = p + i;
            else
                s.list[mr++].x = p + i;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < movers; i += PP_THREADS) {
        const uint32_t src = s.list[i].x, dst = s.spare[i];
        s.list[i] = make_uint4(src, dst, 1u << s.tshift, 0);
        s.remap[src] = dst;
        s.refs[dst] = s.refs[src];
        s.refs[src] = 0;
    }
    if (threadIdx.x == 0) *s.count = movers;
    plan_status(s, QWEN_B200_PAGES_OK, s.pages - live);
}

// ---------------------------------------------------------------- copies
// Copies `tokens` tokens of page src to page dst for each entry of the list,
// in every layer, K and V: 16 KB segments spread over the grid, four 16-byte
// loads in flight per thread. Codes of a whole page are one contiguous run,
// those of a partial page one run per head. `remap` also rewrites the tables.
struct PageCopyArgs {
    uint8_t *pool[2];
    float *scales[2];
    uint64_t layer_rows, page_rows;
    uint32_t layers, pages, hkv, row_bytes;
    int tshift;
    const uint32_t *count;            // nullable: entries of `list`
    const uint4 *list;
    const uint32_t *src, *dst;        // without `list`: n pairs of whole pages
    uint32_t n;
    uint32_t *table;                  // with remap: every sequence's table row
    const uint32_t *lengths, *remap;
    uint32_t seqs, max_pages;
};
constexpr int PC_THREADS = 256;
constexpr uint32_t PC_SEG = PC_THREADS * 4 * 16;

__global__ void __launch_bounds__(PC_THREADS) pages_copy_kernel(PageCopyArgs a) {
    pdl_wait();
    const uint32_t count = a.list ? *a.count : a.n;
    const uint32_t page_bytes = (a.hkv * a.row_bytes) << a.tshift;  // at most 2^14 heads * 2^8 tokens * 2^8 bytes
    const uint32_t segs = (page_bytes + PC_SEG - 1) / PC_SEG;
    const uint64_t work = (uint64_t)count * a.layers * 2 * segs;
    for (uint64_t w = blockIdx.x; w < work; w += gridDim.x) {
        unsigned long long item, seg64, e64, layer64;
        div64(w, segs, item, seg64);
        div64(item >> 1, a.layers, e64, layer64);
        const uint32_t seg = (uint32_t)seg64, which = (uint32_t)(item & 1), layer = (uint32_t)layer64, e = (uint32_t)e64;
        const uint4 m = a.list ? a.list[e] : make_uint4(a.src[e], a.dst[e], 1u << a.tshift, 0);
        if (m.x >= a.pages || m.y >= a.pages) continue;
        const bool whole = m.z == 1u << a.tshift;
        const uint64_t from = layer * a.layer_rows + (uint64_t)m.x * a.page_rows,
                       to = layer * a.layer_rows + (uint64_t)m.y * a.page_rows;
        const uint32_t run = (whole ? page_bytes : m.z * a.row_bytes) >> 4;  // 16-byte units of one run
        const uint32_t units = whole ? run : run * a.hkv;
        const uint32_t run_stride = a.row_bytes << a.tshift;
        const uint8_t *sp = a.pool[which] + from * a.row_bytes;
        uint8_t *dp = a.pool[which] + to * a.row_bytes;
        uint4 x[4];
        uint32_t off[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = seg * (PC_SEG / 16) + i * PC_THREADS + threadIdx.x;
            off[i] = 0xffffffffu;
            if (u < units) {
                off[i] = whole ? u << 4 : (u / run) * run_stride + ((u % run) << 4);
                x[i] = ldg_stream(sp + off[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (off[i] != 0xffffffffu) *reinterpret_cast<uint4 *>(dp + off[i]) = x[i];
        if (a.scales[which] && seg == 0) {
            for (uint32_t u = threadIdx.x; u < a.hkv << a.tshift; u += PC_THREADS)
                if ((u & ((1u << a.tshift) - 1)) < m.z) a.scales[which][to + u] = a.scales[which][from + u];
        }
    }
    if (!a.remap || count == 0) return;  // (no page moves: the tables stand)
    const uint32_t warps = gridDim.x * (PC_THREADS / 32);
    for (uint32_t q = blockIdx.x * (PC_THREADS / 32) + (threadIdx.x >> 5); q < a.seqs; q += warps) {
        const uint32_t held = min(pages_of(a.lengths[q], a.tshift), a.max_pages);
        for (uint32_t j = threadIdx.x & 31; j < held; j += 32) {
            uint32_t *t = a.table + (uint64_t)q * a.max_pages + j;
            const uint32_t page = *t;
            if (page < a.pages) *t = a.remap[page];
        }
    }
}

static PageCopyArgs copy_args(const qwen_b200_paged_kv &kv) {
    PageCopyArgs a = {};
    a.pool[0] = (uint8_t *)kv.k;
    a.pool[1] = (uint8_t *)kv.v;
    if (kv.format == QWEN_B200_KV8) {
        a.scales[0] = kv.kscales;
        a.scales[1] = kv.vscales;
    }
    a.layer_rows = kv.layer_stride;
    a.page_rows = kv.page_stride;
    a.layers = kv.layers;
    a.pages = kv.pages;
    a.hkv = kv.kv_heads;
    a.row_bytes = paged_row_bytes(kv);
    a.tshift = __builtin_ctz(kv.page_tokens);
    return a;
}

static int launch_copy(const qwen_b200_paged_kv &kv, const PageCopyArgs &a, uint64_t most, cudaStream_t st) {
    const uint64_t page_bytes = (uint64_t)kv.kv_heads * kv.page_tokens * a.row_bytes;
    const uint64_t segs = (page_bytes + PC_SEG - 1) / PC_SEG;
    const int sms = paged_sms();
    if (!sms) return -3;
    const uint64_t work = most * kv.layers * 2 * segs;
    const unsigned grid = (unsigned)(work < 8ull * sms ? work : 8ull * sms);
    return launch_pdl(pages_copy_kernel, dim3(grid), dim3(PC_THREADS), 0, st, 1, a);
}

// ---------------------------------------------------------------- launchers
int launch_pages_reserve(const qwen_b200_paged_kv &kv, const uint32_t *seqs, const uint32_t *tokens, uint32_t n,
                         uint32_t *status, void *ws, cudaStream_t st) {
    pages_reserve_kernel<<<1, PP_THREADS, 0, st>>>(pages_state(kv, status, ws), seqs, tokens, n);
    return QB_LAUNCH_CHECK();
}

int launch_pages_free(const qwen_b200_paged_kv &kv, const uint32_t *seqs, uint32_t n, uint32_t *status,
                      cudaStream_t st) {
    pages_free_kernel<<<1, PP_THREADS, 0, st>>>(pages_state(kv, status, nullptr), seqs, n);
    return QB_LAUNCH_CHECK();
}

int launch_pages_fork(const qwen_b200_paged_kv &kv, const uint32_t *parents, const uint32_t *children,
                      const uint32_t *prefix, uint32_t n, uint32_t *status, void *ws, cudaStream_t st) {
    const PagesState s = pages_state(kv, status, ws);
    PdlChain chain;
    if (int rc = launch_pdl(pages_fork_kernel, dim3(1), dim3(PP_THREADS), 0, st, 1, s, parents, children, prefix, n))
        return rc;
    PageCopyArgs a = copy_args(kv);
    a.count = s.count;
    a.list = s.list;
    return launch_copy(kv, a, n, st);
}

int launch_pages_compact(const qwen_b200_paged_kv &kv, uint32_t *status, void *ws, cudaStream_t st) {
    const PagesState s = pages_state(kv, status, ws);
    PdlChain chain;
    if (int rc = launch_pdl(pages_compact_kernel, dim3(1), dim3(PP_THREADS), 0, st, 1, s)) return rc;
    PageCopyArgs a = copy_args(kv);
    a.count = s.count;
    a.list = s.list;
    a.table = kv.table;
    a.lengths = kv.lengths;
    a.remap = s.remap;
    a.seqs = kv.seqs;
    a.max_pages = kv.max_pages;
    return launch_copy(kv, a, kv.pages, st);
}

int launch_pages_copy(const qwen_b200_paged_kv &kv, const uint32_t *src, const uint32_t *dst, uint32_t n,
                      cudaStream_t st) {
    PageCopyArgs a = copy_args(kv);
    a.src = src;
    a.dst = dst;
    a.n = n;
    return launch_copy(kv, a, n, st);
}

}  // namespace qb
