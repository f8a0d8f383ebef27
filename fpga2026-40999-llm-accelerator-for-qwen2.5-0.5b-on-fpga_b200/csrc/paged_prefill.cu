// Causal attention of the newest rows of several sequences over their pages,
// with a sliding window and first tokens that stay visible; both products on
// the tensor cores (tcgen05.mma kind::f16, bf16 operands, fp32 accumulators in
// TMEM).
//
// Mathematics, per (row, query head), over its visible keys j in blocks of 128:
//   x_j = log2(e) scale q.k_j,  p_j = 2^(x_j - m),  ctx = sum p_j v_j / sum p_j
// m is a reference for 2^x in place of the running maximum: fp32 and bf16 keep
// their relative precision far above and below 1, so it starts at 0 and only
// moves where the weights of some keys sum to more than 2^15 (or the first ones
// to less than 2^-20), and most keys need no comparison and no rescaling. The
// weights are rounded to bf16 for the second product (half a step is 2^-8 of a
// weight, unbiased); bf16 pools sum the rounded ones, so that a row's dominant
// key cancels exactly. Everything else is fp32. KV8: codes become bf16 exactly
// on the way to shared memory, the key's scale multiplies its column of scores
// and the value's scale its column of weights.
//
// Tiles: the rows of a sequence and the query heads that share a KV head are one
// axis (row-major: token, head), cut into tiles of 512 (64 dims) or 256 (128
// dims) = four or two MMA tiles of 128 rows, so any group size fills them and a
// block of keys is read once for all of them. Per tile only the blocks that
// some row sees are visited. All (tile, KV head, block) units are numbered in a
// row and CTA c of G takes the c-th equal run: long and short prompts, windows
// and single rows balance by themselves, and few rows over many keys split
// along the keys. A tile that two or more CTAs share is joined by a second
// kernel (at most two pieces per CTA, fp32, added in CTA order).
//
// A step is 64 keys (half a block) of one MMA tile: scores into 64 TMEM columns,
// weights (bf16) back over them, second product into the tile's context
// columns. At 64 dims TMEM holds four tiles with one score buffer each, at 128
// dims two tiles with two each: either way four steps are in flight and the
// tensor cores work on three while the softmax has one. (64 dims with two buffers
// of 32 keys for each tile: 390 us for the first case below, against 336 with the
// softmax code of that time.)
//
// Warps (one CTA per SM, registers moved to the softmax warps):
//   0 ..      four softmax warps per MMA tile, one thread per row
//   then 4    tile warps: queries (cp.async), key masks and scales, KV8 codes to
//             bf16, bf16 values that are not visible to 0 (what a page
//             holds there never reaches the products); 128-byte swizzled
//             K-major tiles, the value tile read as an MN-major operand
//   then 2    a thread of each issues the MMAs of every second tile (with one
//             issuer the tensor cores idled while it waited for the next weights)
//   1         walks the units and publishes segments (tile, KV head, block
//             range), then zeroes the rows in front of a sequence's first token
//   1         copies pages into shared memory: KV8 codes by bulk copies, bf16 rows by TMA
// Measured: 8 prompts of 4096 rows, window 1024, 14 heads on 2 of 64 dims, KV8:
// 303 us, 350 TF/s (the exponentials alone, 16 per clock and SM, take 117 us, the
// products 64). 3 prompts of up to 8192 rows, window 4096, 32 heads on 8 of 128
// dims, bf16: 517 us, 764 TF/s on the same inputs again and again, 545 us, 725
// TF/s (44 % of the GEMM rate) on new ones each time. Bound by the chain from
// scores to weights to product within a tile: without any softmax work the two
// still take 230 and 456 us, and issue slots (47 and 41 % busy), exponentials
// (32 and 42 %) and tensor cores (19 and 44 %) all have room. 16 rows on 1000
// keys take 18.6 us, the latency of two launches and of a CTA's one pass.
// Every wait is bounded (error codes 57-69).
#include <type_traits>

#include "kernels.h"
#include "paged.cuh"
#include "tc05.cuh"

namespace qb {

constexpr int PP_BLK = 128;
constexpr int PP_MAX_SMS = 192;
constexpr uint32_t PP_MIN_UNITS = 1;  // blocks a CTA takes at least (16 rows on 276 keys: 2 us more with 2, 6 us more with 4)
constexpr int PP_SC = 4;              // blocks of scales and key masks in flight
constexpr int PP_SEG = 2;             // segments published ahead

template <bool KV8, int DIM>
struct PpCfg {
    static constexpr int TILES = DIM == 64 ? 4 : 2, NB = 4 / TILES;  // MMA tiles, score buffers of each
    static constexpr int TILE = 128 * TILES;                         // flattened rows of a tile
    static constexpr int SW = 4 * TILES, WARPS = SW + 8, THREADS = 32 * WARPS;
    static constexpr int HALVES = DIM / 64;
    static constexpr int TILE_BYTES = 128 * 128 * HALVES;  // 128 rows of DIM bf16, 64 dims per swizzled half
    // K and V tiles in flight (K0 V0 K1 V1 ..), and KV8 tiles as codes in front of them
    static constexpr int SLOTS = DIM == 64 ? 4 : KV8 ? 3 : 4;
    static constexpr int RAW = KV8 ? 2 : SLOTS / 2, RAW_BYTES = KV8 ? 128 * DIM : 0;
    static constexpr int QBUFS = DIM == 64 ? 2 : 1;        // the next segment's queries load behind the current one
    static constexpr int Q = 0, RING = QBUFS * TILES * TILE_BYTES;
    static constexpr int CODES = RING + SLOTS * TILE_BYTES;  // [RAW][128][DIM] codes
    static constexpr int SC = CODES + RAW * RAW_BYTES;       // [PP_SC][ks 128 | vs 128] floats, [PP_SC][4] mask words
    static constexpr int MASK = SC + PP_SC * 256 * 4;
    static constexpr int SEG = MASK + PP_SC * 16;
    static constexpr int BARS = SEG + PP_SEG * 64;
    static constexpr int NBARS = 2 * SLOTS + 2 * PP_SC + 2 * PP_SEG + 13 + 2 * RAW;
    static constexpr int SLOT = BARS + NBARS * 8;
    static constexpr int TOTAL = SLOT + 16;
    static constexpr int ALLOC = TOTAL + 1024;
    static constexpr int PIECE = 2 * TILE + TILE * DIM;  // floats: m, l, o
    static_assert(ALLOC <= 232448, "shared memory per CTA");
    static_assert(KV8 || SLOTS % 2 == 0, "bf16: even slots hold keys, odd ones values");
};

// One tile's run of blocks for one KV head.
struct PpSeg {
    uint32_t seq, row0, m0, mrows;  // rows of q from row0; flattened rows m0 .. of mrows
    int pos0;                       // position of the sequence's first row (negative: more rows than tokens)
    uint32_t kvh;
    int b0, nblk;                   // virtual blocks; nblk 0 ends the list
    int s128, low128;               // virtual block b: b < s128 ? b : b - s128 + low128
    int first, low, last;           // keys that some row sees: [0, first) and [low, last]
    int piece;                      // -1: the tile's whole list; else the piece's index
    int pad[2];
};
static_assert(sizeof(PpSeg) == 64, "segment record");

struct PpRec {  // the tile that a CTA starts in the middle of
    uint32_t valid, row0, m0, mrows, kvh, c0, c1, slot0;
    int pos0;
    uint32_t pad[7];
};
static_assert(sizeof(PpRec) == 64, "join record");

struct PpWork {
    uint32_t group, max_ctas;
    uint32_t tile;   // flattened rows of a tile
    float fac;       // log2(e) |scale|
    uint32_t negate; // scale < 0: the first product negates the queries
    unsigned *err;
    PpRec *recs;     // [max_ctas]
    float *pieces;   // [max_ctas][2][PIECE]
};

struct PpMaps {  // bf16 pools
    CUtensorMap k, v;
};

struct PpSeqInfo {
    uint32_t row0, seq, rows, mrows;
    int pos0, nt;
};
__device__ __forceinline__ PpSeqInfo pp_seq(const PagedAttnArgs &a, const PpWork &w, uint32_t i) {
    PpSeqInfo s;
    const uint32_t s0 = min(a.starts[i], a.rows), s1 = min(max(a.starts[i + 1], s0), a.rows);
    s.row0 = s0;
    s.seq = a.seqs ? a.seqs[i] : i;
    s.rows = s1 - s0;
    s.mrows = s.rows * w.group;
    const int len = paged_length(a.c, s.seq);
    s.pos0 = len - (int)s.rows;
    s.nt = len > 0 ? (int)((s.mrows + w.tile - 1) / w.tile) : 0;
    return s;
}
// Rows of a sequence in front of its first token (all of them, where there is no token or no sequence): zero.
__device__ __forceinline__ uint32_t pp_dead(const PpSeqInfo &s) {
    return s.pos0 >= 0 ? 0u : min((uint32_t)-s.pos0, s.rows);
}
// The most of them that one CTA's warp writes alone; more are shared by all CTAs, each of which then looks at each such
// sequence: 14 heads of 64 dims, alone against shared, one sequence of 4096 rows 842 and 17 us, 256 of 200 rows 92 and
// 129, 256 of 48 rows 29 and 70, 4096 of 40 rows 254 and 794.
__device__ __forceinline__ uint32_t pp_dead_alone(const PagedAttnArgs &a) { return max(32u, a.n); }
struct PpBlocks {
    int s128, low128, first, low, last, n;
};
__device__ __forceinline__ PpBlocks pp_blocks(const PagedAttnArgs &a, const PpWork &w, int pos0, uint32_t mrows, int k) {
    PpBlocks b;
    const uint32_t m0 = (uint32_t)k * w.tile, m1 = min(m0 + w.tile, mrows) - 1;
    const int pmin = max(pos0 + (int)(m0 / w.group), 0);
    b.last = pos0 + (int)(m1 / w.group);
    b.low = key_span(pmin, a.window, a.sinks).low;
    b.first = key_span(max(b.last, 0), a.window, a.sinks).first;
    b.low128 = b.low >> 7;
    b.s128 = min((b.first + 127) >> 7, b.low128);
    b.n = b.last < 0 ? 0 : b.s128 + (b.last >> 7) + 1 - b.low128;
    return b;
}
// Blocks of a sequence's tiles, summed by a whole warp.
__device__ __forceinline__ uint32_t pp_units_warp(const PagedAttnArgs &a, const PpWork &w, int pos0, uint32_t mrows,
                                                  int nt) {
    uint32_t u = 0;
    for (int k = threadIdx.x & 31; k < nt; k += 32) u += pp_blocks(a, w, pos0, mrows, k).n;
    return __reduce_add_sync(0xffffffffu, u);
}
// Blocks of the sequences base + lane < end, one per lane; `dead` is set where the rows of one are zeroed by all CTAs.
__device__ __forceinline__ uint32_t pp_units_lane(const PagedAttnArgs &a, const PpWork &w, uint32_t base, uint32_t end,
                                                  bool &dead) {
    const uint32_t i = base + (threadIdx.x & 31);
    PpSeqInfo s = {};
    uint32_t u = 0;
    if (i < end) {
        s = pp_seq(a, w, i);
        if (pp_dead(s) > pp_dead_alone(a)) dead = true;
        if (s.nt <= 4)
            for (int k = 0; k < s.nt; ++k) u += pp_blocks(a, w, s.pos0, s.mrows, k).n;
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, s.nt > 4); todo; todo &= todo - 1) {
        const int l = __ffs(todo) - 1;
        const uint32_t x = pp_units_warp(a, w, __shfl_sync(0xffffffffu, s.pos0, l), __shfl_sync(0xffffffffu, s.mrows, l),
                                         __shfl_sync(0xffffffffu, s.nt, l));
        if ((int)(threadIdx.x & 31) == l) u = x;
    }
    return u;
}

// ---------------------------------------------------------------- tcgen05
// kind::f16: D f32, A and B bf16, M 128.
__host__ __device__ constexpr uint32_t pp_idesc(int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void pp_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void pp_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
// Descriptor of the value tile as an MN-major operand (dims contiguous): rows
// (keys) of 128 bytes = 64 dims, 8-row groups 1024 bytes apart, the next 64
// dims one half further.
__device__ __forceinline__ uint64_t pp_desc_mn(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)((128u * 128u) >> 4) << 16;  // leading byte offset: next 64 dims
    d |= (uint64_t)(1024u >> 4) << 32;          // stride byte offset: next 8 keys
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;  // SWIZZLE_128B
    return d;
}
#define PP_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define PP_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void pp_st32(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PP_W8(r, 0),
        PP_W8(r, 8), PP_W8(r, 16), PP_W8(r, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void pp_ld16(uint32_t addr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : PP_R8(r, 0), PP_R8(r, 8)
                 : "r"(addr));
}
__device__ __forceinline__ void pp_st16(uint32_t addr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::PP_W8(
                     r, 0),
                 PP_W8(r, 8), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void pp_ld8(uint32_t addr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : PP_R8(r, 0) : "r"(addr));
}
__device__ __forceinline__ void pp_st8(uint32_t addr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::PP_W8(r, 0), "r"(addr) : "memory");
}
__device__ __forceinline__ void pp_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pp_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float pp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pp_pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ void pp_cp16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pp_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pp_cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void pp_sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Byte offset of 16-byte chunk c (of DIM / 8) of row r in a swizzled tile.
__device__ __forceinline__ uint32_t pp_off(int r, int c) {
    return (uint32_t)((c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void pp_tma_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// One lane of a converged warp. A branch on its result is known to the compiler to
// be taken by one thread, so that tcgen05 instructions inside it take their
// operands from uniform registers directly; under `lane == 0` each of
// them cost 110-150 cycles of issue (half of the kernel's time).
__device__ __forceinline__ bool pp_elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// tc::mbar_wait in few instructions: the compiler unrolls its loop, and the
// kernel has some 50 of them (147 KB of text in all with them unrolled, 95 KB so).
__device__ __forceinline__ bool pp_wait(uint64_t *bar, uint32_t parity, unsigned *err, unsigned code) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 21); ++i)
        if (tc::mbar_try_wait(bar, parity)) return true;
    atomicExch(err, code);
    return false;
}

// The reading side of the segment ring.
struct PpReader {
    const PpSeg *ring;
    uint64_t *full, *empty;
    uint32_t n = 0;
    // Copies the next segment; every lane of the warp calls it. false: a wait ran out.
    __device__ __forceinline__ bool next(PpSeg &s, unsigned *err) {
        const uint32_t d = n % PP_SEG;
        const bool ok = pp_wait(&full[d], (n / PP_SEG) & 1, err, 60);
        s = ring[d];
        __syncwarp();
        if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&empty[d]);
        ++n;
        return __all_sync(0xffffffffu, ok);
    }
};

template <bool KV8, int DIM>
__global__ void __launch_bounds__(PpCfg<KV8, DIM>::THREADS, 1) paged_prefill_kernel(const __grid_constant__ PpMaps maps, PagedAttnArgs a, PpWork w) {
    using C = PpCfg<KV8, DIM>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ unsigned long long wsum[C::WARPS], at_prefix;
    __shared__ uint32_t at_seq, wdead[C::WARPS];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = tc::smem_u32(sm);
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + C::BARS);
    uint64_t *kv_full = bars, *kv_empty = kv_full + C::SLOTS, *sc_full = kv_empty + C::SLOTS, *sc_empty = sc_full + PP_SC;
    uint64_t *seg_full = sc_empty + PP_SC, *seg_empty = seg_full + PP_SEG;
    uint64_t *q_full = seg_empty + PP_SEG, *q_empty = q_full + 2, *s_full = q_full + 4, *p_ready = q_full + 8,
             *mdone = q_full + 12, *raw_full = mdone + 1, *raw_empty = raw_full + C::RAW;
    uint32_t *slot_p = reinterpret_cast<uint32_t *>(sm + C::SLOT);
    float *scales = reinterpret_cast<float *>(sm + C::SC);
    uint32_t *masks = reinterpret_cast<uint32_t *>(sm + C::MASK);
    PpSeg *ring = reinterpret_cast<PpSeg *>(sm + C::SEG);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_trigger();  // the join kernel waits for this one to end

    if (tid == 0) {
        for (int i = 0; i < C::SLOTS; ++i) {
            tc::mbar_init(&kv_full[i], KV8 || (i & 1) ? 4 : 1);  // the converting warps; bf16 keys: the copy itself
            tc::mbar_init(&kv_empty[i], 2);  // both issuers
        }
        for (int i = 0; i < PP_SC; ++i) {
            tc::mbar_init(&sc_full[i], 4);
            tc::mbar_init(&sc_empty[i], C::SW);
        }
        for (int i = 0; i < PP_SEG; ++i) {
            tc::mbar_init(&seg_full[i], 1);
            tc::mbar_init(&seg_empty[i], 7 + C::SW);  // 4 tile warps, the copy warp, 2 issuers, the softmax warps
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&q_full[i], 4);
            tc::mbar_init(&q_empty[i], 2);
        }
        for (int i = 0; i < 4; ++i) {  // [tile][score buffer]
            tc::mbar_init(&s_full[i], 1);
            tc::mbar_init(&p_ready[i], 4);
        }
        tc::mbar_init(mdone, 2);
        for (int i = 0; i < C::RAW; ++i) {
            tc::mbar_init(&raw_full[i], 1);
            tc::mbar_init(&raw_empty[i], 4);
        }
        tc::mbar_fence_init();
    }
    if (warp == C::SW + 4) tc::tmem_alloc(slot_p, 512);

    // ---- numbering of the units: a warp takes a run of sequences
    const uint32_t per = (a.n + C::WARPS - 1) / C::WARPS, i0 = min(warp * per, a.n), i1 = min(i0 + per, a.n);
    unsigned long long mine = 0;
    bool dead = false;
    for (uint32_t b = i0; b < i1; b += 32) mine += __reduce_add_sync(0xffffffffu, pp_units_lane(a, w, b, i1, dead));
    dead = __any_sync(0xffffffffu, dead);
    if (lane == 0) {
        wsum[warp] = mine;
        wdead[warp] = dead;
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *slot_p;
    unsigned long long before = 0, all = 0;
    for (int i = 0; i < C::WARPS; ++i) {
        if (i < warp) before += wsum[i];
        all += wsum[i];
    }
    const UnitSplit split(all * a.c.hkv, w.max_ctas, PP_MIN_UNITS);
    const bool active = blockIdx.x < split.g && all > 0;
    const unsigned long long u0 = split.start(blockIdx.x), u1 = split.start(blockIdx.x + 1);
    if (active && before * a.c.hkv <= u0 && u0 < (before + mine) * a.c.hkv) {
        unsigned long long p = before;
        for (uint32_t b = i0; b < i1; b += 32) {
            uint32_t u = pp_units_lane(a, w, b, i1, dead), x = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const bool here = (p + x - u) * a.c.hkv <= u0 && u0 < (p + x) * a.c.hkv;
            if (here) {
                at_seq = b + lane;
                at_prefix = p + x - u;
            }
            if (__any_sync(0xffffffffu, here)) break;
            p += __shfl_sync(0xffffffffu, x, 31);
        }
    }
    __syncthreads();
    bool ok = true;

    if (!active) {
        // ---------------- nothing to compute
        if (tid == 0) w.recs[blockIdx.x].valid = 0;
    } else if (warp < C::SW) {
        // ---------------- softmax: thread = row r of MMA tile `x`
        if constexpr (DIM == 64)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
        else
            asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int x = warp >> 2, r = tid & 127;
        const uint32_t lane_addr = tmem + ((uint32_t)(warp & 3) << 21);  // lanes 32 (warp % 4) ..
        const uint32_t s_base = lane_addr + x * (64 * C::NB), o_addr = lane_addr + 256 + x * DIM;
        uint64_t *const s_bar = s_full + x * C::NB, *const p_bar = p_ready + x * C::NB;
        PpReader rd{ring, seg_full, seg_empty};
        uint32_t bc = 0, round = 0;  // blocks of the CTA; rounds of this tile's score barriers before the segment
        PpSeg g;
        while (ok) {
            ok = rd.next(g, w.err);
            if (!ok || g.nblk == 0) break;
            const uint32_t mt = g.m0 + 128 * x;  // this MMA tile's first flattened row
            if (mt >= g.mrows) {                 // no rows: only let the scales go
                for (int i = 0; i < g.nblk && ok; ++i, ++bc) {
                    ok = __all_sync(0xffffffffu, pp_wait(&sc_full[bc % PP_SC], (bc / PP_SC) & 1, w.err, 61));
                    if (lane == 0) tc::mbar_arrive(&sc_empty[bc % PP_SC]);
                }
                continue;
            }
            const uint32_t m_row = mt + r, row_i = m_row / w.group;
            const int pos = m_row < g.mrows ? g.pos0 + (int)row_i : -1;
            const KeySpan ks = key_span(max(pos, 0), a.window, a.sinks);
            const int first = pos < 0 ? 0 : ks.first, low = ks.low;
            // keys seen by every row of the MMA tile: [0, all_first) and [all_low, all_last]
            const uint32_t m_end = min(mt + 128, g.mrows) - 1;
            const int all_last = m_end == mt + 127 ? g.pos0 + (int)(mt / w.group) : -1;
            const int all_first = key_span(max(all_last, 0), a.window, a.sinks).first;
            const int all_low = key_span(max(g.pos0 + (int)(m_end / w.group), 0), a.window, a.sinks).low;
            // The reference starts at 0 and stands if the weights of the row's first keys sum to something in
            // [2^-20, 2^15] (scores within some 15 of 0, the usual case); else it becomes their maximum.
            float m = 0.f, l = 0.f;
            bool fresh = true;  // no key seen yet
            bool far = false;   // some row's reference is so large that x has to be rounded before it is subtracted
            const uint32_t steps = 2 * g.nblk;
            uint32_t st = 0;
            int kb = 0;
            for (uint32_t n = 0; n < steps && ok; ++n) {
                const int h = n & 1;
                if (h == 0) {
                    const int vb = g.b0 + (int)(n >> 1);
                    kb = (vb < g.s128 ? vb : vb - g.s128 + g.low128) * PP_BLK;
                    st = bc % PP_SC;
                    ok = pp_wait(&sc_full[st], (bc / PP_SC) & 1, w.err, 61);
                }
                const uint32_t buf = n % C::NB, sh = s_base + 64 * buf;
                ok = __all_sync(0xffffffffu, ok && pp_wait(&s_bar[buf], (round + n / C::NB) & 1, w.err, 62));
                if (!ok) break;
                tc::tc_fence_after();
                const int k0 = kb + 64 * h;
                const float4 *kf = reinterpret_cast<const float4 *>(scales + st * 256 + 64 * h), *vf = kf + 32;
                const uint2 there = *reinterpret_cast<const uint2 *>(masks + 4 * st + 2 * h);
                // the 64 keys' visibility to this row
                uint32_t bits[2] = {there.x, there.y};
                const bool full = k0 + 63 <= all_last && (k0 >= all_low || k0 + 64 <= all_first) &&
                                  (there.x & there.y) == 0xffffffffu;
                if (!full) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        auto below = [&](int e) {  // bits j with k0 + 32 k + j < e
                            const int d = e - (k0 + 32 * k);
                            return d >= 32 ? 0xffffffffu : d <= 0 ? 0u : (1u << d) - 1;
                        };
                        bits[k] &= below(pos + 1) & (~below(low) | below(first));
                    }
                }
                // 64 at once at 64 dims: 336 us against 303 for the first case above; 32 at 128 dims: 535 us against
                // 517 for the second. A second copy of this code behind the test, for the rows that fail it,
                // in place of the path below: 338 and 543 us.
                constexpr int COLS = DIM == 64 ? 32 : 64;
                int c = 0;  // keys done
                if (full && !far) {
                    // every key counts: the weights as they are with the row's reference, unless they sum to more
                    // than 2^15 or a row's first ones to less than 2^-20
#pragma unroll 1
                    for (; c < 64; c += COLS) {
                        uint32_t p[COLS / 2];
                        const float4 *kc = kf + c / 4, *vc = vf + c / 4;
                        unsigned long long part[2] = {0ull, 0ull};
                        const unsigned long long mu = dup2(-m);
#pragma unroll
                        for (int b = 0; b < COLS; b += 8) {  // (16 or 32 at a time: 1 % slower)
                            float s[8];
                            pp_ld8(sh + c + b, reinterpret_cast<uint32_t *>(s));
                            pp_ld_wait();
#pragma unroll
                            for (int i = 0; i < 8; i += 4) {
                                const int j = b + i;
                                float e[4], f[4] = {w.fac, w.fac, w.fac, w.fac};
                                if constexpr (KV8) {
                                    const float4 k4 = kc[j >> 2];
                                    f[0] = k4.x, f[1] = k4.y, f[2] = k4.z, f[3] = k4.w;
                                }
                                unpk2(fma2(pk2(s[i], s[i + 1]), pk2(f[0], f[1]), mu), e[0], e[1]);
                                unpk2(fma2(pk2(s[i + 2], s[i + 3]), pk2(f[2], f[3]), mu), e[2], e[3]);
#pragma unroll
                                for (int k = 0; k < 4; ++k) e[k] = pp_ex2(e[k]);
                                if constexpr (KV8) {
                                    part[0] = add2(part[0], pk2(e[0], e[1]));
                                    part[1] = add2(part[1], pk2(e[2], e[3]));
                                    const float4 v4 = vc[j >> 2];
                                    unpk2(mul2(pk2(e[0], e[1]), pk2(v4.x, v4.y)), e[0], e[1]);
                                    unpk2(mul2(pk2(e[2], e[3]), pk2(v4.z, v4.w)), e[2], e[3]);
                                }
                                p[j / 2] = pp_pack(e[0], e[1]);
                                p[j / 2 + 1] = pp_pack(e[2], e[3]);
                                if constexpr (!KV8) {  // the rounded weights: what dominates a row cancels exactly
                                    part[0] = add2(part[0], pk2(bflo(p[j / 2]), bfhi(p[j / 2])));
                                    part[1] = add2(part[1], pk2(bflo(p[j / 2 + 1]), bfhi(p[j / 2 + 1])));
                                }
                            }
                        }
                        float a0, a1;
                        unpk2(add2(part[0], part[1]), a0, a1);
                        const float sum = a0 + a1;
                        if (__builtin_expect(__any_sync(0xffffffffu, sum > 32768.f || (fresh && sum < 0x1p-20f)), 0)) break;
                        fresh = false;
                        l += sum;
                        // over columns whose scores have been read
                        if constexpr (COLS == 64)
                            pp_st32(sh, p);
                        else
                            pp_st16(sh + c / 2, p);
                    }
                }
                if (c == 64) {
                } else if (__any_sync(0xffffffffu, (bits[0] | bits[1]) != 0)) {
                    // The same for some of the keys, 32 at a time. Where it does not do, the reference moves to the
                    // largest of them and their weights are formed anew (the scores are still in TMEM): for a row that
                    // has summed something by a whole number, so that what is done is rescaled exactly.
#pragma unroll 1
                    for (; c < 64; c += 32) {
                        const uint32_t sc = sh + c, bt = c == 0 ? bits[0] : bits[1];
                        const float4 *kc = kf + c / 4, *vc = vf + c / 4;
                        uint32_t p[16];
                        if (!__any_sync(0xffffffffu, bt != 0)) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) p[j] = 0;
                            pp_st16(sh + c / 2, p);
                            continue;
                        }
                        float sum;
#pragma unroll 1
                        for (bool again = false;; again = true) {
                            unsigned long long part[2] = {0ull, 0ull};
#pragma unroll
                            for (int b = 0; b < 32; b += 8) {
                                float s[8];
                                pp_ld8(sc + b, reinterpret_cast<uint32_t *>(s));
                                pp_ld_wait();
#pragma unroll
                                for (int i = 0; i < 8; i += 4) {
                                    const int j = b + i;
                                    float e[4], f[4] = {w.fac, w.fac, w.fac, w.fac};
                                    if constexpr (KV8) {
                                        const float4 k4 = kc[j >> 2];
                                        f[0] = k4.x, f[1] = k4.y, f[2] = k4.z, f[3] = k4.w;
                                    }
#pragma unroll
                                    for (int k = 0; k < 4; ++k) {  // x rounded before m is subtracted, as below
                                        const float y = __fadd_rn(__fmul_rn(s[i + k], f[k]), -m);
                                        e[k] = pp_ex2(bt & (1u << (j + k)) ? y : -INFINITY);
                                    }
                                    if constexpr (KV8) {
                                        part[0] = add2(part[0], pk2(e[0], e[1]));
                                        part[1] = add2(part[1], pk2(e[2], e[3]));
                                        const float4 v4 = vc[j >> 2];
                                        unpk2(mul2(pk2(e[0], e[1]), pk2(v4.x, v4.y)), e[0], e[1]);
                                        unpk2(mul2(pk2(e[2], e[3]), pk2(v4.z, v4.w)), e[2], e[3]);
#pragma unroll
                                        for (int k = 0; k < 4; ++k)  // 0 whatever the scale of a value that the row does not see
                                            e[k] = bt & (1u << (j + k)) ? e[k] : 0.f;
                                    }
                                    p[j / 2] = pp_pack(e[0], e[1]);
                                    p[j / 2 + 1] = pp_pack(e[2], e[3]);
                                    if constexpr (!KV8) {
                                        part[0] = add2(part[0], pk2(bflo(p[j / 2]), bfhi(p[j / 2])));
                                        part[1] = add2(part[1], pk2(bflo(p[j / 2 + 1]), bfhi(p[j / 2 + 1])));
                                    }
                                }
                            }
                            float a0, a1;
                            unpk2(add2(part[0], part[1]), a0, a1);
                            sum = a0 + a1;
                            const bool lift = sum > 32768.f || (fresh && bt != 0 && sum < 0x1p-20f);
                            // once more at most: then the largest weight is in (1/2, 1] and the sum at most 32 (or NaN)
                            if (again || !__any_sync(0xffffffffu, lift)) break;
                            float top = -INFINITY;
#pragma unroll 1
                            for (int j = 0; j < 32; j += 8) {
                                uint32_t o[8];
                                pp_ld8(sc + j, o);
                                pp_ld_wait();
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float f = KV8 ? reinterpret_cast<const float *>(kc)[j + k] : w.fac;
                                    if (bt >> (j + k) & 1) top = fmaxf(top, __fmul_rn(__uint_as_float(o[k]), f));
                                }
                            }
                            // 2^-by in two factors (nothing that counts is that far below: 0 beyond 2^-252)
                            float f = 1.f, f2 = 1.f;
                            if (lift) {
                                const float by = ceilf(top - m);
                                if (fresh || by > 252.f) {
                                    f = 0.f;
                                    m = top;
                                } else if (by > 0.f) {
                                    const int d = (int)by;
                                    f = pow2i(-(d >> 1));
                                    f2 = pow2i(-(d - (d >> 1)));
                                    m += by;
                                }
                            }
                            l = l * f * f2;
                            // scores so large that their own rounding shows: an fma would weigh equal ones
                            // differently here and above, by 2^-12 at this size and without bound beyond
                            far = far || __any_sync(0xffffffffu, fabsf(m) > 4096.f);
                            if (n > 0) {
                                // every product into the context so far is complete: those over this buffer precede
                                // its scores, that over the other buffer precedes that buffer's next scores
                                if (C::NB == 2)
                                    ok = __all_sync(0xffffffffu, pp_wait(&s_bar[buf ^ 1], (round + (n + 1) / C::NB) & 1, w.err, 63));
                                tc::tc_fence_after();
#pragma unroll 1
                                for (int j = 0; j < DIM; j += 8) {
                                    uint32_t o[8];
                                    pp_ld8(o_addr + j, o);
                                    pp_ld_wait();
#pragma unroll
                                    for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f * f2);
                                    pp_st8(o_addr + j, o);
                                }
                            }
#pragma unroll 1
                            for (int j = 0; j < c / 2; j += 8) {  // this step's weights so far
                                uint32_t o[8];
                                pp_st_wait();
                                pp_ld8(sh + j, o);
                                pp_ld_wait();
#pragma unroll
                                for (int k = 0; k < 8; ++k) o[k] = pp_pack(bflo(o[k]) * f * f2, bfhi(o[k]) * f * f2);
                                pp_st8(sh + j, o);
                            }
                            if (!ok) break;
                        }
                        fresh = fresh && bt == 0;
                        l += sum;
                        pp_st16(sh + c / 2, p);
                    }
                } else {
                    const uint32_t zero[32] = {};
                    pp_st32(sh, zero);
                }
                if (!ok) break;
                pp_st_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (pp_elect()) tc::mbar_arrive(&p_bar[buf]);
                if (h == 1) {
                    if (lane == 0) tc::mbar_arrive(&sc_empty[st]);
                    ++bc;
                }
            }
            if (!ok) break;
            // the last products: one more round of each barrier
            round += steps / C::NB;
            for (int b = 0; b < C::NB; ++b) ok = ok && pp_wait(&s_bar[b], round & 1, w.err, 63);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++round;
            tc::tc_fence_after();
            const bool live = m_row < g.mrows && pos >= 0;
            if (g.piece < 0) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint16_t *out = a.ctx + (g.row0 + (uint64_t)row_i) * a.ctx_stride +
                                (uint64_t)(g.kvh * w.group + m_row % w.group) * DIM;
#pragma unroll 1
                for (int j = 0; j < DIM; j += 16) {
                    uint32_t o[16];
                    pp_ld16(o_addr + j, o);
                    pp_ld_wait();
                    if (live) {
#pragma unroll
                        for (int k = 0; k < 16; k += 8) {
                            uint4 v;
                            v.x = pp_pack(__uint_as_float(o[k]) * inv, __uint_as_float(o[k + 1]) * inv);
                            v.y = pp_pack(__uint_as_float(o[k + 2]) * inv, __uint_as_float(o[k + 3]) * inv);
                            v.z = pp_pack(__uint_as_float(o[k + 4]) * inv, __uint_as_float(o[k + 5]) * inv);
                            v.w = pp_pack(__uint_as_float(o[k + 6]) * inv, __uint_as_float(o[k + 7]) * inv);
                            if (l == 0.f) v = make_uint4(0, 0, 0, 0);
                            *reinterpret_cast<uint4 *>(out + j + k) = v;
                        }
                    }
                }
            } else {
                float *piece = w.pieces + (uint64_t)g.piece * C::PIECE;
                const int t = 128 * x + r;
                piece[t] = l == 0.f ? -INFINITY : m;
                piece[C::TILE + t] = l;
                float *po = piece + 2 * C::TILE + (uint64_t)t * DIM;
#pragma unroll 1
                for (int j = 0; j < DIM; j += 16) {
                    uint32_t o[16];
                    pp_ld16(o_addr + j, o);
                    pp_ld_wait();
#pragma unroll
                    for (int k = 0; k < 16; k += 4)
                        *reinterpret_cast<uint4 *>(po + j + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
            }
            tc::tc_fence_before();
        }
    } else if (warp < C::SW + 4) {
        // ---------------- tile warps: warp lw has keys 32 lw .. of each block
        if constexpr (DIM == 64)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        else
            asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const int lw = warp - C::SW;
        constexpr int CPR = DIM / 8;  // 16-byte chunks of a bf16 row
        PpReader rd{ring, seg_full, seg_empty};
        uint32_t bc = 0, nseg = 0, tiles = 0;  // blocks; segments; K and V tiles
        PpSeg g;
        while (ok) {
            ok = rd.next(g, w.err);
            if (!ok || g.nblk == 0) break;
            const uint32_t *table = a.c.table + (uint64_t)g.seq * a.c.max_pages;
            // lane = key: its page two blocks ahead, its pool row and scales one ahead
            auto key_of = [&](int i) {
                const int vb = g.b0 + i;
                return (vb < g.s128 ? vb : vb - g.s128 + g.low128) * PP_BLK + 32 * lw + lane;
            };
            auto page_of = [&](int i) {
                const int key = key_of(i);
                return i < g.nblk && key <= g.last && (key >= g.low || key < g.first) ? __ldg(&table[key >> a.c.tshift])
                                                                                       : PG_NO_PAGE;
            };
            uint32_t bits = 0;
            float ksc = 0.f, vsc = 0.f;
            auto scales_of = [&](int i, uint32_t page) {
                const bool vis = page < a.c.pages;
                bits = __ballot_sync(0xffffffffu, vis);
                ksc = vsc = 0.f;
                if (KV8 && vis) {
                    const uint64_t row = paged_row(a.c, page, g.kvh) + (key_of(i) & ((1 << a.c.tshift) - 1));
                    ksc = __ldg(a.c.ks + row);
                    vsc = __ldg(a.c.vs + row);
                }
            };
            scales_of(0, page_of(0));
            uint32_t page = page_of(1);
            for (int i = 0; i < g.nblk && ok; ++i, ++bc) {
                // scales and the mask of keys that are there
                const uint32_t st = bc % PP_SC;
                if (bc >= PP_SC)
                    ok = __all_sync(0xffffffffu, pp_wait(&sc_empty[st], ((bc / PP_SC) & 1) ^ 1, w.err, 65));
                if (!ok) break;
                if constexpr (KV8) {
                    scales[st * 256 + 32 * lw + lane] = w.negate ? -ksc * w.fac : ksc * w.fac;
                    scales[st * 256 + 128 + 32 * lw + lane] = vsc;
                }
                const uint32_t now = bits;
                if (lane == 0) masks[4 * st + lw] = now;
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sc_full[st]);
                scales_of(i + 1, page);
                page = page_of(i + 2);
                if (i == 0) {
                    // queries: flattened row m of the tile is token m / group, head m % group of this KV
                    // head; lane = row, its address handed to the lanes that copy it (rows of whole lines)
                    const uint32_t qb = nseg % C::QBUFS, use = nseg / C::QBUFS;
                    if (use > 0) ok = __all_sync(0xffffffffu, pp_wait(&q_empty[qb], (use - 1) & 1, w.err, 64));
                    if (!ok) break;
                    ++nseg;
#pragma unroll 1
                    for (int x = 0; x < C::TILES; ++x) {
                        if (g.m0 + 128 * x >= g.mrows) break;
                        const uint32_t mr = g.m0 + 128 * x + 32 * lw + lane, token = mr / w.group;
                        const bool live = mr < g.mrows;
                        const uint64_t mine = live ? (g.row0 + (uint64_t)token) * a.q_stride +
                                                         (uint64_t)(g.kvh * w.group + mr - token * w.group) * DIM
                                                   : 0;
                        const uint32_t lives = __ballot_sync(0xffffffffu, live);
                        const uint32_t dst = sbase + C::Q + (qb * C::TILES + x) * C::TILE_BYTES;
#pragma unroll 4
                        for (int j = 0; j < CPR; ++j) {
                            const int n = j * 32 + lane, rl = n / CPR, c = n % CPR;
                            const uint64_t src = __shfl_sync(0xffffffffu, mine, rl);
                            pp_cp16(dst + pp_off(32 * lw + rl, c), a.q + src + 8 * c, lives >> rl & 1 ? 16 : 0);
                        }
                    }
                    pp_cp_commit();
                    pp_cp_wait<0>();
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&q_full[qb]);
                }
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv, ++tiles) {
                    const uint32_t slot = tiles % C::SLOTS, dst = sbase + C::RING + slot * C::TILE_BYTES;
                    if constexpr (KV8) {
                        // codes -> bf16, exactly; a code that is not visible is some code, and its
                        // scale and weight are 0
                        const uint32_t rs = tiles % C::RAW;
                        ok = pp_wait(&raw_full[rs], (tiles / C::RAW) & 1, w.err, 58) &&
                             (tiles < C::SLOTS || pp_wait(&kv_empty[slot], ((tiles / C::SLOTS) & 1) ^ 1, w.err, 66));
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        constexpr int NL = DIM / 16;
                        const uint32_t src = sbase + C::CODES + rs * C::RAW_BYTES + 32 * lw * DIM;
#pragma unroll
                        for (int j = 0; j < NL; ++j) {
                            const int n = j * 32 + lane, r = 32 * lw + n / NL, c = n % NL;
                            uint32_t wd[4], o[8];
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(wd[0]), "=r"(wd[1]), "=r"(wd[2]), "=r"(wd[3])
                                         : "r"(src + n * 16));
#pragma unroll
                            for (int k = 0; k < 4; ++k) {  // bytes (0, 1) and (2, 3) of each word as bf16 pairs
                                const uint32_t lo = __byte_perm(wd[k], 0, 0x4140), hi = __byte_perm(wd[k], 0, 0x4342);
                                o[2 * k] = bf16x2_sub(lop_or(lo, 0x007F007Fu, 0x43004300u), lop_or(lo, 0x00800080u, 0x43004300u));
                                o[2 * k + 1] = bf16x2_sub(lop_or(hi, 0x007F007Fu, 0x43004300u), lop_or(hi, 0x00800080u, 0x43004300u));
                            }
                            pp_sts128(dst + pp_off(r, 2 * c), o[0], o[1], o[2], o[3]);
                            pp_sts128(dst + pp_off(r, 2 * c + 1), o[4], o[5], o[6], o[7]);
                        }
                        tc::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tc::mbar_arrive(&kv_full[slot]);
                            tc::mbar_arrive(&raw_empty[rs]);
                        }
                    } else if (kv == 1) {
                        // values that are not visible become 0 (a weight of 0 times NaN would not be)
                        const uint32_t vt = tiles / 2, rs = vt % C::RAW;
                        ok = __all_sync(0xffffffffu, pp_wait(&raw_full[rs], (vt / C::RAW) & 1, w.err, 58));
                        if (!ok) break;
                        if (now != 0xffffffffu) {
                            if (!(now >> lane & 1))
                                for (int c = 0; c < CPR; ++c) pp_sts128(dst + pp_off(32 * lw + lane, c), 0, 0, 0, 0);
                            tc::fence_proxy_async_smem();
                        }
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&kv_full[slot]);
                    }
                }
            }
        }
    } else {
        if constexpr (DIM == 64)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        else
            asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp < C::SW + 6) {
            // ---------------- MMA issuers: tiles `who`, who + 2
            const int who = warp - (C::SW + 4);
            PpReader rd{ring, seg_full, seg_empty};
            uint32_t bc = 0, nseg = 0, round[C::TILES / 2] = {};  // rounds of the tiles' barriers before the segment
            const uint32_t id_qk = pp_idesc(64, false) | (!KV8 && w.negate ? 1u << 13 : 0u);
            constexpr uint32_t id_pv = pp_idesc(DIM, true);
            const uint64_t q_desc = tc::smem_desc_sw128(sbase + C::Q), k_desc = tc::smem_desc_sw128(sbase + C::RING),
                           v_desc = pp_desc_mn(sbase + C::RING);
            PpSeg g;
            while (ok) {
                ok = rd.next(g, w.err);
                if (!ok || g.nblk == 0) break;
                const int all_tiles = (int)min((g.mrows - g.m0 + 127) / 128, (uint32_t)C::TILES);
                const int tiles = (all_tiles + 1 - who) / 2, steps = 2 * g.nblk;  // this issuer's
                if (pp_elect()) {
                    auto wait_tile = [&](uint32_t n) {
                        return pp_wait(&kv_full[n % C::SLOTS], (n / C::SLOTS) & 1, w.err, 67);
                    };
                    // step n: the weights' product of step n - NB, then the scores of step n over its
                    // columns; descriptors differ in their address field only
                    const uint32_t qb = nseg % C::QBUFS;
                    ok = pp_wait(&q_full[qb], (nseg / C::QBUFS) & 1, w.err, 68);
                    for (int n = 0; n < steps + C::NB && ok; ++n) {
                        const int pn = n - C::NB, h = n & 1, ph = pn & 1;
                        const bool scores = n < steps, product = pn >= 0;
                        const uint32_t kt = 2 * (bc + n / 2), vt = 2 * (bc + pn / 2) + 1;
                        if (scores && h == 0) ok = wait_tile(kt);
                        if (ok && product && ph == 0) ok = wait_tile(vt);
                        const uint32_t buf = n % C::NB;
#pragma unroll
                        for (int t = 0; t < C::TILES / 2; ++t) {
                            if (t >= tiles || !ok) break;
                            const int x = 2 * t + who;
                            const uint32_t sc = tmem + 64 * (x * C::NB + buf);
                            if (product) ok = pp_wait(&p_ready[x * C::NB + buf], (round[t] + pn / C::NB) & 1, w.err, 69);
                            if (!ok) break;
                            tc::tc_fence_after();
                            if (product) {
                                const uint64_t vd = v_desc + (((vt % C::SLOTS) * C::TILE_BYTES + ph * 8192) >> 4);
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    pp_mma_ts(tmem + 256 + x * DIM, sc + 8 * j, vd + j * (2048 >> 4), id_pv, pn > 0 || j > 0);
                            }
                            if (scores) {
                                const uint64_t qd = q_desc + (((qb * C::TILES + x) * C::TILE_BYTES) >> 4),
                                               kd = k_desc + (((kt % C::SLOTS) * C::TILE_BYTES + h * 8192) >> 4);
#pragma unroll
                                for (int j = 0; j < DIM / 16; ++j) {
                                    const uint32_t off = ((j >> 2) * (128 * 128) + (j & 3) * 32) >> 4;
                                    pp_mma_ss(sc, qd + off, kd + off, id_qk, j > 0);
                                }
                            }
                            tc::mma_commit(&s_full[x * C::NB + buf]);
                        }
                        // an issuer without a tile here only lets the slots go (its commit follows nothing)
                        if (ok && product && ph == 1) tc::mma_commit(&kv_empty[vt % C::SLOTS]);
                        if (ok && scores && h == 1) {
                            tc::mma_commit(&kv_empty[kt % C::SLOTS]);
                            if (n + 1 == steps) tc::mma_commit(&q_empty[qb]);
                        }
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                bc += g.nblk;
#pragma unroll
                for (int t = 0; t < C::TILES / 2; ++t)
                    if (t < tiles) round[t] += steps / C::NB;
                ++nseg;
            }
            // every MMA is complete before TMEM is freed (the commit is the thread's that issued them)
            if (pp_elect()) {
                tc::mma_commit(mdone);
                pp_wait(mdone, 0, w.err, 69);
            }
            __syncwarp();
        } else if (warp == C::SW + 7) {
            // ---------------- copies: lane p has page p of a block (its first 128 tokens' worth
            // of it); KV8 pages as runs of codes, bf16 pages as swizzled boxes
            PpReader rd{ring, seg_full, seg_empty};
            const int per = min(1 << a.c.tshift, PP_BLK), npages = PP_BLK / per;  // tokens of a copy, copies of a block
            constexpr uint32_t RB = KV8 ? DIM : 2 * DIM, RING = KV8 ? C::RAW : C::SLOTS;
            uint32_t tiles = 0;
            auto full_of = [&](uint32_t t) {  // what the copies of tile t (K and V in turn) complete on
                return KV8 ? &raw_full[t % C::RAW] : t & 1 ? &raw_full[t / 2 % C::RAW] : &kv_full[t % C::SLOTS];
            };
            PpSeg g;
            while (ok) {
                ok = rd.next(g, w.err);
                if (!ok || g.nblk == 0) break;
                const uint32_t *table = a.c.table + (uint64_t)g.seq * a.c.max_pages;
                auto page_of = [&](int i) {
                    const int vb = g.b0 + i, key = (vb < g.s128 ? vb : vb - g.s128 + g.low128) * PP_BLK + lane * per;
                    const bool some = i < g.nblk && lane < npages && key <= g.last && (key + per > g.low || key < g.first);
                    return some ? __ldg(&table[key >> a.c.tshift]) : PG_NO_PAGE;
                };
                uint32_t next = page_of(0);
                for (int i = 0; i < g.nblk && ok; ++i) {
                    const uint32_t page = next;
                    next = page_of(i + 1);
                    const int vb = g.b0 + i, key = (vb < g.s128 ? vb : vb - g.s128 + g.low128) * PP_BLK + lane * per;
                    const bool have = page < a.c.pages;
                    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, have)) * per * RB;
                    const int row = ((int)g.kvh << a.c.tshift) + (key & ((1 << a.c.tshift) - 1));  // within the page
#pragma unroll 1
                    for (int kv = 0; kv < 2; ++kv, ++tiles) {
                        uint64_t *bar = full_of(tiles);
                        const uint32_t slot = tiles % RING;
                        if (tiles >= RING)
                            ok = pp_wait(KV8 ? &raw_empty[slot] : &kv_empty[slot], ((tiles / RING) & 1) ^ 1, w.err, 57);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) tc::mbar_arrive_expect_tx(bar, bytes);
                        __syncwarp();
                        if (have) {
                            if constexpr (KV8) {
                                const uint8_t *src = (kv ? a.c.v : a.c.k) + ((uint64_t)page * a.c.page_rows + row) * RB;
                                tc::bulk_load(sm + C::CODES + slot * C::RAW_BYTES + lane * per * RB, src, per * RB, bar);
                            } else {
#pragma unroll
                                for (int h = 0; h < C::HALVES; ++h)
                                    pp_tma_3d(sm + C::RING + slot * C::TILE_BYTES + h * (128 * 128) + lane * per * 128,
                                              kv ? &maps.v : &maps.k, bar, 64 * h, row, (int)page);
                            }
                        }
                    }
                }
            }
            // No copy is in flight when the CTA ends, also where a wait ran out and nobody waits for the last ones.
            for (uint32_t t = tiles > RING ? tiles - RING : 0; t < tiles; ++t) pp_wait(full_of(t), (t / RING) & 1, w.err, 57);
        } else if (warp == C::SW + 6) {
            // ---------------- segments
            uint32_t n = 0;
            uint32_t i = at_seq;
            unsigned long long u = u0, base = at_prefix * a.c.hkv;  // units before sequence i
            bool first_segment = true;
            if (lane == 0) w.recs[blockIdx.x].valid = 0;
            while (ok) {
                const uint32_t d = n % PP_SEG;
                PpSeg g = {};
                if (u < u1) {
                    const PpSeqInfo s = pp_seq(a, w, i);
                    const uint32_t units = pp_units_warp(a, w, s.pos0, s.mrows, s.nt);
                    if (units == 0 || u >= base + (unsigned long long)units * a.c.hkv) {
                        base += (unsigned long long)units * a.c.hkv;
                        ++i;
                        continue;
                    }
                    unsigned long long kvh64, off64;
                    div64(u - base, units, kvh64, off64);
                    const uint32_t kvh = (uint32_t)kvh64, off = (uint32_t)off64;
                    // the tile that holds unit `off` of this KV head
                    uint32_t seen = 0;
                    int k = 0, b0 = 0;
                    PpBlocks bl = {};
                    for (int kb = 0;; kb += 32) {
                        const PpBlocks mine_b = pp_blocks(a, w, s.pos0, s.mrows, min(kb + lane, s.nt - 1));
                        const uint32_t cnt = kb + lane < s.nt ? mine_b.n : 0;
                        uint32_t xs = cnt;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const uint32_t y = __shfl_up_sync(0xffffffffu, xs, o);
                            if (lane >= o) xs += y;
                        }
                        const uint32_t hit = __ballot_sync(0xffffffffu, seen + xs > off);
                        if (hit || kb + 32 >= s.nt) {
                            const int l = hit ? __ffs(hit) - 1 : 31;
                            k = kb + l;
                            b0 = (int)(off - (seen + __shfl_sync(0xffffffffu, xs - cnt, l)));
                            break;
                        }
                        seen += __shfl_sync(0xffffffffu, xs, 31);
                    }
                    // this tile and those behind it in the KV head: one segment each
                    bool more = true;
                    while (more && ok) {
                        bl = pp_blocks(a, w, s.pos0, s.mrows, k);
                        const int cnt = (int)min((unsigned long long)(bl.n - b0), u1 - u);
                        if (cnt > 0) {
                            g.seq = s.seq;
                            g.row0 = s.row0;
                            g.m0 = (uint32_t)k * C::TILE;
                            g.mrows = s.mrows;
                            g.pos0 = s.pos0;
                            g.kvh = kvh;
                            g.b0 = b0;
                            g.nblk = cnt;
                            g.s128 = bl.s128;
                            g.low128 = bl.low128;
                            g.first = bl.first;
                            g.low = bl.low;
                            g.last = bl.last;
                            g.piece = cnt == bl.n ? -1 : (int)(2 * blockIdx.x + (first_segment ? 0 : 1));
                            const uint32_t dd = n % PP_SEG;
                            if (n >= PP_SEG)
                                ok = __all_sync(0xffffffffu, pp_wait(&seg_empty[dd], ((n / PP_SEG) & 1) ^ 1, w.err, 60));
                            if (!ok) break;
                            if (lane == 0) {
                                ring[dd] = g;
                                tc::mbar_arrive(&seg_full[dd]);
                            }
                            __syncwarp();
                            ++n;
                            if (first_segment && b0 > 0 && lane == 0) {
                                PpRec rec = {};
                                const unsigned long long t0 = u - b0;
                                rec.valid = 1;
                                rec.row0 = s.row0;
                                rec.m0 = g.m0;
                                rec.mrows = s.mrows;
                                rec.kvh = kvh;
                                rec.pos0 = s.pos0;
                                rec.c0 = split.cta_of(t0);
                                rec.c1 = split.cta_of(t0 + bl.n - 1);
                                rec.slot0 = split.start(rec.c0) < t0;
                                w.recs[blockIdx.x] = rec;
                            }
                            first_segment = false;
                            u += cnt;
                        }
                        ++k;
                        b0 = 0;
                        more = u < u1 && k < s.nt;
                    }
                    continue;
                }
                if (n >= PP_SEG) ok = __all_sync(0xffffffffu, pp_wait(&seg_empty[d], ((n / PP_SEG) & 1) ^ 1, w.err, 60));
                if (ok && lane == 0) {
                    ring[d] = g;  // nblk 0: the end
                    tc::mbar_arrive(&seg_full[d]);
                }
                break;
            }
        }
    }
    if (warp == C::SW + 6) {  // (behind its segments)
        // ---------------- rows in front of the first token, and of no sequence
        const uint32_t chunks = a.qh * (DIM / 8);
        auto zero = [&](uint32_t row0, uint32_t n, uint32_t r0, uint32_t step) {
            for (uint32_t r = r0; r < n; r += step)
                for (uint32_t c = lane; c < chunks; c += 32)
                    *reinterpret_cast<uint4 *>(a.ctx + (row0 + (uint64_t)r) * a.ctx_stride + 8 * c) = make_uint4(0, 0, 0, 0);
        };
        for (uint32_t i = blockIdx.x; i < a.n; i += gridDim.x) {
            const PpSeqInfo s = pp_seq(a, w, i);
            if (pp_dead(s) <= pp_dead_alone(a)) zero(s.row0, pp_dead(s), 0, 1);
        }
        // the runs of sequences in which the numbering met more rows (padded prompts)
        for (uint32_t runs = __ballot_sync(0xffffffffu, lane < C::WARPS && wdead[lane]); runs; runs &= runs - 1) {
            for (uint32_t b = min((__ffs(runs) - 1) * per, a.n), e = min(b + per, a.n); b < e; b += 32) {
                const PpSeqInfo s = pp_seq(a, w, min(b + lane, e - 1));
                const uint32_t n = b + lane < e ? pp_dead(s) : 0;
                for (uint32_t todo = __ballot_sync(0xffffffffu, n > pp_dead_alone(a)); todo; todo &= todo - 1) {
                    const int l = __ffs(todo) - 1;
                    zero(__shfl_sync(0xffffffffu, s.row0, l), __shfl_sync(0xffffffffu, n, l), (blockIdx.x + b + l) % gridDim.x,
                         gridDim.x);
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == C::SW + 4) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
}

// Tiles that several CTAs share. Block (c, y): 32 rows of the tile in whose
// middle CTA c starts, if c is the tile's second CTA; 8 threads per row.
template <int DIM>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(PagedAttnArgs a, PpWork w) {
    constexpr int TILE = PpCfg<false, DIM>::TILE, PIECE = 2 * TILE + TILE * DIM, PER = DIM / 8;
    pdl_wait();
    const PpRec rec = w.recs[blockIdx.x];
    if (!rec.valid || rec.c0 + 1 != blockIdx.x) return;
    const uint32_t t = blockIdx.y * 32 + threadIdx.x / 8, d0 = (threadIdx.x % 8) * PER, m = rec.m0 + t;
    if (m >= rec.mrows || rec.pos0 + (int)(m / w.group) < 0) return;
    const uint32_t n = rec.c1 - rec.c0 + 1;
    auto piece = [&](uint32_t i) { return w.pieces + ((uint64_t)(rec.c0 + i) * 2 + (i == 0 ? rec.slot0 : 0)) * PIECE; };
    float M = -INFINITY, L = 0.f, O[PER];
    for (uint32_t i = 0; i < n; ++i) M = fmaxf(M, piece(i)[t]);
    const float M0 = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int j = 0; j < PER; ++j) O[j] = 0.f;
#pragma unroll 2
    for (uint32_t i = 0; i < n; ++i) {
        const float *p = piece(i);
        const float f = pp_ex2(0.5f * (p[t] - M0));  // applied twice: 2^(m - M) itself may underflow where o f does not
        L += p[TILE + t] * f * f;
        const float4 *o = reinterpret_cast<const float4 *>(p + 2 * TILE + (uint64_t)t * DIM + d0);
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) {
            const float4 v = o[j];
            O[4 * j] += v.x * f * f;
            O[4 * j + 1] += v.y * f * f;
            O[4 * j + 2] += v.z * f * f;
            O[4 * j + 3] += v.w * f * f;
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint16_t *out = a.ctx + (rec.row0 + (uint64_t)(m / w.group)) * a.ctx_stride +
                    (uint64_t)(rec.kvh * w.group + m % w.group) * DIM + d0;
#pragma unroll
    for (int j = 0; j < PER; j += 8) {
        uint4 v = make_uint4(pp_pack(O[j] * inv, O[j + 1] * inv), pp_pack(O[j + 2] * inv, O[j + 3] * inv),
                             pp_pack(O[j + 4] * inv, O[j + 5] * inv), pp_pack(O[j + 6] * inv, O[j + 7] * inv));
        if (L == 0.f) v = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4 *>(out + j) = v;
    }
}

// The same for few tiles of many pieces each: a thread takes four dims, so that
// more blocks share a tile, and four pieces' loads are in flight; the factors are
// formed first, by the row's threads together.
template <int DIM>
struct PjCfg {
    static constexpr int PER_ROW = DIM / 4, THREADS = 256, ROWS = THREADS / PER_ROW;
};
template <int DIM>
__global__ void __launch_bounds__(PjCfg<DIM>::THREADS) paged_prefill_join_few_kernel(PagedAttnArgs a, PpWork w) {
    constexpr int TILE = PpCfg<false, DIM>::TILE, PIECE = 2 * TILE + TILE * DIM, T = PjCfg<DIM>::PER_ROW;
    constexpr uint32_t BATCH = 4;
    __shared__ float fs[PjCfg<DIM>::ROWS][PP_MAX_SMS];
    pdl_wait();
    const PpRec rec = w.recs[blockIdx.x];
    if (!rec.valid || rec.c0 + 1 != blockIdx.x) return;
    const uint32_t r = threadIdx.x / T, j = threadIdx.x % T, t = blockIdx.y * PjCfg<DIM>::ROWS + r, m = rec.m0 + t;
    const bool live = m < rec.mrows && rec.pos0 + (int)(m / w.group) >= 0;
    const uint32_t n = live ? rec.c1 - rec.c0 + 1 : 0;
    auto piece = [&](uint32_t i) { return w.pieces + ((uint64_t)(rec.c0 + i) * 2 + (i == 0 ? rec.slot0 : 0)) * PIECE; };
    float M = -INFINITY, L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t i = j; i < n; i += T) {
        fs[r][i] = piece(i)[t];
        M = fmaxf(M, fs[r][i]);
    }
#pragma unroll
    for (int o = T / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float M0 = M == -INFINITY ? 0.f : M;
    for (uint32_t i = j; i < n; i += T) {
        const float f = pp_ex2(0.5f * (fs[r][i] - M0));  // applied twice, as above
        fs[r][i] = f;
        L += piece(i)[TILE + t] * f * f;
    }
#pragma unroll
    for (int o = T / 2; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    __syncwarp();
    for (uint32_t i0 = 0; i0 < n; i0 += BATCH) {
        float4 v[BATCH];
#pragma unroll
        for (uint32_t k = 0; k < BATCH; ++k)
            v[k] = i0 + k < n ? __ldcg(reinterpret_cast<const float4 *>(piece(i0 + k) + 2 * TILE + (uint64_t)t * DIM) + j)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t k = 0; k < BATCH; ++k) {
            if (i0 + k >= n) break;
            const float f = fs[r][i0 + k];
            O[0] += v[k].x * f * f;
            O[1] += v[k].y * f * f;
            O[2] += v[k].z * f * f;
            O[3] += v[k].w * f * f;
        }
    }
    if (!live) return;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint2 out = make_uint2(pp_pack(O[0] * inv, O[1] * inv), pp_pack(O[2] * inv, O[3] * inv));
    if (L == 0.f) out = make_uint2(0, 0);
    *reinterpret_cast<uint2 *>(a.ctx + (rec.row0 + (uint64_t)(m / w.group)) * a.ctx_stride +
                               (uint64_t)(rec.kvh * w.group + m % w.group) * DIM + 4 * j) = out;
}

size_t paged_prefill_ws(uint32_t, uint32_t, uint32_t dim, uint32_t, uint32_t) {
    const size_t tile = dim == 64 ? PpCfg<false, 64>::TILE : PpCfg<false, 128>::TILE;
    return 256 + (size_t)PP_MAX_SMS * (sizeof(PpRec) + 2 * (2 * tile + tile * dim) * 4);
}

// From what the host knows: the tiles that the rows can be cut into, times the
// blocks that a tile can see in the widest table row, or in its window (that of
// all its tokens, cut at both ends) and the first tokens.
bool paged_prefill_fits(const PagedAttnArgs &a) {
    const uint64_t tile = a.dim == 64 ? PpCfg<false, 64>::TILE : PpCfg<false, 128>::TILE, group = a.qh / a.c.hkv;
    const uint64_t tiles = a.rows * group / tile + a.n;
    uint64_t blocks = (((uint64_t)a.c.max_pages << a.c.tshift) + PP_BLK - 1) / PP_BLK;
    if (a.window) {
        const uint64_t seen = (a.window + tile / group + 1) / PP_BLK + 2 + ((uint64_t)a.sinks + PP_BLK - 1) / PP_BLK;
        blocks = blocks < seen ? blocks : seen;
    }
    return tiles * blocks < 1ull << 32;
}

template <bool KV8, int DIM>
static int launch_prefill(const PagedAttnArgs &a, const PpWork &w, cudaStream_t st) {
    using C = PpCfg<KV8, DIM>;
    auto *kernel = paged_prefill_kernel<KV8, DIM>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::ALLOC) != cudaSuccess) return -3;
    PpMaps maps = {};
    if (!KV8) {
        const uint64_t rows = (uint64_t)a.c.hkv << a.c.tshift, stride = (a.c.page_rows > rows ? a.c.page_rows : rows) * DIM * 2;
        const int box = a.c.tshift < 7 ? 1 << a.c.tshift : PP_BLK;
        if (int rc = make_page_map(&maps.k, a.c.k, DIM, rows, a.c.pages, stride, box)) return rc;
        if (int rc = make_page_map(&maps.v, a.c.v, DIM, rows, a.c.pages, stride, box)) return rc;
    }
    PdlChain chain;
    if (int rc = launch_pdl(kernel, dim3(w.max_ctas), dim3(C::THREADS), C::ALLOC, st, 1, maps, a, w)) return rc;
    // Few tiles are in many pieces: first way against second, 14 heads on 2 of 64 dims KV8, 128 rows on 4000 keys 35.1
    // and 41.7 us, 8 x 64 rows on 2000 keys 37.2 and 39.2, 16 x 64 47.7 and 47.2, 32 x 64 70.0 and 67.5; 32 heads on 8
    // of 128 dims bf16, 4 x 32 rows on 8000 keys 41.7 and 45.6.
    const uint64_t flat = (uint64_t)a.rows * w.group, tiles = a.c.hkv * (flat / C::TILE + a.n);
    if (3 * tiles <= w.max_ctas) {
        using J = PjCfg<DIM>;
        const unsigned groups = (unsigned)(((flat < C::TILE ? flat : C::TILE) + J::ROWS - 1) / J::ROWS);
        return launch_pdl(paged_prefill_join_few_kernel<DIM>, dim3(w.max_ctas, groups), dim3(J::THREADS), 0, st, 1, a, w);
    }
    return launch_pdl(paged_prefill_join_kernel<DIM>, dim3(w.max_ctas, C::TILE / 32), dim3(256), 0, st, 1, a, w);
}

int launch_paged_prefill(const PagedAttnArgs &a, void *ws, cudaStream_t st) {
    const int sms = paged_sms();
    if (sms <= 0) return -3;
    PpWork w;
    w.group = a.qh / a.c.hkv;
    w.max_ctas = (uint32_t)(sms < PP_MAX_SMS ? sms : PP_MAX_SMS);
    w.tile = a.dim == 64 ? PpCfg<false, 64>::TILE : PpCfg<false, 128>::TILE;
    w.negate = a.scale < 0.f;
    w.fac = fabsf(a.scale) * 1.44269504f;
    w.err = (unsigned *)ws;
    w.recs = reinterpret_cast<PpRec *>((char *)ws + 256);
    w.pieces = reinterpret_cast<float *>((char *)ws + 256 + PP_MAX_SMS * sizeof(PpRec));
    if (a.format == QWEN_B200_KV8)
        return a.dim == 64 ? launch_prefill<true, 64>(a, w, st) : launch_prefill<true, 128>(a, w, st);
    return a.dim == 64 ? launch_prefill<false, 64>(a, w, st) : launch_prefill<false, 128>(a, w, st);
}

}  // namespace qb
