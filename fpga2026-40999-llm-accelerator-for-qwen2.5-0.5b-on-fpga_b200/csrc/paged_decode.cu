// Decode attention over the paged KV cache: one query token per sequence, the
// context split evenly over the GPU and joined.
//
// Mathematics, per (row, query head), over the visible keys j:
//   x_j = log2(e) scale q.k_j,  p_j = 2^(x_j - m),  ctx = sum p_j v_j / sum p_j
// with a running maximum m that is only raised when some x_j passes m + 8 (p
// stays below 2^8, so nothing overflows and the rescaling is rare), sums in
// fp32. KV8: the key's scale multiplies its score and the value's scale its
// weight, so both products run on the codes.
//
// Work: an item is a row with a block of up to 8 query heads that share a KV
// head. Usually one CTA, or a cluster of up to 16 that split the context evenly
// and join over distributed shared memory, takes an item: one launch, nothing
// in the workspace. Where that would leave the GPU idle (few items, long
// contexts), steps of 16 or 32 keys of all items are numbered in a row and CTA c
// of G takes the c-th equal run (every CTA derives the numbering from the
// lengths, so the launch does not depend on them and can be captured); a run
// that covers an item alone writes ctx, pieces go to the workspace (at most two
// per CTA) and a join kernel, launched behind with programmatic serialisation,
// adds them in CTA order.
//
// Measured: one row over 32768 keys of 8 heads x 128 bf16 28.8 us (4.66 TB/s, 71 %
// of the copy rate), 64 rows over 2048 keys of 2 heads x 64 KV8 14.7 us (2.4 TB/s:
// instruction issue and the start's chain of length, page and key), one row over
// 96 keys 6.3 us (that chain alone).
//
// 8 query heads share each key that is read; a KV head of more is read once for
// each block of 8. Keys are copied to shared memory by 16-byte cp.async, every warp with
// a ring of its own, so no barrier stands between the loads and the products. Both products
// are mma.sync m16n8k16 with the keys (then the dims) as the 16-row side and the
// heads as the 8-column side: a row has up to 8 useful columns, where a
// 128-row tcgen05 tile would be 6 % full, and per byte of cache these
// instructions need less than half of the issue slots. S^T = K Q^T: int8 codes
// become fp16 exactly (1024 + 128 + c minus 1152), q is scaled by a power of
// two into fp16 range (bf16 values fit its 11 bits); bf16 keys are used as they
// are. O^T = V^T P^T: weights as two bf16 halves (hi + lo, 16 bits together, and
// bf16's range for any value scale), V^T fragments by byte permutes from the
// row-major rows.
#include "paged.cuh"
#include "tc05.cuh"

namespace qb {

constexpr int PD_WARPS = 8, PD_THREADS = 32 * PD_WARPS, PD_SUB = 16, PD_HEADS = 8;
constexpr uint32_t PD_MAX_PARTS = 16;  // CTAs of a cluster
constexpr int PD_MAX_SMS = 192;  // sizes the workspace whatever the device
constexpr uint32_t PD_PART_KEYS = 512;  // keys that a CTA of a cluster has at least to be worth its join
constexpr uint32_t PD_PART_MOST = 2048; // and at most where the clusters leave most of the GPU idle
constexpr uint32_t PD_MIN_UNITS = 8;  // steps that a CTA takes at least (1 per warp)

template <bool KV8, int DIM>
struct PdCfg {
    static constexpr int RB = KV8 ? DIM : 2 * DIM;  // bytes of a row
    static constexpr int CPR = RB / 16;             // 16-byte chunks of a row
    static constexpr int SUBS = RB == 64 ? 2 : 1, STEP = SUBS * PD_SUB;  // 16-key pieces of a step; its keys
    static constexpr int LOG = STEP == 32 ? 5 : 4;
    static constexpr int SUB_BYTES = 2 * PD_SUB * RB + (KV8 ? 2 * PD_SUB * 4 : 0), STEP_BYTES = SUBS * SUB_BYTES;
    static constexpr int STAGES = 3;
    static constexpr int MINB = RB == 256 ? 1 : 2;  // CTAs per SM
    static constexpr int RING = PD_WARPS * STAGES * STEP_BYTES;
    static constexpr int OUT = PD_WARPS * PD_HEADS * (DIM + 1) * 4;  // the warps' contexts, over the drained ring
    static constexpr int SMEM = RING > OUT ? RING : OUT;
    static constexpr int PIECE = 2 * PD_HEADS + PD_HEADS * DIM;  // floats of a partial result: m, l, o
};

struct PdWork {
    uint32_t group, hb;   // query heads per KV head, blocks of 8 of them
    uint32_t items;       // (KV head, block) pairs of a row
    uint32_t parts;       // CTAs of a cluster (one launch)
    uint32_t max_ctas;
    uint32_t *prefix;     // [rows + 1] units of one item in the rows before
    float *pieces;        // [CTA][2][PIECE]
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ float lds32f(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four codes (bytes of w) as two fp16 pairs, exactly.
__device__ __forceinline__ void codes4_to_f16(uint32_t w, uint32_t &k01, uint32_t &k23) {
    const uint32_t u = w ^ 0x80808080u;  // c + 128
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(k01) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(k23) : "r"(b), "r"(0x64806480u));
}
// Byte i of wa and of wb as a bf16 pair, exactly (see codes4_to_bf16).
template <int I>
__device__ __forceinline__ uint32_t codes_pair_bf16(uint32_t wa, uint32_t wb) {
    const uint32_t t = __byte_perm(wa, wb, ((4 + I) << 8) | I);
    return bf16x2_sub(lop_or(t, 0x007F007Fu, 0x43004300u), lop_or(t, 0x00800080u, 0x43004300u));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// v to the word at this address of CTA `rank`'s shared memory.
__device__ __forceinline__ void pd_dsmem_store(uint32_t local_saddr, uint32_t rank, float v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_saddr), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}
// Heads that a CTA of a cluster joins at most (CTA c those with h % parts == c).
__device__ __forceinline__ uint32_t pd_heads_here(uint32_t parts) { return (PD_HEADS + parts - 1) / parts; }
__device__ __forceinline__ void pd_cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void pd_cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// Visible keys of a row as steps of 2^LOG: those of the first tokens [0, nfirst),
// then those from nlow on.
struct PdRow {
    int len, first, low, nfirst, nlow;
    uint32_t steps;
};
template <int LOG>
__device__ __forceinline__ PdRow pd_row(const PagedAttnArgs &a, uint32_t row) {
    PdRow r;
    r.len = paged_length(a.c, a.seqs ? a.seqs[row] : row);
    const KeySpan k = key_span(r.len - 1, a.window, a.sinks);
    r.first = k.first;
    r.low = k.low;
    constexpr int up = (1 << LOG) - 1;
    r.nlow = k.low >> LOG;
    r.nfirst = min((k.first + up) >> LOG, r.nlow);
    r.steps = r.len > 0 ? (uint32_t)(r.nfirst + ((r.len + up) >> LOG) - r.nlow) : 0u;
    return r;
}

// DIRECT: CTA (or cluster of `parts` CTAs) b has row b / items, item b % items;
// its CTAs take equal parts of the context and join them over distributed
// shared memory. Otherwise CTA c takes the c-th run of all units.
template <bool KV8, int DIM, bool DIRECT>
__global__ void __launch_bounds__(PD_THREADS, PdCfg<KV8, DIM>::MINB) paged_decode_kernel(PagedAttnArgs a, PdWork w) {
    using C = PdCfg<KV8, DIM>;
    constexpr int KS = DIM / 16;  // k-steps of the first product, and 16-dim tiles of the second
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float wm[PD_WARPS][PD_HEADS], wl[PD_WARPS][PD_HEADS], wf[PD_WARPS][PD_HEADS], wM[PD_HEADS];
    __shared__ float fin[DIRECT ? PD_MAX_PARTS * (DIM + 2) : 1];  // m, l, o of the heads that this CTA joins, from every CTA of the cluster
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    // 16-byte chunks of a lane's query head: head 8 hblk + g, dims by the permutation that the key rows' chunks
    // give the first product (chunk t + 4 j of a row of keys)
    constexpr int NQ = DIM / 32;
    uint4 qraw[NQ];
    auto load_q = [&](uint32_t row_, uint32_t item_) {
        const uint32_t kvh_ = item_ / w.hb, hl = item_ % w.hb * PD_HEADS + g;
        const uint16_t *qp = a.q + row_ * a.q_stride + (uint64_t)(kvh_ * w.group + (hl < w.group ? hl : 0)) * DIM;
#pragma unroll
        for (int j = 0; j < NQ; ++j)
            qraw[j] = *reinterpret_cast<const uint4 *>(qp + (KV8 ? 16 * (t + 4 * (j >> 1)) + 8 * (j & 1) : 8 * (t + 4 * j)));
    };
    uint32_t row, u, u_end, base;  // units: u .. u_end, of the row's first one at `base`
    UnitSplit split;
    if constexpr (DIRECT) {
        const uint32_t unit = blockIdx.x / w.parts, part = blockIdx.x % w.parts;
        if (w.parts > 1) pd_cluster_arrive();
        row = unit / w.items;
        load_q(row, unit % w.items);  // needs no length
        const PdRow R = pd_row<C::LOG>(a, row);
        base = 0;
        const uint32_t first = unit % w.items * R.steps;
        u = first + (uint32_t)((uint64_t)R.steps * part / w.parts);
        u_end = first + (uint32_t)((uint64_t)R.steps * (part + 1) / w.parts);
        if (R.steps == 0) {  // no key (the whole cluster): zero
            const uint32_t item = unit % w.items, kvh = item / w.hb, h0 = item % w.hb * PD_HEADS;
            const uint32_t heads = min(w.group - h0, (uint32_t)PD_HEADS);
            uint16_t *out = a.ctx + row * a.ctx_stride + (uint64_t)(kvh * w.group + h0) * DIM;
            if (part == 0)
                for (uint32_t x = tid; x < heads * DIM / 8; x += PD_THREADS)
                    reinterpret_cast<uint4 *>(out)[x] = make_uint4(0, 0, 0, 0);
            if (w.parts > 1) pd_cluster_wait();
            return;
        }
    } else {
        // ---- the numbering of the units: prefix sums of the rows' steps
        __shared__ uint32_t wsum[PD_WARPS], at_prefix, at_row;
        pdl_trigger();  // the join kernel waits for this one to end
        const uint32_t per = (a.rows + PD_THREADS - 1) / PD_THREADS, r0 = min(tid * per, a.rows),
                       r1 = min(r0 + per, a.rows);
        uint32_t mine = 0;
        for (uint32_t r = r0; r < r1; ++r) mine += pd_row<C::LOG>(a, r).steps;
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < PD_WARPS; ++i) {
            if (i < warp) incl += wsum[i];
            all += wsum[i];
        }
        const uint32_t before = incl - mine;
        if (blockIdx.x == 0) {
            uint32_t p = before;
            for (uint32_t r = r0; r < r1; ++r) {
                w.prefix[r] = p;
                p += pd_row<C::LOG>(a, r).steps;
            }
            if (tid == 0) w.prefix[a.rows] = all;
        }
        split = UnitSplit(all * w.items, w.max_ctas, PD_MIN_UNITS);
        if (blockIdx.x >= split.g || all == 0) return;
        u = split.start(blockIdx.x);
        u_end = split.start(blockIdx.x + 1);
        if (before * w.items <= u && u < incl * w.items) {
            uint32_t p = before, r = r0;
            for (;; ++r) {
                const uint32_t n = pd_row<C::LOG>(a, r).steps;
                if (u < (p + n) * w.items) break;
                p += n;
            }
            at_row = r;
            at_prefix = p;
        }
        __syncthreads();
        row = at_row;
        base = at_prefix * w.items;
    }

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (C::STAGES * C::STEP_BYTES);
    const float fac0 = a.scale * 1.44269504f;
    bool first_segment = true;
    while (DIRECT || u < u_end) {  // DIRECT: once, also for a CTA of a cluster that has no step
        const PdRow R = pd_row<C::LOG>(a, row);
        if (!DIRECT && R.steps == 0) {
            ++row;
            continue;
        }
        const uint32_t item = (u - base) / R.steps, rem = u - base - item * R.steps;
        const int cnt = (int)min(R.steps - rem, u_end - u);
        const uint32_t kvh = item / w.hb, hblk = item % w.hb;
        if constexpr (!DIRECT) load_q(row, item);
        const uint32_t seq = a.seqs ? a.seqs[row] : row;
        const uint32_t *table = a.c.table + (uint64_t)seq * a.c.max_pages;
        const int pmask = (1 << a.c.tshift) - 1;

        // ---- this warp's steps: warp, warp + 8, .. of the segment
        const int nst = cnt > warp ? (cnt - warp + PD_WARPS - 1) / PD_WARPS : 0;
        auto key_of = [&](int i) {
            const int s = (int)rem + warp + i * PD_WARPS;
            return (s < R.nfirst ? s : s - R.nfirst + R.nlow) << C::LOG;
        };
        struct Pages {
            uint32_t id[C::SUBS];
        };
        auto pages_at = [&](int i) {
            Pages p;
#pragma unroll
            for (int b = 0; b < C::SUBS; ++b) {
                const int key = key_of(i) + PD_SUB * b;
                p.id[b] = i < nst && key < R.len ? __ldg(&table[key >> a.c.tshift]) : PG_NO_PAGE;
            }
            return p;
        };
        uint32_t there = 0;  // bit (i SUBS + b) % 32: that piece's page exists
        const uint64_t head_row = (uint64_t)kvh << a.c.tshift;
        auto load = [&](int i, Pages page) {
#pragma unroll
            for (int b = 0; i < nst && b < C::SUBS; ++b) {
                const int key = key_of(i) + PD_SUB * b;
                const bool ok = page.id[b] < a.c.pages;
                const uint32_t bit = (i * C::SUBS + b) & 31;
                there = (there & ~(1u << bit)) | ((uint32_t)ok << bit);
                const uint64_t r = ok ? page.id[b] * a.c.page_rows + head_row + (key & pmask) : 0;
                const uint8_t *kp = a.c.k + r * C::RB, *vp = a.c.v + r * C::RB;
                const uint32_t dst = ring + (i % C::STAGES) * C::STEP_BYTES + b * C::SUB_BYTES;
                // only visible keys are read; the others are zero
                auto copy = [&](auto bytes_of) {
#pragma unroll
                    for (int j = 0; j < C::CPR / 2; ++j) {
                        const int n = j * 32 + lane, kr = n / C::CPR, c = n % C::CPR;
                        const uint32_t bytes = bytes_of(kr, 16);
                        const int kc = C::CPR == 4 ? c : c ^ ((kr & 1) << 2);
                        const int vpos = C::CPR == 4 ? ((kr >> 1) << 3) + ((((kr & 1) << 2) | c) ^ (((kr >> 1) & 3) << 1))
                                                     : kr * C::CPR + (c ^ (((kr >> 1) & 3) << 1));
                        cp16(dst + (kr * C::CPR + kc) * 16, kp + n * 16, bytes);
                        cp16(dst + PD_SUB * C::RB + vpos * 16, vp + n * 16, bytes);
                    }
                    if constexpr (KV8)
                        cp4(dst + 2 * PD_SUB * C::RB + lane * 4, (lane < 16 ? a.c.ks : a.c.vs) + r + (lane & 15),
                            bytes_of(lane & 15, 4));
                };
                if (ok && key + 16 <= R.len && (key >= R.low || key + 16 <= R.first))
                    copy([](int, int n) { return n; });
                else
                    copy([&](int kr, int n) {
                        const int key_r = key + kr;
                        return ok && key_r < R.len && (key_r >= R.low || key_r < R.first) ? n : 0;
                    });
            }
            cp_commit();
        };
        Pages next;
        {
            Pages start[C::STAGES - 1];
#pragma unroll
            for (int i = 0; i < C::STAGES - 1; ++i) start[i] = pages_at(i);
            next = pages_at(C::STAGES - 1);
#pragma unroll
            for (int i = 0; i < C::STAGES - 1; ++i) load(i, start[i]);
        }

        // ---- the query heads as B fragments
        uint32_t qf[KS][2];
        float fac[2];
        {
            const bool live = hblk * PD_HEADS + g < w.group;
            if constexpr (KV8) {
                float x[KS][4], amax = 0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const uint4 v = qraw[k >> 1];
                    const uint32_t w0 = k & 1 ? v.z : v.x, w1 = k & 1 ? v.w : v.y;
                    x[k][0] = bflo(w0), x[k][1] = bfhi(w0), x[k][2] = bflo(w1), x[k][3] = bfhi(w1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[k][i]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                // 2^(14 - e): the largest |q| lands in [2^14, 2^15); values 2^-28 of it and smaller lose bits
                const int e = amax > 0.f ? min(max(ilogbf(amax), -100), 127) : 0;
                const float up = live ? pow2i(min(14 - e, 126)) : 0.f;
                const float down = fac0 * pow2i(-min(14 - e, 126));
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    qf[k][0] = pack_f16(x[k][0] * up, x[k][1] * up);
                    qf[k][1] = pack_f16(x[k][2] * up, x[k][3] * up);
                }
                fac[0] = __shfl_sync(0xffffffffu, down, 8 * t);  // of head 2t: lane 4 (2t)
                fac[1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
            } else {
#pragma unroll
                for (int j = 0; j < KS / 2; ++j) {
                    const uint4 v = live ? qraw[j] : make_uint4(0, 0, 0, 0);
                    qf[2 * j][0] = v.x;
                    qf[2 * j][1] = v.y;
                    qf[2 * j + 1][0] = v.z;
                    qf[2 * j + 1][1] = v.w;
                }
                fac[0] = fac[1] = fac0;
            }
        }

        float o[KS][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KS; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

        for (int i = 0; i < nst; ++i) {
            {
                const Pages page = next;
                next = pages_at(i + C::STAGES);
                load(i + C::STAGES - 1, page);
            }
            cp_wait<C::STAGES - 1>();
            __syncwarp();
            const uint32_t stage = ring + (i % C::STAGES) * C::STEP_BYTES;
            const int key0 = key_of(i);
            float s[C::SUBS][4], vs[C::SUBS][2];
#pragma unroll
            for (int b = 0; b < C::SUBS; ++b) {
                const uint32_t buf = stage + b * C::SUB_BYTES;
                // ---- scores of 16 keys (rows g, g + 8) x 8 heads (columns 2t, 2t + 1)
                float (&sb)[4] = s[b];
                sb[0] = sb[1] = sb[2] = sb[3] = 0.f;
                if constexpr (KV8) {
#pragma unroll
                    for (int j = 0; j < C::CPR / 4; ++j) {
                        const int c = t + 4 * j, x = C::CPR == 4 ? 0 : (g & 1) << 2;
                        const uint4 lo = lds128(buf + (g * C::CPR + (c ^ x)) * 16);
                        const uint4 hi = lds128(buf + ((g + 8) * C::CPR + (c ^ x)) * 16);
                        const uint32_t wl4[4] = {lo.x, lo.y, lo.z, lo.w}, wh4[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t a0, a1, a2, a3;
                            codes4_to_f16(wl4[k], a0, a2);
                            codes4_to_f16(wh4[k], a1, a3);
                            mma16816<true>(sb, a0, a1, a2, a3, qf[4 * j + k][0], qf[4 * j + k][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < C::CPR / 4; ++j) {
                        const int c = t + 4 * j, x = (g & 1) << 2;
                        const uint4 lo = lds128(buf + (g * C::CPR + (c ^ x)) * 16);
                        const uint4 hi = lds128(buf + ((g + 8) * C::CPR + (c ^ x)) * 16);
                        mma16816<false>(sb, lo.x, hi.x, lo.y, hi.y, qf[2 * j][0], qf[2 * j][1]);
                        mma16816<false>(sb, lo.z, hi.z, lo.w, hi.w, qf[2 * j + 1][0], qf[2 * j + 1][1]);
                    }
                }
                if constexpr (KV8) {
                    const uint32_t sc = buf + 2 * PD_SUB * C::RB;
                    const float k0 = lds32f(sc + g * 4), k1 = lds32f(sc + g * 4 + 32);
                    vs[b][0] = lds32f(sc + 64 + g * 4);
                    vs[b][1] = lds32f(sc + 96 + g * 4);
                    sb[0] *= k0 * fac[0];
                    sb[1] *= k0 * fac[1];
                    sb[2] *= k1 * fac[0];
                    sb[3] *= k1 * fac[1];
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) sb[k] *= fac0;
                }
                const int key = key0 + PD_SUB * b;
                const bool ok = there >> ((i * C::SUBS + b) & 31) & 1;
                if (!ok || key + 16 > R.len || (key < R.low && key + 16 > R.first)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int kr = key + g + 8 * h;
                        if (!ok || kr >= R.len || (kr < R.low && kr >= R.first))
                            sb[2 * h] = sb[2 * h + 1] = -INFINITY;
                    }
                }
            }
            // ---- the maximum, raised only where a score passes it by 2^8
            float top[2] = {fmaxf(s[0][0], s[0][2]), fmaxf(s[0][1], s[0][3])};
#pragma unroll
            for (int b = 1; b < C::SUBS; ++b) {
                top[0] = fmaxf(top[0], fmaxf(s[b][0], s[b][2]));
                top[1] = fmaxf(top[1], fmaxf(s[b][1], s[b][3]));
            }
            if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float x = top[h];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    x = fmaxf(x, m[h]);
                    const float f = m[h] == x ? 1.f : ex2(0.5f * (m[h] - x));
                    m[h] = x;
                    l[h] = l[h] * f * f;
#pragma unroll
                    for (int j = 0; j < KS; ++j) {
                        o[j][h] = o[j][h] * f * f;
                        o[j][h + 2] = o[j][h + 2] * f * f;
                    }
                }
            }
            const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
            for (int b = 0; b < C::SUBS; ++b) {
                const uint32_t buf = stage + b * C::SUB_BYTES;
                float p[4] = {ex2(s[b][0] - m0), ex2(s[b][1] - m1), ex2(s[b][2] - m0), ex2(s[b][3] - m1)};
                l[0] += p[0] + p[2];
                l[1] += p[1] + p[3];
                if constexpr (KV8) {
                    p[0] *= vs[b][0];
                    p[1] *= vs[b][0];
                    p[2] *= vs[b][1];
                    p[3] *= vs[b][1];
                }
                // ---- weights as hi + lo, transposed to (keys x heads) B fragments
                const uint32_t h0 = pack_bf16(p[0], p[1]), h1 = pack_bf16(p[2], p[3]);
                const uint32_t b0 = movmatrix(h0), b1 = movmatrix(h1);
                const uint32_t c0 = movmatrix(pack_bf16(p[0] - bflo(h0), p[1] - bfhi(h0)));
                const uint32_t c1 = movmatrix(pack_bf16(p[2] - bflo(h1), p[3] - bfhi(h1)));
                // ---- O^T += V^T P^T: tile j holds dims D0(g) + 2 j (row g) and + 1 (row g + 8)
                const uint32_t vb = buf + PD_SUB * C::RB;
                const int ra = 2 * t, rb = 2 * t + 8;  // keys 2t, 2t + 1 and 2t + 8, 2t + 9
                if constexpr (KV8 && DIM == 64) {
                    uint2 v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int kr = (k < 2 ? ra : rb) + (k & 1);
                        const int pos = ((kr >> 1) << 3) + ((((kr & 1) << 2) | (g >> 1)) ^ (((kr >> 1) & 3) << 1));
                        v[k] = lds64(vb + pos * 16 + (g & 1) * 8);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t x0 = j < 2 ? v[0].x : v[0].y, x1 = j < 2 ? v[1].x : v[1].y,
                                       x2 = j < 2 ? v[2].x : v[2].y, x3 = j < 2 ? v[3].x : v[3].y;
                        uint32_t a0, a1, a2, a3;
                        if (j & 1) {
                            a0 = codes_pair_bf16<2>(x0, x1), a1 = codes_pair_bf16<3>(x0, x1);
                            a2 = codes_pair_bf16<2>(x2, x3), a3 = codes_pair_bf16<3>(x2, x3);
                        } else {
                            a0 = codes_pair_bf16<0>(x0, x1), a1 = codes_pair_bf16<1>(x0, x1);
                            a2 = codes_pair_bf16<0>(x2, x3), a3 = codes_pair_bf16<1>(x2, x3);
                        }
                        mma16816<false>(o[j], a0, a1, a2, a3, b0, b1);
                        mma16816<false>(o[j], a0, a1, a2, a3, c0, c1);
                    }
                } else {
                    constexpr int NC = KV8 ? 1 : DIM / 64;  // 16-byte chunks of a key that this lane's dims take
#pragma unroll
                    for (int q = 0; q < NC; ++q) {
                        uint4 v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int kr = (k < 2 ? ra : rb) + (k & 1);
                            v[k] = lds128(vb + (kr * C::CPR + ((g + 8 * q) ^ (((kr >> 1) & 3) << 1))) * 16);
                        }
                        const uint32_t x[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w},
                                                  {v[1].x, v[1].y, v[1].z, v[1].w},
                                                  {v[2].x, v[2].y, v[2].z, v[2].w},
                                                  {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {  // word k of the chunks
                            if constexpr (KV8) {
                                uint32_t a0 = codes_pair_bf16<0>(x[0][k], x[1][k]), a1 = codes_pair_bf16<1>(x[0][k], x[1][k]);
                                uint32_t a2 = codes_pair_bf16<0>(x[2][k], x[3][k]), a3 = codes_pair_bf16<1>(x[2][k], x[3][k]);
                                mma16816<false>(o[2 * k], a0, a1, a2, a3, b0, b1);
                                mma16816<false>(o[2 * k], a0, a1, a2, a3, c0, c1);
                                a0 = codes_pair_bf16<2>(x[0][k], x[1][k]), a1 = codes_pair_bf16<3>(x[0][k], x[1][k]);
                                a2 = codes_pair_bf16<2>(x[2][k], x[3][k]), a3 = codes_pair_bf16<3>(x[2][k], x[3][k]);
                                mma16816<false>(o[2 * k + 1], a0, a1, a2, a3, b0, b1);
                                mma16816<false>(o[2 * k + 1], a0, a1, a2, a3, c0, c1);
                            } else {
                                const uint32_t a0 = __byte_perm(x[0][k], x[1][k], 0x5410),
                                               a1 = __byte_perm(x[0][k], x[1][k], 0x7632);
                                const uint32_t a2 = __byte_perm(x[2][k], x[3][k], 0x5410),
                                               a3 = __byte_perm(x[2][k], x[3][k], 0x7632);
                                mma16816<false>(o[4 * q + k], a0, a1, a2, a3, b0, b1);
                                mma16816<false>(o[4 * q + k], a0, a1, a2, a3, c0, c1);
                            }
                        }
                    }
                }
            }
            __syncwarp();  // the stage may be refilled
        }
        cp_wait<0>();

        // ---- the warps' results joined through shared memory (over the drained rings)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
        __syncthreads();
        float *os = reinterpret_cast<float *>(smem);
        if (g == 0) {
            wm[warp][2 * t] = m[0];
            wm[warp][2 * t + 1] = m[1];
            wl[warp][2 * t] = l[0];
            wl[warp][2 * t + 1] = l[1];
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            int d = 2 * j + (KV8 || DIM == 64 ? (DIM / 8) * g : 0);
            if (!KV8 && DIM == 128) d = (j < 4 ? 8 * g + 2 * j : 64 + 8 * g + 2 * (j - 4));
#pragma unroll
            for (int k = 0; k < 4; ++k)
                os[(warp * PD_HEADS + 2 * t + (k & 1)) * (DIM + 1) + d + (k >> 1)] = o[j][k];
        }
        __syncthreads();
        if (tid < PD_HEADS * PD_WARPS) {  // each warp's factor, applied twice: 2^(m - M) may underflow where o 2^(m - M) does not
            const int h = tid % PD_HEADS, i = tid / PD_HEADS;
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < PD_WARPS; ++k) M = fmaxf(M, wm[k][h]);
            wf[i][h] = ex2(0.5f * (wm[i][h] - (M == -INFINITY ? 0.f : M)));
            if (i == 0) wM[h] = M;
        }
        __syncthreads();
        const bool whole = DIRECT ? w.parts == 1 : cnt == R.steps;
        float *piece = w.pieces + ((uint64_t)blockIdx.x * 2 + (first_segment ? 0 : 1)) * C::PIECE;
        const uint32_t part = DIRECT ? blockIdx.x % w.parts : 0;
        if constexpr (DIRECT)
            if (w.parts > 1) pd_cluster_wait();  // every CTA of the cluster has started
        for (int x = tid; x < PD_HEADS * DIM; x += PD_THREADS) {
            const int h = x / DIM, d = x % DIM;
            float L = 0.f, O = 0.f;
#pragma unroll
            for (int i = 0; i < PD_WARPS; ++i) {
                const float f = wf[i][h];
                L += wl[i][h] * f * f;
                O += os[(i * PD_HEADS + h) * (DIM + 1) + d] * f * f;
            }
            const uint32_t hl = hblk * PD_HEADS + h;
            if (whole) {
                if (hl < w.group)
                    a.ctx[row * a.ctx_stride + (uint64_t)(kvh * w.group + hl) * DIM + d] = f2bf(L == 0.f ? 0.f : O / L);
            } else if constexpr (DIRECT) {
                // head h is joined by CTA h % parts, from slot `part` of its shared memory
                const uint32_t slot = (part * pd_heads_here(w.parts) + h / w.parts) * (DIM + 2);
                const uint32_t to = (uint32_t)__cvta_generic_to_shared(fin + slot);
                pd_dsmem_store(to + 4 * (2 + d), h % w.parts, O);
                if (d == 0) {
                    pd_dsmem_store(to, h % w.parts, wM[h]);
                    pd_dsmem_store(to + 4, h % w.parts, L);
                }
            } else {
                piece[2 * PD_HEADS + x] = O;
                if (d == 0) {
                    piece[h] = wM[h];
                    piece[PD_HEADS + h] = L;
                }
            }
        }
        if constexpr (DIRECT) {
            if (w.parts > 1) {
                tc::cluster_sync();
                const uint32_t mine = pd_heads_here(w.parts);  // part, part + parts, .. as far as there are heads
                for (uint32_t x = tid; x < mine * DIM && part + x / DIM * w.parts < PD_HEADS; x += PD_THREADS) {
                    const uint32_t k = x / DIM, d = x % DIM;
                    float M = -INFINITY, L = 0.f, O = 0.f;
                    for (uint32_t i = 0; i < w.parts; ++i) M = fmaxf(M, fin[(i * mine + k) * (DIM + 2)]);
                    const float M0 = M == -INFINITY ? 0.f : M;
                    for (uint32_t i = 0; i < w.parts; ++i) {
                        const float *p = fin + (i * mine + k) * (DIM + 2);
                        const float f = ex2(0.5f * (p[0] - M0));
                        L += p[1] * f * f;
                        O += p[2 + d] * f * f;
                    }
                    const uint32_t hl = hblk * PD_HEADS + part + k * w.parts;
                    if (hl < w.group)
                        a.ctx[row * a.ctx_stride + (uint64_t)(kvh * w.group + hl) * DIM + d] = f2bf(L == 0.f ? 0.f : O / L);
                }
            }
            return;
        }
        __syncthreads();  // os is read before the next segment's loads
        first_segment = false;
        u += cnt;
        if (u == base + R.steps * w.items) {
            base = u;
            ++row;
        }
    }
}

// One CTA per (item, query head): the pieces of the item's context, PJ_GROUPS of
// them at a time, added in a fixed order; items without keys are zero, items
// of one CTA are already written.
constexpr int PJ_GROUPS = 8;
template <int DIM>
__global__ void __launch_bounds__(DIM *PJ_GROUPS) paged_join_kernel(PagedAttnArgs a, PdWork w) {
    constexpr int PIECE = 2 * PD_HEADS + PD_HEADS * DIM;
    __shared__ float wt[2 * PD_MAX_SMS], lt[2 * PD_MAX_SMS], top[PJ_GROUPS * DIM / 32], so[PJ_GROUPS][DIM];
    pdl_wait();
    const uint32_t qh = w.items * PD_HEADS;  // heads, the last block of each KV head filled up
    const uint32_t row = blockIdx.x / qh, item = blockIdx.x % qh / PD_HEADS, h = blockIdx.x % PD_HEADS;
    const uint32_t kvh = item / w.hb, hl = (item % w.hb) * PD_HEADS + h;
    if (hl >= w.group) return;
    const int d = threadIdx.x % DIM, grp = threadIdx.x / DIM;
    uint16_t *out = a.ctx + row * a.ctx_stride + (uint64_t)(kvh * w.group + hl) * DIM + d;
    const uint32_t p0 = w.prefix[row], steps = w.prefix[row + 1] - p0;
    if (steps == 0) {
        if (grp == 0) *out = 0;
        return;
    }
    const UnitSplit split(w.prefix[a.rows] * w.items, w.max_ctas, PD_MIN_UNITS);
    const uint32_t u0 = p0 * w.items + item * steps;
    const uint32_t c0 = split.cta_of(u0), c1 = split.cta_of(u0 + steps - 1), n = c1 - c0 + 1;
    if (n == 1) return;
    auto piece = [&](uint32_t i) {  // the item's segment of CTA c0 + i: the CTA's first one unless c0 began before the item
        return w.pieces + ((uint64_t)(c0 + i) * 2 + (i == 0 && split.start(c0) < u0)) * PIECE;
    };
    float M = -INFINITY;
    for (uint32_t i = threadIdx.x; i < n; i += DIM * PJ_GROUPS) {
        const float *p = piece(i);
        wt[i] = p[h];
        lt[i] = p[PD_HEADS + h];
        M = fmaxf(M, wt[i]);
    }
    M = warp_max(M);
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = M;
    __syncthreads();
    M = top[0];
#pragma unroll
    for (int i = 1; i < PJ_GROUPS * DIM / 32; ++i) M = fmaxf(M, top[i]);
    const float M0 = M == -INFINITY ? 0.f : M;
    float O = 0.f;
#pragma unroll 4
    for (uint32_t i = grp; i < n; i += PJ_GROUPS) {
        const float f = ex2(0.5f * (wt[i] - M0));
        O += piece(i)[2 * PD_HEADS + h * DIM + d] * f * f;
    }
    so[grp][d] = O;
    __syncthreads();
    if (grp) return;
    float L = 0.f;
    for (uint32_t i = 0; i < n; ++i) {
        const float f = ex2(0.5f * (wt[i] - M0));
        L += lt[i] * f * f;
    }
#pragma unroll
    for (int i = 1; i < PJ_GROUPS; ++i) O += so[i][d];
    *out = f2bf(L == 0.f ? 0.f : O / L);
}

static size_t pd_prefix_bytes(uint32_t rows) { return (((size_t)rows + 1) * 4 + 255) & ~(size_t)255; }

size_t paged_decode_ws(uint32_t, uint32_t, uint32_t dim, uint32_t rows) {
    return pd_prefix_bytes(rows) + (size_t)2 * PD_MAX_SMS * 2 * (2 * PD_HEADS + PD_HEADS * dim) * 4;
}

// Whether the current device holds `units` clusters of `parts` CTAs (9 to 16) at once; asked once per device and size.
template <bool KV8, int DIM>
static bool pd_fits(uint32_t parts, uint32_t units) {
    using C = PdCfg<KV8, DIM>;
    static int known[64][PD_MAX_PARTS + 1];  // 1 + the answer, written with the same value by every thread that finds 0
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    int n = __atomic_load_n(&known[dev][parts], __ATOMIC_RELAXED);
    if (!n) {
        auto *kernel = paged_decode_kernel<KV8, DIM, true>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(parts);
        cfg.blockDim = dim3(PD_THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = parts;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            clusters = 0;
        }
        n = 1 + clusters;
        __atomic_store_n(&known[dev][parts], n, __ATOMIC_RELAXED);
    }
    return n - 1 >= (int)units;
}

template <bool KV8, int DIM>
static int launch_decode(const PagedAttnArgs &a, PdWork w, int sms, cudaStream_t st) {
    using C = PdCfg<KV8, DIM>;
    // Which way: a CTA or cluster per (row, item) where those fill a third of the GPU, or where no context can be
    // longer than its CTAs are worth (the host knows the table's width and the window only); else equal runs of
    // units and a join kernel. Measured, first way against second: 64 rows x 2 KV heads x 2048 keys KV8 14.9 and
    // 24.9 us, one row x 8 heads x 32768 keys bf16 28.9 and 37.7 us, one row x 2 heads KV8 8192 keys 8.5 and 11.4,
    // 32768 keys 16.2 and 15.2, 131072 keys 41.7 and 22.4 us.
    const uint32_t slots = (uint32_t)(sms * C::MINB), units = a.rows * w.items;
    uint64_t most = (uint64_t)a.c.max_pages << a.c.tshift;
    if (a.window) {
        const uint64_t seen = (uint64_t)a.window + a.sinks;
        most = most < seen ? most : seen;
    }
    const uint64_t want = (most + PD_PART_KEYS - 1) / PD_PART_KEYS, room = units < slots ? slots / units : 1;
    uint64_t parts = want < room ? want : room;
    parts = parts < 1 ? 1 : parts < PD_MAX_PARTS ? parts : PD_MAX_PARTS;
    while (parts > 8 && !pd_fits<KV8, DIM>((uint32_t)parts, units)) --parts;
    w.parts = (uint32_t)parts;
    if (units * parts * 3 >= slots || most <= parts * PD_PART_MOST) {
        auto *kernel = paged_decode_kernel<KV8, DIM, true>;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return -3;
        if (parts > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return -3;
        return launch_pdl(kernel, dim3(units * w.parts), dim3(PD_THREADS), C::SMEM, st, w.parts, a, w);
    }
    auto *kernel = paged_decode_kernel<KV8, DIM, false>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return -3;
    w.max_ctas = slots;
    PdlChain chain;
    if (int rc = launch_pdl(kernel, dim3(w.max_ctas), dim3(PD_THREADS), C::SMEM, st, 1, a, w)) return rc;
    return launch_pdl(paged_join_kernel<DIM>, dim3(units * PD_HEADS), dim3(DIM * PJ_GROUPS), 0, st, 1, a, w);
}

int launch_paged_decode(const PagedAttnArgs &a, void *ws, cudaStream_t st) {
    const int sms = paged_sms();
    if (sms <= 0) return -3;
    PdWork w;
    w.group = a.qh / a.c.hkv;
    w.hb = (w.group + PD_HEADS - 1) / PD_HEADS;
    w.items = a.c.hkv * w.hb;
    // units are counted in 32 bits
    if ((uint64_t)a.rows * w.items * PD_HEADS >= 1ull << 31) return -1;
    if ((uint64_t)a.rows * w.items * ((((uint64_t)a.c.max_pages << a.c.tshift) >> 4) + 3) >= 1ull << 32) return -1;
    w.prefix = (uint32_t *)ws;
    w.pieces = reinterpret_cast<float *>((char *)ws + pd_prefix_bytes(a.rows));
    const int n = sms < PD_MAX_SMS ? sms : PD_MAX_SMS;
    if (a.format == QWEN_B200_KV8)
        return a.dim == 64 ? launch_decode<true, 64>(a, w, n, st) : launch_decode<true, 128>(a, w, n, st);
    return a.dim == 64 ? launch_decode<false, 64>(a, w, n, st) : launch_decode<false, 128>(a, w, n, st);
}

}  // namespace qb
