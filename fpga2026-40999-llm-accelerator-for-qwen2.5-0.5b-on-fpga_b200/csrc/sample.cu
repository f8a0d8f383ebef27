// One token per row of bf16 logits from a given random number, under a
// temperature, top-k, top-p and min-p.
//
// Mathematics: the candidates in the order of their logits, the lower id first
// among equals; w_i = exp((l_i - l_max) / T). Every filter keeps a prefix of
// that order, so the kept candidates are the shortest of them; the token is the
// first whose running sum of weights passes u times the kept weights' sum.
//
// A bf16 logit is one of 65536 values and the weight depends on nothing else,
// so the row is never sorted: it is counted. A histogram of the values (exact
// whole numbers), one exponential in 64 bits for each value that occurs, and
// scans over the values in falling order give every border; the token is
// then the j-th occurrence of one value. Weights are whole multiples of
// 2^-(63 - bits of the vocabulary), summed as 64-bit integers: exact in any
// order, so the answer does not depend on the launch.
//
// The histogram has a window of 12288 values in shared memory. One window holds
// 0 and every magnitude in [2^-39, 2^8), which is all of a row in practice: what
// lies below it (masks such as -1e4 or the lowest value) has no weight and is left
// out. A row for which that does not hold goes through 6 windows of 12288 of the
// 65536 values instead, counted anew at each step (about ten times slower).
//
// A cluster of C CTAs has a row: each counts a part of it, then takes 12288 / C
// values, 32 a step: a warp adds the CTAs' counts of a step over distributed
// shared memory, forms the weights, sums them and gives the sums to every CTA.
// From there each CTA finds every border by itself: a thread has the sums of a
// step, and the one in whose step a border lies looks closer with its warp.
//
// Bound by counting where every logit matters: adds to shared memory take 3.4
// clocks a warp at random banks (1.0 without conflicts; copies of the counters
// do not help), 17 us of 256 rows of 151936 on 148 SMs, and about 12 instructions a
// logit. 256 rows, top_p alone, 49 us (DRAM floor 12): counting 28, sums 8, the
// last look 11. 64 rows with all filters and 8 masked rows 21 us on the device, one
// row 11.5: there latency, of the loads, two exchanges and the sums.
// CTAs of a row: as many of 8, 4, 2 and 1 as leave room for all rows at once (33, 71 and
// 148 rows on 148 SMs). Rows of 151936, top_p, by 8, 4, 2 and 1 CTAs each, us of a captured
// call with L2 flushed: 33 rows 27, 29, 33, 41; 37 rows 39, 27, 33, 39; 64 rows 47, 29, 33, 41;
// 74 rows 57, 43, 33, 39; 148 rows 92, 61, 39, 41; 149 rows 92, 61, 53, 51; 256 rows 143, 90, 68, 53.
#include "kernels.h"
#include "qwen_b200.h"
#include "sample.cuh"
#include "tc05.cuh"

namespace qb {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_MAX_CTAS = 8;
constexpr uint32_t SM_BINS = 12288, SM_WINDOWS = (65536 + SM_BINS - 1) / SM_BINS;
// The usual window: magnitudes from SM_LOW on (as bf16 bits), SM_SIDE of them on each side of 0.
constexpr uint32_t SM_LOW = 0x2c00, SM_SIDE = 47 * 128;
constexpr int SM_BATCH = 2, SM_LOOK = 8;   // 16-byte loads of a thread in flight: counting, and at the last look
constexpr uint32_t SM_NONE = 0xff80ff80u;  // two logits of -infinity
constexpr uint32_t SM_BELOW = (0x8000u | (SM_LOW + SM_SIDE - 1)) * 0x10001u;  // two of the lowest of the window

// What a cluster's CTAs tell one another; written by their peers.
struct SmShared {
    uint32_t first[SM_MAX_CTAS];           // lowest order (largest logit) of each CTA's part
    uint32_t below[SM_MAX_CTAS];           // the same of its values below the usual window
    uint32_t odd[SM_MAX_CTAS];             // whether it has values that the window's two sides do not hold
    // this CTA's own
    unsigned long long top_k, top_p;       // weights of the k first, and of those that top_p leaves
    uint32_t bin, nth;                     // the token: nth occurrence of a value
    uint32_t found;                        // in this window
    uint32_t wcount[SM_WARPS], wbelow[SM_WARPS], wodd;
    unsigned long long wsum[SM_WARPS], whigh[SM_WARPS];
};

__device__ __forceinline__ uint32_t sm_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t sm_remote(const void *p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tc::smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void sm_put32(void *p, uint32_t rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(sm_remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void sm_put64(void *p, uint32_t rank, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(sm_remote(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t sm_get32(const void *p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sm_remote(p, rank)) : "memory");
    return v;
}
// All CTAs of the row have started: a store to another's shared memory is defined from then on. Arrived at first thing, waited
// for behind the counting.
template <int C>
__device__ __forceinline__ void sm_arrive() {
    if constexpr (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
template <int C>
__device__ __forceinline__ void sm_started() {
    if constexpr (C > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// All CTAs of the row.
template <int C>
__device__ __forceinline__ void sm_sync() {
    if constexpr (C > 1)
        tc::cluster_sync();
    else
        __syncthreads();
}

// A logit's place in falling order: 0x007f is +infinity, 0xff7f the lowest finite value. Both zeros are +0.
__device__ __forceinline__ uint32_t sm_order(uint32_t b) {
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? b : 0x7fffu - b;
}
__device__ __forceinline__ float sm_value(uint32_t order) { return bf2f(order & 0x8000u ? order : 0x7fffu - order); }
__device__ __forceinline__ bool sm_counts(uint32_t order) { return order >= 0x7fu && order < 0xff80u; }  // no NaN, no -infinity
// Bin of a value in a window: -1 if it is not there. Window SM_WINDOWS is the usual one.
__device__ __forceinline__ int sm_bin(uint32_t b, uint32_t window) {
    const uint32_t mag = b & 0x7fffu;
    if (window == SM_WINDOWS) {
        const uint32_t t = mag - SM_LOW, negative = (uint32_t)((int)(b << 16) >> 31);
        if (t < SM_SIDE) return (int)((t ^ ~negative) + SM_SIDE - negative);  // SM_SIDE - 1 - t, or SM_SIDE + 1 + t
        return mag == 0 ? (int)SM_SIDE : -1;
    }
    const uint32_t d = sm_order(b);
    return sm_counts(d) && d / SM_BINS == window ? (int)(d % SM_BINS) : -1;
}
// The counter of a bin: in the usual window magnitudes rise on both sides, so that counting needs a sign and a sum.
__device__ __forceinline__ uint32_t sm_place(uint32_t bin, uint32_t window) {
    if (window != SM_WINDOWS || bin > 2 * SM_SIDE) return bin;
    return bin < SM_SIDE ? SM_SIDE - 1 - bin : bin == SM_SIDE ? 2 * SM_SIDE : bin - 1;
}
__device__ __forceinline__ float sm_bin_value(uint32_t bin, uint32_t window) {
    if (window == SM_WINDOWS)
        return bf2f(bin < SM_SIDE ? SM_LOW + SM_SIDE - 1 - bin : bin == SM_SIDE ? 0u : 0x8000u | (SM_LOW + bin - SM_SIDE - 1));
    return sm_value(window * SM_BINS + bin);
}

// The logits of a row in 16-byte groups by their addresses: group i has the elements 8 i - skew ..
static __device__ __noinline__ uint4 sm_edge(const uint16_t *base, uint32_t at, uint32_t begin, uint32_t end) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t b = at + k >= begin && at + k < end ? base[at + k] : 0xff80u;  // -infinity
        w[k >> 1] = k & 1 ? w[k >> 1] | b << 16 : b;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
struct SmRow {
    const uint16_t *base;  // the group that holds element 0
    uint32_t skew, vocab;
    uint32_t whole0, whole;  // groups whole0 .. whole0 + whole - 1 lie inside the row
    __device__ __forceinline__ uint4 group(uint32_t i) const {
        if (i - whole0 < whole) return *reinterpret_cast<const uint4 *>(base + 8 * i);
        return sm_edge(base, 8 * i, skew, skew + vocab);
    }
};
__device__ __forceinline__ uint32_t sm_half(const uint4 &v, int k) {
    const uint32_t w = k < 4 ? (k < 2 ? v.x : v.y) : (k < 6 ? v.z : v.w);
    return k & 1 ? w >> 16 : w & 0xffffu;
}

// Shared memory beside SmShared: the histogram, of this CTA's values the counts of all CTAs, and of all steps the weights,
// those of at least min_p, and the counts.
constexpr int SM_STEPS = SM_BINS / 32;
template <int C>
struct SmCfg {
    static constexpr int SEG = SM_BINS / C, STEPS = SEG / 32;  // values and steps of a CTA
    static constexpr int COUNTS = SM_BINS * 4, SUMS = COUNTS + (C > 1 ? SEG * 4 : 0), BYTES = SUMS + SM_STEPS * 20;
    static_assert(STEPS % SM_WARPS == 0 && SM_STEPS <= SM_THREADS, "steps");
};

template <typename T>
__device__ __forceinline__ T sm_warp_sum(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename T>
__device__ __forceinline__ T sm_warp_scan(T v) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T y = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += y;
    }
    return v;
}
// Of two bf16 pairs, all ones in the halves for which it holds.
__device__ __forceinline__ uint32_t sm_ge2(uint32_t a, uint32_t b) {
    return __hge2_mask(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
}
__device__ __forceinline__ uint32_t sm_lt2(uint32_t a, uint32_t b) {
    return __hlt2_mask(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
}
__device__ __forceinline__ uint32_t sm_eq2(uint32_t a, uint32_t b) {
    return __heq2_mask(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
}
__device__ __forceinline__ uint32_t sm_max2(uint32_t a, uint32_t b) {  // of two bf16 pairs; NaN counts as nothing
    uint32_t d;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

template <int C>
__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(SampleArgs a) {
    using K = SmCfg<C>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ SmShared sh;
    uint32_t *const hist = reinterpret_cast<uint32_t *>(smem);
    uint32_t *const counts = reinterpret_cast<uint32_t *>(smem + (C > 1 ? K::COUNTS : 0));
    unsigned long long *const step_sum = reinterpret_cast<unsigned long long *>(smem + K::SUMS), *const step_high = step_sum + SM_STEPS;
    uint32_t *const step_count = reinterpret_cast<uint32_t *>(step_high + SM_STEPS);
    sm_arrive<C>();
    const uint32_t rank = C > 1 ? sm_rank() : 0, row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits + row * a.stride);
    SmRow x;
    x.base = reinterpret_cast<const uint16_t *>(at & ~(uintptr_t)15);
    x.skew = (uint32_t)(at & 15) / 2;
    x.vocab = a.vocab;
    x.whole0 = x.skew ? 1 : 0;
    x.whole = max((x.skew + a.vocab) / 8, x.whole0) - x.whole0;
    const uint32_t groups = (x.skew + a.vocab + 7) / 8, g0 = min(rank * a.part, groups), g1 = min(g0 + a.part, groups);
    const float temperature = a.temperature ? a.temperature[row] : 1.f;
    const bool greedy = !(temperature > 0.f);
    const uint32_t k_of = a.top_k && !greedy ? a.top_k[row] : 0;
    const float p = a.top_p && !greedy ? a.top_p[row] : 1.f, least = a.min_p && !greedy ? a.min_p[row] : 0.f, u = a.u[row];

    // Weights are whole numbers of 1 / unit, from an exponential in 64 bits. 1 / T is rounded first, which spares each value a
    // division: it, l - top and their product take a weight e^-x off by up to x e^-x 2^-53 each (x e^-x is at most 0.37), exp
    // by its last place, 2^-53 below 1: 2.2 * 2^-53 in all, less than half a unit from vocabularies of 4096 on.
    const double slope = 1.0 / temperature, unit = __longlong_as_double((long long)(1023 + a.unit) << 52);
    // the least weight that min_p leaves (NaN: none)
    const unsigned long long floor = least <= 0.f ? 0 : least <= 1.f ? __double2ull_ru(least * unit) : ~0ull;

    // ---- this CTA's part of the row, counted in the usual window
    auto clear = [&] {
        for (uint32_t i = tid; i < SM_BINS / 4; i += SM_THREADS) reinterpret_cast<uint4 *>(hist)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    };
    // visit(16 bytes) for this CTA's part, SM_BATCH loads of a thread in flight
    auto each_group = [&](auto &&visit) {
        uint4 next[SM_BATCH];
#pragma unroll
        for (int i = 0; i < SM_BATCH; ++i)
            if (g0 + tid + i * SM_THREADS < g1) next[i] = x.group(g0 + tid + i * SM_THREADS);
        for (uint32_t g = g0 + tid; g < g1; g += SM_BATCH * SM_THREADS) {
#pragma unroll
            for (int i = 0; i < SM_BATCH; ++i) {
                const uint4 v = next[i];
                const uint32_t ahead = g + (SM_BATCH + i) * SM_THREADS;
                if (ahead < g1) next[i] = x.group(ahead);
                if (g + i * SM_THREADS < g1) visit(v);
            }
        }
    };
    if (tid == 0) sh.wodd = 0, sh.found = 0;
    clear();
    uint32_t top2 = SM_NONE, below2 = SM_NONE;
    bool odd = false;
    const uint32_t bins = tc::smem_u32(hist);
    each_group([&](uint4 v) {
        const uint32_t w4[4] = {v.x, v.y, v.z, v.w};
        uint32_t in[4];  // halves whose value has a counter of its sign and magnitude
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            top2 = sm_max2(top2, w4[k]);
            const uint32_t mag = w4[k] & 0x7fff7fffu;
            in[k] = sm_ge2(mag, SM_LOW * 0x10001u) & sm_lt2(mag, (SM_LOW + SM_SIDE) * 0x10001u);
        }
        // element k's counter: bins + 4 t, or + 4 (SM_SIDE + t), t the magnitude's bits above SM_LOW
        auto counter = [&](int k) {
            const uint32_t w = w4[k >> 1], mag4 = (k & 1 ? w >> 14 : w << 2) & 0x1fffcu;
            uint32_t negative;  // all ones, or 0
            asm("prmt.b32 %0, %1, 0, %2;" : "=r"(negative) : "r"(w), "r"(k & 1 ? 0xbbbbu : 0x9999u));
            return mag4 + (negative & (4 * SM_SIDE)) + (bins - 4 * SM_LOW);
        };
        if ((in[0] & in[1] & in[2] & in[3]) == 0xffffffffu) {
#pragma unroll
            for (int k = 0; k < 8; ++k) asm volatile("red.shared.add.u32 [%0], 1;" ::"r"(counter(k)) : "memory");
            return;
        }
        // some that have none: below the window, as masked ones, or 0, NaN and the rest
        uint32_t rest = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t low = sm_lt2(w4[k], SM_BELOW);
            below2 = sm_max2(below2, (w4[k] & low) | (SM_NONE & ~low));
            rest |= ~(in[k] | low) & (0x00010001u << k);  // element 2 k in bit k, 2 k + 1 in bit 16 + k
        }
        if (in[0] | in[1] | in[2] | in[3]) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p red.shared.add.u32 [%0], 1;\n\t}" ::"r"(counter(k)),
                             "r"(in[k >> 1] & (k & 1 ? 0xffff0000u : 0xffffu))
                             : "memory");
        }
        for (; rest; rest &= rest - 1) {
            const int i = __ffs(rest) - 1;
            const uint32_t w = (i & 3) < 2 ? (i & 1 ? v.y : v.x) : (i & 1 ? v.w : v.z), b = i < 16 ? w & 0xffffu : w >> 16;
            if ((b & 0x7fffu) == 0)
                atomicAdd(&hist[sm_place(SM_SIDE, SM_WINDOWS)], 1);
            else if (sm_counts(sm_order(b)))
                odd = true;
        }
    });
    uint32_t first = min(sm_order(top2 & 0xffffu), sm_order(top2 >> 16));  // (-infinity: no candidate)
    uint32_t below = min(sm_order(below2 & 0xffffu), sm_order(below2 >> 16));
    first = __reduce_min_sync(0xffffffffu, first);
    below = __reduce_min_sync(0xffffffffu, below);
    if (lane == 0) sh.wcount[warp] = first, sh.wbelow[warp] = below;
    if (odd) sh.wodd = 1;
    __syncthreads();
    sm_started<C>();
    if (warp == 0) {
        first = __reduce_min_sync(0xffffffffu, sh.wcount[lane % SM_WARPS]);
        below = __reduce_min_sync(0xffffffffu, sh.wbelow[lane % SM_WARPS]);
        if (lane < C) {
            sm_put32(&sh.first[rank], lane, first);
            sm_put32(&sh.below[rank], lane, below);
            sm_put32(&sh.odd[rank], lane, sh.wodd);
        }
    }
    sm_sync<C>();
    first = below = 0xffffu;
    odd = false;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        first = min(first, sh.first[c]);
        below = min(below, sh.below[c]);
        odd = odd || sh.odd[c] != 0;
    }
    if (!sm_counts(first)) {  // no candidate
        if (rank == 0 && tid == 0) {
            a.tokens[row] = QWEN_B200_NO_TOKEN;
            if (a.probs) a.probs[row] = 0.f;
        }
        return;  // (no CTA reads another's memory any more)
    }
    const double top = sm_value(first);
    const bool sharp = greedy || isinf(top);  // only the largest counts
    auto weight = [&](double l) {
        return __double2ull_rn((l == top ? 1.0 : sharp ? 0.0 : exp((l - top) * slope)) * unit);
    };
    const bool usual = !odd && (!sm_counts(below) || weight(sm_value(below)) == 0);

    // ---- a window's counts and weights; cb and sb: candidates and weights before this thread's step, cnt and sum of it,
    // cw, sw and hw of the window (hw: of at least `floor`)
    uint32_t window = SM_WINDOWS, cb = 0, cnt = 0, cw = 0;
    unsigned long long sb = 0, sum = 0, sw = 0, hw = 0;
    auto scan = [&](uint32_t c_before, unsigned long long s_before) {
        constexpr int MINE = K::STEPS / SM_WARPS;  // steps of a warp, in turn: the values that occur are neighbours
#pragma unroll(MINE < 6 ? MINE : 6)
        for (int i = 0; i < MINE; ++i) {
            const uint32_t step = SM_WARPS * i + warp, at = 32 * step + lane, place = sm_place(rank * K::SEG + at, window);
            uint32_t n = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) n += C > 1 ? sm_get32(&hist[place], c) : hist[place];
            if (C > 1) counts[at] = n;
            const uint32_t c = __reduce_add_sync(0xffffffffu, n);
            unsigned long long s = 0, h = 0;
            if (c) {
                const unsigned long long w = n ? weight(sm_bin_value(rank * K::SEG + at, window)) : 0;
                s = sm_warp_sum(n * w);
                h = floor == 0 ? s : sm_warp_sum(w >= floor ? n * w : 0ull);
            }
            const uint32_t to = rank * K::STEPS + step;
            if (C == 1) {
                if (lane == 0) step_count[to] = c, step_sum[to] = s, step_high[to] = h;
            } else if (lane < C) {
                sm_put32(&step_count[to], lane, c);
                sm_put64(&step_sum[to], lane, s);
                sm_put64(&step_high[to], lane, h);
            }
        }
        sm_sync<C>();
        unsigned long long high = 0;
        cnt = 0, sum = 0;
        if (tid < SM_STEPS) cnt = step_count[tid], sum = step_sum[tid], high = step_high[tid];
        const uint32_t ic = sm_warp_scan(cnt);
        const unsigned long long is = sm_warp_scan(sum);
        high = sm_warp_sum(high);
        if (lane == 31) sh.wcount[warp] = ic, sh.wsum[warp] = is, sh.whigh[warp] = high;
        __syncthreads();
        cb = c_before + ic - cnt, sb = s_before + is - sum;
        cw = 0, sw = 0, hw = 0;
#pragma unroll
        for (int i = 0; i < SM_WARPS; ++i) {
            const uint32_t y = sh.wcount[i];
            const unsigned long long z = sh.wsum[i];
            if (i < warp) cb += y, sb += z;
            cw += y, sw += z, hw += sh.whigh[i];
        }
    };
    // Where `here` holds for one thread (a border lies in its step): the first value at which `there`(candidates, weights up
    // to its end) holds; tell(its bin, its count and weight, weights and candidates before it) by one lane. Whole warps call
    // it, every CTA with the same result.
    auto find = [&](bool here, auto &&there, auto &&tell) {
        const uint32_t owner = __ballot_sync(0xffffffffu, here);
        if (!owner) return;
        const int l = __ffs(owner) - 1;
        const uint32_t step = 32 * warp + l, at = 32 * step + lane, c = __shfl_sync(0xffffffffu, cb, l);
        const uint32_t n = C > 1 ? sm_get32(&counts[at % K::SEG], step / K::STEPS) : hist[sm_place(at, window)];
        const unsigned long long s = __shfl_sync(0xffffffffu, sb, l), w = n ? weight(sm_bin_value(at, window)) : 0;
        const uint32_t ic = sm_warp_scan(n);
        const unsigned long long is = sm_warp_scan(n * w);
        const uint32_t hit = __ballot_sync(0xffffffffu, n && there(c + ic, s + is));
        if (lane == __ffs(hit) - 1) tell(at, n, w, s + is - n * w, c + ic - n);
    };
    // Moves on to a window (the usual one is there already).
    auto count_window = [&](uint32_t to) {
        window = to;
        sm_sync<C>();  // nobody reads the counts any more
        clear();
        each_group([&](uint4 v) {
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
                const int bin = sm_bin(sm_half(v, k), to);
                if (bin >= 0) atomicAdd(&hist[bin], 1);  // (sm_place is itself there)
            }
        });
        sm_sync<C>();
    };
    // Every value in falling order: visit() behind each window's scan, until it says so.
    if (usual) scan(0, 0);
    auto sweep = [&](auto &&visit) {
        if (usual) {
            visit();
            return;
        }
        uint32_t c = 0;
        unsigned long long s = 0;
        for (uint32_t i = 0; i < SM_WINDOWS; ++i) {
            count_window(i);
            scan(c, s);
            if (visit()) return;
            c += cw, s += sw;
        }
    };

    // ---- the weights of the k first, and of those with a weight of at least min_p
    uint32_t total = 0;
    unsigned long long mass = 0, high = 0;
    sweep([&] {
        if (k_of)
            find(cb < k_of && k_of <= cb + cnt, [&](uint32_t c, unsigned long long) { return c >= k_of; },
                 [&](uint32_t, uint32_t, unsigned long long w, unsigned long long s, uint32_t c) {
                     sh.top_k = s + (k_of - c) * w;
                 });
        total += cw, mass += sw, high += hw;
        return false;
    });
    if (k_of && k_of < total) {
        __syncthreads();
        mass = sh.top_k;
    }
    // ---- the kept candidates: of the k first, those with less than top_p of their weights before them, and min_p themselves.
    // Each leaves a prefix of the order, so the least sum is the shortest one's; the first candidate stays.
    unsigned long long kept = min(mass, high);
    if (!(p >= 1.f)) {
        const unsigned long long share = __double2ull_ru(fmax((double)p, 0.0) * (double)mass);  // (at most mass)
        if (share) {
            sweep([&] {
                find(sb < share && share <= sb + sum, [&](uint32_t, unsigned long long s) { return s >= share; },
                     [&](uint32_t, uint32_t, unsigned long long w, unsigned long long s, uint32_t) {
                         sh.top_p = s + (share - s + w - 1) / w * w;
                     });
                return false;
            });
            __syncthreads();
            kept = min(kept, sh.top_p);
        } else {
            kept = 0;
        }
    }
    kept = max(kept, (unsigned long long)unit);

    // ---- the token's value, and which of its occurrences
    const unsigned long long target = greedy ? 0 : (unsigned long long)((double)fminf(fmaxf(u, 0.f), 0x1.fffffep-1f) * (double)kept);  // (NaN: 0)
    sweep([&] {
        find(sb <= target && target < sb + sum, [&](uint32_t, unsigned long long s) { return s > target; },
             [&](uint32_t bin, uint32_t n, unsigned long long w, unsigned long long s, uint32_t) {
                 sh.bin = bin;
                 sh.nth = greedy ? n - 1 : (uint32_t)((target - s) / w);
                 sh.found = 1;
                 if (a.probs && rank == 0) a.probs[row] = greedy ? 1.f : (float)((double)w / (double)kept);
             });
        __syncthreads();
        return sh.found != 0;
    });

    // ---- its place: the CTA that counted it, the warp, the group
    const uint32_t bin = sh.bin;
    uint32_t nth = sh.nth;
    bool mine = false;
    for (int c = 0; c < C; ++c) {
        const uint32_t here = sm_get32(&hist[sm_place(bin, window)], c);
        if (nth < here) {
            mine = c == (int)rank;
            break;
        }
        nth -= here;
    }
    if constexpr (C > 1) tc::cluster_sync();  // no CTA ends while its counters are read
    if (!mine) return;
    const uint32_t twice = (__float_as_uint(sm_bin_value(bin, window)) >> 16) * 0x10001u;
    auto equal8 = [&](const uint4 &v) {  // element 2 k in bit k, 2 k + 1 in bit 16 + k
        return (sm_eq2(v.x, twice) & 0x10001u) | (sm_eq2(v.y, twice) & 0x20002u) | (sm_eq2(v.z, twice) & 0x40004u) |
               (sm_eq2(v.w, twice) & 0x80008u);
    };
    const uint4 nothing = make_uint4(SM_NONE, SM_NONE, SM_NONE, SM_NONE);
    // the part that holds it in 16 runs, one a warp, until a run is short
    uint32_t lo = g0, hi = g1;
    while (hi - lo > 128) {
        const uint32_t run = (hi - lo + SM_WARPS - 1) / SM_WARPS, w0 = min(lo + warp * run, hi), w1 = min(w0 + run, hi);
        uint32_t m = 0;
        for (uint32_t g = w0 + lane; g < w1; g += 32 * SM_LOOK) {
            uint4 v[SM_LOOK];
#pragma unroll
            for (int i = 0; i < SM_LOOK; ++i) v[i] = g + 32 * i < w1 ? x.group(g + 32 * i) : nothing;
#pragma unroll
            for (int i = 0; i < SM_LOOK; ++i) m += __popc(equal8(v[i]));
        }
        m = __reduce_add_sync(0xffffffffu, m);
        __syncthreads();
        if (lane == 0) sh.wcount[warp] = m;
        __syncthreads();
        int i = 0;
        for (; i < SM_WARPS - 1 && nth >= sh.wcount[i]; ++i) nth -= sh.wcount[i];
        lo = min(lo + i * run, hi);
        hi = min(lo + run, hi);
    }
    if (warp != 0) return;
    for (uint32_t g = lo; g < hi; g += 32) {
        const uint32_t bits = g + lane < hi ? equal8(x.group(g + lane)) : 0, y = __popc(bits), incl = sm_warp_scan(y);
        if (nth >= incl - y && nth < incl) {
            uint32_t left = nth - (incl - y), e = 0;
            for (;; ++e)  // elements in order
                if (bits >> (e & 1 ? 16 + e / 2 : e / 2) & 1 && left-- == 0) break;
            a.tokens[row] = 8 * (g + lane) + e - x.skew;
        }
        const uint32_t all = __shfl_sync(0xffffffffu, incl, 31);
        if (nth < all) return;
        nth -= all;
    }
}

template <int C>
static int launch_sample_ctas(SampleArgs a, uint32_t groups, cudaStream_t st) {
    a.part = (groups + C - 1) / C;
    if (cudaFuncSetAttribute(sample_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, SmCfg<C>::BYTES) != cudaSuccess) return -3;
    return launch_pdl(sample_kernel<C>, dim3(a.rows * C), dim3(SM_THREADS), SmCfg<C>::BYTES, st, C, a);
}

// Whether the current device holds `rows` clusters of C CTAs at once (a cluster lies within a group of SMs, so they are fewer
// than the SMs' room by itself); asked once per device and size.
template <int C>
static bool sample_fits(uint32_t rows) {
    static int known[64];  // 1 + the clusters, written with the same value by every thread that finds 0
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    int n = __atomic_load_n(&known[dev], __ATOMIC_RELAXED);
    if (!n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(C);
        cfg.blockDim = dim3(SM_THREADS);
        cfg.dynamicSmemBytes = SmCfg<C>::BYTES;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = C;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaFuncSetAttribute(sample_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, SmCfg<C>::BYTES) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&clusters, sample_kernel<C>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            clusters = 0;
        }
        n = 1 + clusters;
        __atomic_store_n(&known[dev], n, __ATOMIC_RELAXED);
    }
    return rows <= (uint32_t)(n - 1);
}

int launch_sample(SampleArgs a, cudaStream_t st) {
    const uint32_t groups = (a.vocab + 7 + 7) / 8;
    a.unit = __builtin_clz(a.vocab) + 31;  // 63 - bits of the vocabulary: the sums stay below 2^63
    const uint32_t most = (groups + 511) / 512;  // (a CTA has work for its threads)
    if (most >= 8 && sample_fits<8>(a.rows)) return launch_sample_ctas<8>(a, groups, st);
    if (most >= 4 && sample_fits<4>(a.rows)) return launch_sample_ctas<4>(a, groups, st);
    if (most >= 2 && sample_fits<2>(a.rows)) return launch_sample_ctas<2>(a, groups, st);
    return launch_sample_ctas<1>(a, groups, st);
}

}  // namespace qb
