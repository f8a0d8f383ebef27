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
// A cluster of up to 8 CTAs has a row. Each CTA counts its part of the row
// in its own shared memory (16-bit counters, two a word, 128 KB), then takes an
// equal part of the values, adds the CTAs' counts over distributed shared
// memory and scans; borders are exchanged by the CTA that finds them.
#include "kernels.h"
#include "qwen_b200.h"
#include "sample.cuh"
#include "tc05.cuh"

namespace qb {

constexpr int SM_THREADS = 1024, SM_WARPS = SM_THREADS / 32, SM_MAX_CTAS = 8;
constexpr uint32_t SM_CODES = 65536, SM_HIST = SM_CODES * 2;

// What a cluster's CTAs tell one another; written by their peers.
struct SmShared {
    uint32_t first[SM_MAX_CTAS];            // each CTA's lowest order (largest logit)
    uint32_t count[SM_MAX_CTAS];            // candidates of its values
    unsigned long long sum[SM_MAX_CTAS];    // and their weights
    unsigned long long kept[SM_MAX_CTAS];   // weights up to its last kept candidate
    unsigned long long top_k;               // weights of the k first
    uint32_t order, nth;                    // the token: nth occurrence of a value
    double weight;
    unsigned long long wsum[SM_WARPS];      // this CTA's own
    uint32_t wcount[SM_WARPS];
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
__device__ __forceinline__ uint4 sm_get128(const void *p, uint32_t rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(sm_remote(p, rank)));
    return v;
}
__device__ __forceinline__ uint32_t sm_get16(const void *p, uint32_t rank) {
    uint16_t v;
    asm volatile("ld.shared::cluster.u16 %0, [%1];" : "=h"(v) : "r"(sm_remote(p, rank)));
    return v;
}
// All CTAs of the row.
__device__ __forceinline__ void sm_sync(uint32_t ctas) {
    if (ctas > 1)
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
// Halfword of an order's counter: 16-byte groups permuted, so that threads with runs of 8 groups read without conflicts.
__device__ __forceinline__ uint32_t sm_slot(uint32_t order) {
    const uint32_t g = order >> 3;
    return ((g ^ ((g >> 3) & 7)) << 3) | (order & 7);
}

// The logits of a row in 16-byte groups by their addresses: group i has the elements 8 i - skew ..
struct SmRow {
    const uint16_t *base;  // the group that holds element 0
    uint32_t skew, vocab;
    __device__ __forceinline__ uint4 group(uint32_t i) const {
        const uint32_t lo = 8 * i;
        if (lo >= skew && lo + 8 <= skew + vocab) return *reinterpret_cast<const uint4 *>(base + lo);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t e = lo + k;
            const uint32_t b = e >= skew && e < skew + vocab ? base[e] : 0xff80u;  // -infinity
            w[k >> 1] = k & 1 ? w[k >> 1] | b << 16 : b;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
__device__ __forceinline__ uint32_t sm_half(const uint4 &v, int k) {
    const uint32_t w = k < 4 ? (k < 2 ? v.x : v.y) : (k < 6 ? v.z : v.w);
    return k & 1 ? w >> 16 : w & 0xffffu;
}

__global__ void __launch_bounds__(SM_THREADS, 1) sample_kernel(SampleArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ SmShared sh;
    uint32_t *hist = reinterpret_cast<uint32_t *>(smem);
    const uint32_t C = a.ctas, rank = C > 1 ? sm_rank() : 0, row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits + row * a.stride);
    SmRow x;
    x.base = reinterpret_cast<const uint16_t *>(at & ~(uintptr_t)15);
    x.skew = (uint32_t)(at & 15) / 2;
    x.vocab = a.vocab;
    const uint32_t groups = (x.skew + a.vocab + 7) / 8, g0 = min(rank * a.part, groups), g1 = min(g0 + a.part, groups);

    // ---- this CTA's part of the row, counted
    for (int i = tid; i < (int)(SM_HIST / 16); i += SM_THREADS) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint32_t first = 0xffffu;
    for (uint32_t g = g0 + tid; g < g1; g += SM_THREADS) {
        const uint4 v = x.group(g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t d = sm_order(sm_half(v, k));
            if (sm_counts(d)) {
                const uint32_t s = sm_slot(d);
                atomicAdd(&hist[s >> 1], 1u << (16 * (s & 1)));
                first = min(first, d);
            }
        }
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.wcount[warp] = first;
    __syncthreads();
    if (warp == 0) {
        first = __reduce_min_sync(0xffffffffu, sh.wcount[lane]);
        if (lane < (int)C) sm_put32(&sh.first[rank], lane, first);
    }
    sm_sync(C);
    first = 0xffffu;
    for (uint32_t c = 0; c < C; ++c) first = min(first, sh.first[c]);
    if (first == 0xffffu) {  // no candidate
        if (rank == 0 && tid == 0) {
            a.tokens[row] = QWEN_B200_NO_TOKEN;
            if (a.probs) a.probs[row] = 0.f;
        }
        return;  // (no CTA reads another's memory any more)
    }

    // ---- counts and weights of the values from the rank's first on, GROUPS x 8 of them a thread
    const float temperature = a.temperature ? a.temperature[row] : 1.f;
    const bool greedy = !(temperature > 0.f);
    const double T = temperature, top = sm_value(first);
    const double unit = ldexp(1.0, a.unit);  // weights are whole numbers of 1 / unit
    const uint32_t per = SM_CODES / C / SM_THREADS, d0 = rank * (SM_CODES / C) + tid * per;  // per: 8 to 64
    auto weight = [&](uint32_t d) {
        const double l = sm_value(d);
        return l == top ? 1.0 : greedy ? 0.0 : exp((l - top) / T);
    };
    auto counts = [&](uint32_t d, uint32_t (&n)[8]) {  // of the 8 values from d on
#pragma unroll
        for (int k = 0; k < 8; ++k) n[k] = 0;
        for (uint32_t c = 0; c < C; ++c) {
            const uint4 v = C > 1 ? sm_get128(smem + 2 * sm_slot(d), c) : *reinterpret_cast<uint4 *>(smem + 2 * sm_slot(d));
#pragma unroll
            for (int k = 0; k < 8; ++k) n[k] += sm_half(v, k);
        }
    };
    uint32_t cnt = 0;
    unsigned long long sum = 0;
    for (uint32_t d = d0; d < d0 + per; d += 8) {
        uint32_t n[8];
        counts(d, n);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (n[k]) {
                cnt += n[k];
                sum += n[k] * (unsigned long long)__double2ull_rn(weight(d + k) * unit);
            }
    }
    // exclusive prefixes over the CTA, then over the cluster
    uint32_t ic = cnt;
    unsigned long long is = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t yc = __shfl_up_sync(0xffffffffu, ic, o);
        const unsigned long long ys = __shfl_up_sync(0xffffffffu, is, o);
        if (lane >= o) ic += yc, is += ys;
    }
    if (lane == 31) sh.wcount[warp] = ic, sh.wsum[warp] = is;
    __syncthreads();
    uint32_t cb = ic - cnt, call = 0;
    unsigned long long sb = is - sum, sall = 0;
    for (int i = 0; i < SM_WARPS; ++i) {
        if (i < warp) cb += sh.wcount[i], sb += sh.wsum[i];
        call += sh.wcount[i];
        sall += sh.wsum[i];
    }
    if (tid < (int)C) {
        sm_put32(&sh.count[rank], tid, call);
        sm_put64(&sh.sum[rank], tid, sall);
    }
    sm_sync(C);
    uint32_t total = 0;
    unsigned long long mass = 0;
    for (uint32_t c = 0; c < C; ++c) {
        if (c < rank) cb += sh.count[c], sb += sh.sum[c];
        total += sh.count[c];
        mass += sh.sum[c];
    }

    // ---- the weights of the k first
    const uint32_t k_of = a.top_k && !greedy ? a.top_k[row] : 0, k_first = k_of ? min(k_of, total) : total;
    if (k_first < total) {
        if (cb < k_first && k_first <= cb + cnt) {
            uint32_t left = k_first - cb;
            unsigned long long s = sb;
            for (uint32_t d = d0; left && d < d0 + per; d += 8) {
                uint32_t n[8];
                counts(d, n);
                for (int k = 0; k < 8 && left; ++k) {
                    const uint32_t m = min(n[k], left);
                    if (m) s += m * (unsigned long long)__double2ull_rn(weight(d + k) * unit);
                    left -= m;
                }
            }
            for (uint32_t c = 0; c < C; ++c) sm_put64(&sh.top_k, c, s);
        }
        sm_sync(C);
        mass = sh.top_k;
    }
    // ---- the kept candidates: the first one, and those of the k first with less than top_p before them and min_p themselves
    const float p = a.top_p && !greedy ? a.top_p[row] : 1.f, least = a.min_p && !greedy ? a.min_p[row] : 0.f;
    const bool cut = !(p >= 1.f);
    const unsigned long long share = cut ? __double2ull_ru(fmax((double)p, 0.0) * (double)mass) : 0;
    unsigned long long kept = 0;  // weights up to this thread's last kept one
    auto walk = [&](auto &&visit) {  // (order, weight, kept candidates, weights before them)
        uint32_t i = cb;
        unsigned long long s = sb;
        for (uint32_t d = d0; d < d0 + per && i < k_first; d += 8) {
            uint32_t n[8];
            counts(d, n);
            for (int k = 0; k < 8 && i < k_first; ++k) {
                if (!n[k]) continue;
                const double w = weight(d + k);
                const unsigned long long wi = __double2ull_rn(w * unit);
                uint32_t m = min(n[k], k_first - i);
                if (cut) {
                    if (s >= share)
                        m = 0;
                    else if (wi) {
                        const unsigned long long fit = (share - s + wi - 1) / wi;
                        m = (uint32_t)min((unsigned long long)m, fit);
                    }
                }
                if (!(w >= least)) m = 0;
                if (i == 0) m = max(m, 1u);
                if (m && visit(d + k, w, wi, m, s)) return;
                i += n[k];
                s += n[k] * wi;
            }
        }
    };
    if (cnt) walk([&](uint32_t, double, unsigned long long wi, uint32_t m, unsigned long long s) {
        kept = s + m * wi;
        return false;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, kept, o);
        kept = max(kept, y);
    }
    __syncthreads();
    if (lane == 0) sh.wsum[warp] = kept;
    __syncthreads();
    if (tid < (int)C) {
        for (int i = 0; i < SM_WARPS; ++i) kept = max(kept, sh.wsum[i]);
        sm_put64(&sh.kept[rank], tid, kept);
    }
    sm_sync(C);
    kept = 0;
    for (uint32_t c = 0; c < C; ++c) kept = max(kept, sh.kept[c]);

    // ---- the token's value, and which of its occurrences
    const float u = fminf(fmaxf(a.u[row], 0.f), 0x1.fffffep-1f);  // (NaN: 0)
    const unsigned long long target = greedy ? 0 : (unsigned long long)((double)u * (double)kept);
    if (cnt && sb <= target)
        walk([&](uint32_t d, double w, unsigned long long wi, uint32_t m, unsigned long long s) {
            if (target < s || target >= s + m * wi) return false;
            const uint32_t nth = greedy ? m - 1 : (uint32_t)((target - s) / wi);
            const double prob = greedy ? 1.0 : w * unit / (double)kept;
            for (uint32_t c = 0; c < C; ++c) {
                sm_put32(&sh.order, c, d);
                sm_put32(&sh.nth, c, nth);
            }
            if (a.probs) a.probs[row] = (float)prob;
            return true;
        });
    sm_sync(C);

    // ---- its place: the CTA that counted it, the warp, the group
    const uint32_t order = sh.order;
    uint32_t nth = sh.nth;
    bool mine = false;
    for (uint32_t c = 0; c < C; ++c) {
        const uint32_t here = sm_get16(smem + 2 * sm_slot(order), c);
        if (nth < here) {
            mine = c == rank;
            break;
        }
        nth -= here;
    }
    if (mine) {
        const uint32_t per_warp = (g1 - g0 + SM_WARPS - 1) / SM_WARPS, w0 = min(g0 + warp * per_warp, g1), w1 = min(w0 + per_warp, g1);
        auto matches = [&](uint32_t g) {
            uint32_t bits = 0;
            if (g < w1) {
                const uint4 v = x.group(g);
#pragma unroll
                for (int k = 0; k < 8; ++k) bits |= (uint32_t)(sm_order(sm_half(v, k)) == order) << k;
            }
            return bits;
        };
        uint32_t n = 0;
        for (uint32_t g = w0; g < w1; g += 32) n += __popc(matches(g + lane));
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) sh.wcount[warp] = n;
        __syncthreads();  // (the whole CTA is here)
        for (int i = 0; i < warp; ++i) {
            const uint32_t m = sh.wcount[i];
            nth = nth < m ? 0xffffffffu : nth - m;  // an earlier warp has it
            if (nth == 0xffffffffu) break;
        }
        if (nth < sh.wcount[warp])
            for (uint32_t g = w0; g < w1; g += 32) {
                const uint32_t bits = matches(g + lane), m = __popc(bits);
                uint32_t incl = m;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += y;
                }
                if (nth >= incl - m && nth < incl)
                    a.tokens[row] = 8 * (g + lane) + __fns(bits, 0, nth - (incl - m) + 1) - x.skew;
                const uint32_t all = __shfl_sync(0xffffffffu, incl, 31);
                if (nth < all) break;
                nth -= all;
            }
    }
    if (C > 1) tc::cluster_sync();  // no CTA ends while its counters are read
}

int launch_sample(SampleArgs a, int sms, cudaStream_t st) {
    // 16-bit counters: at most 65528 elements a CTA
    const uint32_t groups = (a.vocab + 7 + 7) / 8;
    uint32_t ctas = 1;
    while (groups > ctas * 8191 || (ctas < SM_MAX_CTAS && a.rows * ctas * 2 <= (uint32_t)sms)) ctas *= 2;
    a.ctas = ctas;
    a.part = (groups + ctas - 1) / ctas;
    a.unit = __builtin_clz(a.vocab) + 31;  // 63 - bits of the vocabulary: the sums stay below 2^63
    if (cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SM_HIST) != cudaSuccess) return -3;
    return launch_pdl(sample_kernel, dim3(a.rows * ctas), dim3(SM_THREADS), SM_HIST, st, ctas, a);
}

}  // namespace qb
