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
// The histogram has a window of 8192 values in shared memory. One window holds
// 0 and every magnitude in [2^-23, 2^8), which is all of a row in practice: what
// lies below it (masks such as -1e4 or the lowest value) has no weight and is left
// out. A row for which that does not hold goes through 8 windows of 8192 of the
// 65536 values instead, counted anew at each step (about ten times slower).
//
// A cluster of C CTAs has a row: each counts a part of it, then takes 8192 / C
// values, adds the CTAs' counts over distributed shared memory and scans;
// borders are exchanged by the CTA that finds them.
#include "kernels.h"
#include "qwen_b200.h"
#include "sample.cuh"
#include "tc05.cuh"

namespace qb {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_MAX_CTAS = 8;
constexpr uint32_t SM_BINS = 8192, SM_WINDOWS = 65536 / SM_BINS;
// The usual window: magnitudes from SM_LOW on (as bf16 bits), SM_SIDE of them on each side of 0.
constexpr uint32_t SM_LOW = 0x3400, SM_SIDE = 31 * 128;

// What a cluster's CTAs tell one another; written by their peers.
struct SmShared {
    uint32_t first[SM_MAX_CTAS];            // lowest order (largest logit) of each CTA's part
    uint32_t below[SM_MAX_CTAS];            // the same of its values below the usual window
    uint32_t odd[SM_MAX_CTAS];              // whether it has values that the window's two sides do not hold
    uint32_t count[SM_MAX_CTAS];            // candidates of its values
    unsigned long long sum[SM_MAX_CTAS];    // and their weights
    unsigned long long kept[SM_MAX_CTAS];   // weights up to its last kept candidate
    unsigned long long top_k;               // weights of the k first
    uint32_t bin, nth;                      // the token: nth occurrence of a value
    uint32_t found;                         // in this window + 1
    uint32_t wcount[SM_WARPS], wbelow[SM_WARPS], wodd;  // this CTA's own
    unsigned long long wsum[SM_WARPS];
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
__device__ __forceinline__ uint2 sm_get64(const void *p, uint32_t rank) {
    uint2 v;
    asm volatile("ld.shared::cluster.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(sm_remote(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t sm_get32(const void *p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sm_remote(p, rank)) : "memory");
    return v;
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
        const uint32_t t = mag - SM_LOW;
        if (t < SM_SIDE) return b & 0x8000u ? SM_SIDE + 1 + t : SM_SIDE - 1 - t;
        return mag == 0 ? (int)SM_SIDE : -1;
    }
    const uint32_t d = sm_order(b);
    return sm_counts(d) && d / SM_BINS == window ? (int)(d % SM_BINS) : -1;
}
__device__ __forceinline__ float sm_bin_value(uint32_t bin, uint32_t window) {
    if (window == SM_WINDOWS)
        return bf2f(bin < SM_SIDE ? SM_LOW + SM_SIDE - 1 - bin : bin == SM_SIDE ? 0u : 0x8000u | (SM_LOW + bin - SM_SIDE - 1));
    return sm_value(window * SM_BINS + bin);
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

template <int C>
__global__ void __launch_bounds__(SM_THREADS, C > 2 ? 2 : 1) sample_kernel(SampleArgs a) {
    constexpr int PER = SM_BINS / C / SM_THREADS;  // values of a thread
    __shared__ __align__(16) uint32_t hist[SM_BINS];
    __shared__ SmShared sh;
    const uint32_t rank = C > 1 ? sm_rank() : 0, row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits + row * a.stride);
    SmRow x;
    x.base = reinterpret_cast<const uint16_t *>(at & ~(uintptr_t)15);
    x.skew = (uint32_t)(at & 15) / 2;
    x.vocab = a.vocab;
    const uint32_t groups = (x.skew + a.vocab + 7) / 8, g0 = min(rank * a.part, groups), g1 = min(g0 + a.part, groups);

    // ---- this CTA's part of the row, counted in the usual window
    auto clear = [&] {
        for (uint32_t i = tid; i < SM_BINS / 4; i += SM_THREADS) reinterpret_cast<uint4 *>(hist)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    };
    if (tid == 0) sh.wodd = 0, sh.found = 0;
    clear();
    uint32_t first = 0xffffu, below = 0xffffu;
    bool odd = false;
    for (uint32_t g = g0 + tid; g < g1; g += SM_THREADS) {
        const uint4 v = x.group(g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t b = sm_half(v, k);
            const int bin = sm_bin(b, SM_WINDOWS);
            if (bin >= 0) {
                atomicAdd(&hist[bin], 1);
                first = min(first, (uint32_t)bin);
            } else {
                const uint32_t d = sm_order(b);
                if (sm_counts(d)) {
                    if (d > 0x8000u + SM_LOW) below = min(below, d); else odd = true;
                }
            }
        }
    }
    // (as orders: a bin of the window lies between 0x7fff - (SM_LOW + SM_SIDE - 1) and the values below it)
    if (first != 0xffffu) {
        const float v = sm_bin_value(first, SM_WINDOWS);
        first = sm_order(__float_as_uint(v) >> 16);
    }
    first = __reduce_min_sync(0xffffffffu, min(first, below));
    below = __reduce_min_sync(0xffffffffu, below);
    if (lane == 0) sh.wcount[warp] = first, sh.wbelow[warp] = below;
    if (odd) sh.wodd = 1;
    __syncthreads();
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
#pragma unroll
    for (int c = 0; c < C; ++c) {
        first = min(first, sh.first[c]);
        below = min(below, sh.below[c]);
        odd = c == 0 ? sh.odd[0] != 0 : odd || sh.odd[c] != 0;
    }

    const float temperature = a.temperature ? a.temperature[row] : 1.f;
    const bool greedy = !(temperature > 0.f);
    const double T = temperature, unit = ldexp(1.0, a.unit);  // weights are whole numbers of 1 / unit
    double top = 0.0;
    auto weight_of = [&](double l) { return l == top ? 1.0 : greedy ? 0.0 : exp((l - top) / T); };
    auto whole = [&](double w) { return (unsigned long long)__double2ull_rn(w * unit); };
    uint32_t window = SM_WINDOWS;
    if (odd) {  // the largest may be one of those: from its order, counted in the first windows
        window = 0;
    } else if (first == 0xffffu) {  // no candidate
        if (rank == 0 && tid == 0) {
            a.tokens[row] = QWEN_B200_NO_TOKEN;
            if (a.probs) a.probs[row] = 0.f;
        }
        return;  // (no CTA reads another's memory any more)
    } else {
        top = sm_value(first);
        if (below != 0xffffu && whole(weight_of(sm_value(below)))) window = 0;
    }
    const bool usual = window == SM_WINDOWS;

    // ---- the counts and weights of a window's values, PER neighbours a thread, and what is before them
    uint32_t n[PER], cb = 0, cnt = 0, cw = 0;              // before; of the thread; of the window
    unsigned long long w[PER], sb = 0, sum = 0, sw = 0;
    const uint32_t bin0 = rank * (SM_BINS / C) + tid * PER;
    auto scan = [&](uint32_t c_before, unsigned long long s_before) {
        cnt = 0, sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) n[j] = 0;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < PER; j += 2) {
                const uint2 v = C > 1 ? sm_get64(&hist[bin0 + j], c) : *reinterpret_cast<uint2 *>(&hist[bin0 + j]);
                n[j] += v.x;
                n[j + 1] += v.y;
            }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            w[j] = 0;
            if (n[j]) {
                w[j] = whole(weight_of(sm_bin_value(bin0 + j, window)));
                cnt += n[j];
                sum += n[j] * w[j];
            }
        }
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
        uint32_t call = 0;
        unsigned long long sall = 0;
        cb = c_before + ic - cnt, sb = s_before + is - sum;
#pragma unroll
        for (int i = 0; i < SM_WARPS; ++i) {
            const uint32_t y = sh.wcount[i];
            const unsigned long long z = sh.wsum[i];
            if (i < warp) cb += y, sb += z;
            call += y, sall += z;
        }
        if (tid < C) {
            sm_put32(&sh.count[rank], tid, call);
            sm_put64(&sh.sum[rank], tid, sall);
        }
        sm_sync<C>();
        cw = 0, sw = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c < (int)rank) cb += sh.count[c], sb += sh.sum[c];
            cw += sh.count[c];
            sw += sh.sum[c];
        }
    };
    // Moves on to a window (the usual one is there already).
    auto count_window = [&](uint32_t to) {
        window = to;
        sm_sync<C>();  // nobody reads the counts any more
        clear();
        for (uint32_t g = g0 + tid; g < g1; g += SM_THREADS) {
            const uint4 v = x.group(g);
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
                const int bin = sm_bin(sm_half(v, k), to);
                if (bin >= 0) atomicAdd(&hist[bin], 1);
            }
        }
        sm_sync<C>();
    };
    // Every value in falling order: visit() behind each window's scan, until it says so.
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
    if (usual) {
        scan(0, 0);
    } else {
        // the largest logit: the first value of the first window that has one
        first = 0xffffu;
        for (uint32_t i = 0; i < SM_WINDOWS && first == 0xffffu; ++i) {
            count_window(i);
            uint32_t f = 0xffffu;
            for (uint32_t j = tid; j < SM_BINS; j += SM_THREADS)
                for (int c = 0; c < C; ++c)
                    if (sm_get32(&hist[j], c)) f = min(f, i * SM_BINS + j);
            f = __reduce_min_sync(0xffffffffu, f);
            if (lane == 0) sh.wcount[warp] = f;
            __syncthreads();
            for (int k = 0; k < SM_WARPS; ++k) first = min(first, sh.wcount[k]);
            __syncthreads();
        }
        top = sm_value(first);
    }

    // ---- the weights of the k first
    const uint32_t k_of = a.top_k && !greedy ? a.top_k[row] : 0;
    uint32_t total = 0;
    unsigned long long mass = 0;
    sweep([&] {
        if (k_of && cb < k_of && k_of <= cb + cnt) {
            uint32_t left = k_of - cb;
            unsigned long long s = sb;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const uint32_t m = min(n[j], left);
                s += m * w[j];
                left -= m;
            }
            for (int c = 0; c < C; ++c) sm_put64(&sh.top_k, c, s);
        }
        total += cw;
        mass += sw;
        return false;
    });
    const uint32_t k_first = k_of ? min(k_of, total) : total;
    if (k_first < total) {
        sm_sync<C>();
        mass = sh.top_k;
    }
    // ---- the kept candidates: the first one, and those of the k first with less than top_p before them and min_p themselves
    const float p = a.top_p && !greedy ? a.top_p[row] : 1.f, least = a.min_p && !greedy ? a.min_p[row] : 0.f;
    const bool cut = !(p >= 1.f), floor = !(least <= 0.f);
    const unsigned long long share = cut ? __double2ull_ru(fmax((double)p, 0.0) * (double)mass) : 0;
    auto keep = [&](int j, uint32_t i, unsigned long long s) {  // of value j, whose first candidate is the i-th, with s before it
        uint32_t m = i < k_first ? min(n[j], k_first - i) : 0;
        if (cut && m) {
            if (s >= share)
                m = 0;
            else if (w[j])
                m = (uint32_t)min((unsigned long long)m, (share - s + w[j] - 1) / w[j]);
        }
        if (floor && m && !(weight_of(sm_bin_value(bin0 + j, window)) >= (double)least)) m = 0;
        return i == 0 && n[j] ? max(m, 1u) : m;
    };
    unsigned long long kept = mass;
    if (cut || floor) {
        kept = 0;
        sweep([&] {
            if (cnt) {
                uint32_t i = cb;
                unsigned long long s = sb;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const uint32_t m = keep(j, i, s);
                    if (m) kept = s + m * w[j];
                    i += n[j];
                    s += n[j] * w[j];
                }
            }
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
        if (tid < C) {
            for (int i = 0; i < SM_WARPS; ++i) kept = max(kept, sh.wsum[i]);
            sm_put64(&sh.kept[rank], tid, kept);
        }
        sm_sync<C>();
        kept = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) kept = max(kept, sh.kept[c]);
    }

    // ---- the token's value, and which of its occurrences
    const float u = fminf(fmaxf(a.u[row], 0.f), 0x1.fffffep-1f);  // (NaN: 0)
    const unsigned long long target = greedy ? 0 : (unsigned long long)((double)u * (double)kept);
    sweep([&] {
        if (cnt && sb <= target && target < sb + sum) {
            uint32_t i = cb;
            unsigned long long s = sb;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (target >= s && target < s + n[j] * w[j]) {
                    const uint32_t nth = greedy ? n[j] - 1 : (uint32_t)((target - s) / w[j]);
                    for (int c = 0; c < C; ++c) {
                        sm_put32(&sh.bin, c, bin0 + j);
                        sm_put32(&sh.nth, c, nth);
                        sm_put32(&sh.found, c, 1);
                    }
                    if (a.probs)
                        a.probs[row] = greedy ? 1.f : (float)(weight_of(sm_bin_value(bin0 + j, window)) * unit / (double)kept);
                }
                i += n[j];
                s += n[j] * w[j];
            }
        }
        sm_sync<C>();
        return sh.found != 0;
    });

    // ---- its place: the CTA that counted it, the warp, the group
    const uint32_t bin = sh.bin;
    uint32_t nth = sh.nth;
    bool mine = false;
    for (int c = 0; c < C; ++c) {
        const uint32_t here = sm_get32(&hist[bin], c);
        if (nth < here) {
            mine = c == (int)rank;
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
                for (int k = 0; k < 8; ++k) bits |= (uint32_t)(sm_bin(sm_half(v, k), window) == (int)bin) << k;
            }
            return bits;
        };
        uint32_t m = 0;
        for (uint32_t g = w0; g < w1; g += 32) m += __popc(matches(g + lane));
        m = __reduce_add_sync(0xffffffffu, m);
        if (lane == 0) sh.wcount[warp] = m;
        __syncthreads();  // (the whole CTA is here)
        for (int i = 0; i < warp; ++i) {
            const uint32_t y = sh.wcount[i];
            nth = nth < y ? 0xffffffffu : nth - y;  // an earlier warp has it
            if (nth == 0xffffffffu) break;
        }
        if (nth < sh.wcount[warp])
            for (uint32_t g = w0; g < w1; g += 32) {
                const uint32_t bits = matches(g + lane), y = __popc(bits);
                uint32_t incl = y;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t z = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += z;
                }
                if (nth >= incl - y && nth < incl)
                    a.tokens[row] = 8 * (g + lane) + __fns(bits, 0, nth - (incl - y) + 1) - x.skew;
                const uint32_t all = __shfl_sync(0xffffffffu, incl, 31);
                if (nth < all) break;
                nth -= all;
            }
    }
    if constexpr (C > 1) tc::cluster_sync();  // no CTA ends while its counters are read
}

template <int C>
static int launch_sample_ctas(SampleArgs a, uint32_t groups, cudaStream_t st) {
    a.part = (groups + C - 1) / C;
    return launch_pdl(sample_kernel<C>, dim3(a.rows * C), dim3(SM_THREADS), 0, st, C, a);
}

int launch_sample(SampleArgs a, int sms, cudaStream_t st) {
    const uint32_t groups = (a.vocab + 7 + 7) / 8;
    a.unit = __builtin_clz(a.vocab) + 31;  // 63 - bits of the vocabulary: the sums stay below 2^63
    const uint32_t want = (2 * (uint32_t)sms + a.rows - 1) / a.rows, most = (groups + 511) / 512;
    const uint32_t ctas = want < most ? want : most;
    if (ctas >= 8) return launch_sample_ctas<8>(a, groups, st);
    if (ctas >= 3 || (a.vocab > 32768 && most >= 4)) return launch_sample_ctas<4>(a, groups, st);
    if (ctas == 2) return launch_sample_ctas<2>(a, groups, st);
    return launch_sample_ctas<1>(a, groups, st);
}

}  // namespace qb
