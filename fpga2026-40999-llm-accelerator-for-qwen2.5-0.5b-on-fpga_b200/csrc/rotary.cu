// Rotary positions: the table of angles (host), rotation of heads, and the
// append of rotated keys to the paged cache.
//
// Mathematics: pair i of a head at position p turns by the angle a = p f_i:
//   y1 = x1 cos a - x2 sin a,  y2 = x2 cos a + x1 sin a,
// pairs (i, i + rotated / 2) or (2 i, 2 i + 1); dims from `rotated` on stay.
// Each product and each sum is rounded to fp32 (no fma), the result once to
// bf16, so the fused append gives the bits of the two calls that it replaces.
// cos and sin come from a table: an angle of a far position needs 64 bits
// (65536 rad in fp32 is off by 2^-9), too many for the kernel.
#include <float.h>
#include <math.h>

#include "paged.cuh"

namespace qb {

// A thread has one item of a head: 8 pairs, two runs of 8 dims; the items of
// a head behind the rotated dims are two neighbouring runs that stay.
struct RotItem {
    uint32_t d0, d1;  // first dims of the two runs
    uint32_t at;      // first of the 8 angles
    bool turn;
};
template <bool PAIRS>
__device__ __forceinline__ RotItem rot_item(uint32_t item, uint32_t rotated) {
    RotItem r;
    r.turn = 16 * item < rotated;
    r.at = 8 * item;
    r.d0 = PAIRS || !r.turn ? 16 * item : 8 * item;
    r.d1 = PAIRS || !r.turn ? 16 * item + 8 : 8 * item + rotated / 2;
    return r;
}

struct RotAngles {
    float c[8], s[8];
};
__device__ __forceinline__ void rot_angles(RotAngles &a, const float *row, uint32_t at, uint32_t rotated) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        const float4 c = __ldg(reinterpret_cast<const float4 *>(row + at + i));
        const float4 s = __ldg(reinterpret_cast<const float4 *>(row + rotated / 2 + at + i));
        a.c[i] = c.x, a.c[i + 1] = c.y, a.c[i + 2] = c.z, a.c[i + 3] = c.w;
        a.s[i] = s.x, a.s[i + 1] = s.y, a.s[i + 2] = s.z, a.s[i + 3] = s.w;
    }
}
__device__ __forceinline__ uint32_t rot_pack(float lo, float hi) { return (uint32_t)f2bf(lo) | ((uint32_t)f2bf(hi) << 16); }
__device__ __forceinline__ void rot_pair(float x1, float x2, float c, float s, float &y1, float &y2) {
    y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
    y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
}
// Turns an item in place, as bf16.
template <bool PAIRS>
__device__ __forceinline__ void rot_turn(uint4 &v0, uint4 &v1, const RotAngles &a) {
    uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    if constexpr (PAIRS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float y1, y2;
            rot_pair(bflo(w[i]), bfhi(w[i]), a.c[i], a.s[i], y1, y2);
            w[i] = rot_pack(y1, y2);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float p1, p2, q1, q2;
            rot_pair(bflo(w[i]), bflo(w[i + 4]), a.c[2 * i], a.s[2 * i], p1, p2);
            rot_pair(bfhi(w[i]), bfhi(w[i + 4]), a.c[2 * i + 1], a.s[2 * i + 1], q1, q2);
            w[i] = rot_pack(p1, q1);
            w[i + 4] = rot_pack(p2, q2);
        }
    }
    v0 = make_uint4(w[0], w[1], w[2], w[3]);
    v1 = make_uint4(w[4], w[5], w[6], w[7]);
}

// ---------------------------------------------------------------- rotation of heads
// A thread has one item of RT_HEADS heads of a row: their loads are in flight together
// and the angles are read once for them. Bound by HBM: 32768 rows of 40 heads x 128,
// half of each turned in pairs, 103 us on the device (672 MB, the copy rate); two
// heads a thread 105 us. 64 rows of 16 heads x 64 3.9 us.
constexpr int RT_THREADS = 128, RT_HEADS = 4;
template <bool PAIRS>
__global__ void __launch_bounds__(RT_THREADS)
    rotary_kernel(RotaryView t, const uint16_t *x, uint64_t x_stride, uint32_t heads, uint32_t dim, uint32_t rows,
                  const uint32_t *__restrict__ positions, uint16_t *out, uint64_t out_stride) {
    const uint32_t items = dim / 16;
    const uint64_t n = (uint64_t)blockIdx.x * RT_THREADS + threadIdx.x;
    const uint32_t row = (uint32_t)(n / items), item = (uint32_t)(n % items);
    if (row >= rows) return;
    const uint32_t h0 = blockIdx.y * RT_HEADS, count = min(heads - h0, (uint32_t)RT_HEADS);
    const RotItem r = rot_item<PAIRS>(item, t.rotated);
    const uint32_t pos = positions[row];
    uint4 v[RT_HEADS][2];
#pragma unroll
    for (int i = 0; i < RT_HEADS; ++i) {
        const uint16_t *p = x + row * x_stride + (uint64_t)(h0 + (i < (int)count ? i : 0)) * dim;
        v[i][0] = *reinterpret_cast<const uint4 *>(p + r.d0);
        v[i][1] = *reinterpret_cast<const uint4 *>(p + r.d1);
    }
    if (pos >= t.positions) return;
    RotAngles a;
    if (r.turn) rot_angles(a, t.table + (uint64_t)pos * t.rotated, r.at, t.rotated);
#pragma unroll
    for (int i = 0; i < RT_HEADS; ++i) {
        if (i >= (int)count) break;
        if (r.turn) rot_turn<PAIRS>(v[i][0], v[i][1], a);
        uint16_t *p = out + row * out_stride + (uint64_t)(h0 + i) * dim;
        *reinterpret_cast<uint4 *>(p + r.d0) = v[i][0];
        *reinterpret_cast<uint4 *>(p + r.d1) = v[i][1];
    }
}

int launch_rotary(const RotaryView &t, const uint16_t *x, uint64_t x_stride, uint32_t heads, uint32_t dim, uint32_t rows,
                  const uint32_t *positions, uint16_t *out, uint64_t out_stride, cudaStream_t st) {
    const uint64_t threads = (uint64_t)rows * (dim / 16);
    const dim3 grid((unsigned)((threads + RT_THREADS - 1) / RT_THREADS), (heads + RT_HEADS - 1) / RT_HEADS);
    auto *kernel = t.pairs ? rotary_kernel<true> : rotary_kernel<false>;
    kernel<<<grid, RT_THREADS, 0, st>>>(t, x, x_stride, heads, dim, rows, positions, out, out_stride);
    return QB_LAUNCH_CHECK();
}

// ---------------------------------------------------------------- rotated append
// blockIdx.y: up to AR_HEADS query heads, or some key or value heads. A thread has
// one item of them; the DIM / 16 threads of a head are neighbours and agree on its
// row. Bound by HBM for prompts and by the chain of sequence, length and page for
// single tokens: 12.8k rows of 32 + 8 + 8 heads x 128 bf16 52 us on the device (318 MB,
// 94 % of the copy rate), 7.4k rows of 14 + 2 + 2 x 64 KV8 10.7 us (33 MB), 64 rows 5.1 us.
// With two query heads a thread 54, 10.8 and 5.0 us, with seven 60, 13.1 and 6.3; KV8 keys
// two at a time 12.7 us (their divisions), bf16 ones one at a time 57 us.
constexpr int AR_THREADS = 128, AR_HEADS = 4;
template <bool KV8>
struct ArKv {
    static constexpr int HEADS = KV8 ? 1 : 4;
};
template <bool KV8, int DIM, bool PAIRS>
__global__ void __launch_bounds__(AR_THREADS) paged_append_rotary_kernel(PagedView c, RotaryView t, AppendRotary a) {
    constexpr uint32_t ITEMS = DIM / 16;
    const uint64_t n = (uint64_t)blockIdx.x * AR_THREADS + threadIdx.x;
    const uint32_t row = (uint32_t)(n / ITEMS), item = (uint32_t)(n % ITEMS);
    if (row >= a.rows) return;  // (a head's threads leave together)
    constexpr int KVH = ArKv<KV8>::HEADS;
    static_assert(KVH <= AR_HEADS, "v");
    const uint32_t nq = (a.q_heads + AR_HEADS - 1) / AR_HEADS, nk = (c.hkv + KVH - 1) / KVH, y = blockIdx.y;
    const bool is_q = y < nq, is_v = y >= nq + nk;
    const uint32_t head = is_q ? AR_HEADS * y : KVH * (y - nq - (is_v ? nk : 0));
    const int count = (int)(is_q ? min(a.q_heads - head, (uint32_t)AR_HEADS) : min(c.hkv - head, (uint32_t)KVH));
    const RotItem r = is_v ? RotItem{16 * item, 16 * item + 8, 0, false} : rot_item<PAIRS>(item, t.rotated);
    const uint32_t seq = a.seqs[row], pos = a.positions[row];
    const uint16_t *src = (is_q ? a.q + row * a.q_stride : (is_v ? a.v : a.k) + row * a.kv_stride) + head * DIM;
    uint4 v[AR_HEADS][2];
#pragma unroll
    for (int i = 0; i < AR_HEADS; ++i) {
        if (i >= count) break;
        v[i][0] = *reinterpret_cast<const uint4 *>(src + i * DIM + r.d0);
        v[i][1] = *reinterpret_cast<const uint4 *>(src + i * DIM + r.d1);
    }
    // (the angles do not wait for the page)
    RotAngles g;
    if (r.turn && pos < t.positions) rot_angles(g, t.table + (uint64_t)pos * t.rotated, r.at, t.rotated);
    uint32_t page = PG_NO_PAGE;
    if (pos < t.positions && pos < (uint32_t)paged_length(c, seq))
        page = c.table[(uint64_t)seq * c.max_pages + (pos >> c.tshift)];
    if (page >= c.pages) return;
    if (r.turn) {
#pragma unroll
        for (int i = 0; i < AR_HEADS; ++i)
            if (i < count) rot_turn<PAIRS>(v[i][0], v[i][1], g);
    }
    if (is_q) {
#pragma unroll
        for (int i = 0; i < AR_HEADS; ++i) {
            if (i >= count) break;
            uint16_t *p = a.q_out + row * a.q_out_stride + (head + i) * DIM;
            *reinterpret_cast<uint4 *>(p + r.d0) = v[i][0];
            *reinterpret_cast<uint4 *>(p + r.d1) = v[i][1];
        }
        return;
    }
    uint8_t *pool = const_cast<uint8_t *>(is_v ? c.v : c.k);
#pragma unroll
    for (int i = 0; i < KVH; ++i) {
        if (i >= count) break;
        const uint64_t dst = paged_row(c, page, head + i) + (pos & ((1u << c.tshift) - 1));
        if constexpr (!KV8) {
            *reinterpret_cast<uint4 *>(pool + (dst * DIM + r.d0) * 2) = v[i][0];
            *reinterpret_cast<uint4 *>(pool + (dst * DIM + r.d1) * 2) = v[i][1];
        } else {
            // the rule of paged_append_kernel, on the bf16 values
            const uint32_t w[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
            float x[16], amax = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[2 * j] = bflo(w[j]);
                x[2 * j + 1] = bfhi(w[j]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(x[j]));
            const uint32_t mates = ((1u << ITEMS) - 1) << (threadIdx.x & 31 & ~(ITEMS - 1));  // this head's threads
#pragma unroll
            for (int o = ITEMS / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mates, amax, o));
            const float s = __fdiv_rn(amax, 127.0f);
            uint32_t b[4] = {0u, 0u, 0u, 0u};
            if (s > 0.f) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int code = (int)fminf(fmaxf(rintf(__fdiv_rn(x[j], s)), -127.f), 127.f);
                    b[j >> 2] |= ((uint32_t)code & 0xffu) << (8 * (j & 3));
                }
            }
            *reinterpret_cast<uint2 *>(pool + dst * DIM + r.d0) = make_uint2(b[0], b[1]);
            *reinterpret_cast<uint2 *>(pool + dst * DIM + r.d1) = make_uint2(b[2], b[3]);
            if (item == 0) const_cast<float *>(is_v ? c.vs : c.ks)[dst] = s;
        }
    }
}

template <bool KV8, int DIM>
static int launch_append_rotary(const PagedView &c, const RotaryView &t, const AppendRotary &a, cudaStream_t st) {
    const uint64_t threads = (uint64_t)a.rows * (DIM / 16);
    const dim3 grid((unsigned)((threads + AR_THREADS - 1) / AR_THREADS), (a.q_heads + AR_HEADS - 1) / AR_HEADS + 2 * ((c.hkv + ArKv<KV8>::HEADS - 1) / ArKv<KV8>::HEADS));
    auto *kernel = t.pairs ? paged_append_rotary_kernel<KV8, DIM, true> : paged_append_rotary_kernel<KV8, DIM, false>;
    kernel<<<grid, AR_THREADS, 0, st>>>(c, t, a);
    return QB_LAUNCH_CHECK();
}

int launch_paged_append_rotary(const qwen_b200_paged_kv &kv, uint32_t layer, const RotaryView &t, const AppendRotary &a,
                               cudaStream_t st) {
    const PagedView c = paged_view(kv, layer);
    if (kv.format == QWEN_B200_KV8)
        return kv.head_dim == 64 ? launch_append_rotary<true, 64>(c, t, a, st) : launch_append_rotary<true, 128>(c, t, a, st);
    return kv.head_dim == 64 ? launch_append_rotary<false, 64>(c, t, a, st) : launch_append_rotary<false, 128>(c, t, a, st);
}

}  // namespace qb

// ---------------------------------------------------------------- the table (host)
extern "C" int qwen_b200_rotary_table(const qwen_b200_rotary_angles *a, uint32_t positions, float *table) {
    if (!a || !table || !positions || positions > QWEN_B200_ROTARY_POSITIONS) return QWEN_B200_EINVAL;
    const uint32_t rot = a->rotated, half = rot / 2;
    if (!rot || rot % 16 || rot > QWEN_B200_ROTARY_DIMS || a->scaling > QWEN_B200_ROTARY_YARN) return QWEN_B200_EINVAL;
    if (!(a->theta > 1.0) || !isfinite(a->theta) || !(a->size >= 0.0) || !isfinite(a->size)) return QWEN_B200_EINVAL;
    const double factor = a->scaling == QWEN_B200_ROTARY_PLAIN ? 1.0 : a->factor;
    if (!(factor > 0.0) || !isfinite(factor)) return QWEN_B200_EINVAL;
    double theta = a->theta, size = 1.0, freq[QWEN_B200_ROTARY_DIMS / 2];
    if (a->scaling == QWEN_B200_ROTARY_NTK) theta *= pow(factor, (double)rot / (rot - 2));
    if (!isfinite(theta) || !(theta > 0.0)) return QWEN_B200_EINVAL;
    for (uint32_t i = 0; i < half; ++i) freq[i] = pow(theta, -2.0 * i / rot);
    if (a->scaling == QWEN_B200_ROTARY_LINEAR)
        for (uint32_t i = 0; i < half; ++i) freq[i] /= factor;
    if (a->scaling == QWEN_B200_ROTARY_YARN) {
        if (!a->trained || !(a->fast > a->slow) || !(a->slow > 0.0) || !isfinite(a->fast)) return QWEN_B200_EINVAL;
        // the pair that turns n times in the positions of training: trained theta^(-2 i / rot) = 2 pi n
        auto pair_of = [&](double turns) { return rot * log(a->trained / (turns * 2 * M_PI)) / (2 * log(theta)); };
        const double low = fmax(floor(pair_of(a->fast)), 0.0), high = fmin(ceil(pair_of(a->slow)), rot - 1.0);
        for (uint32_t i = 0; i < half; ++i) {
            // (no pair turns as often as `slow` if the border lies at or in front of pair 0)
            const double ramp = high <= 0 ? 1.0 : fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
            freq[i] = freq[i] * (1 - ramp) + freq[i] / factor * ramp;
        }
        size = factor > 1.0 ? 0.1 * log(factor) + 1 : 1.0;
    }
    if (a->size > 0.0) size = a->size;
    if (!(size <= FLT_MAX)) return QWEN_B200_EINVAL;  // (the last position's angles and the size bound every entry)
    for (uint32_t i = 0; i < half; ++i)
        if (!isfinite((positions - 1.0) * freq[i])) return QWEN_B200_EINVAL;
#pragma omp parallel for
    for (int64_t p = 0; p < (int64_t)positions; ++p)
        for (uint32_t i = 0; i < half; ++i) {
            const double angle = (double)p * freq[i];
            table[p * rot + i] = (float)(cos(angle) * size);
            table[p * rot + half + i] = (float)(sin(angle) * size);
        }
    return QWEN_B200_OK;
}
