// Attention over the paged KV cache, one warp per (row, query head): the
// scores, the running maximum and sum of the softmax and the context in fp32,
// lane l holding dims l, l + 32, ..
#include "paged.cuh"

namespace qb {

template <bool KV8, int DIM>
__global__ void __launch_bounds__(128) paged_attn_kernel(PagedAttnArgs a) {
    constexpr int N = DIM / 32;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (item >= (uint64_t)a.rows * a.qh) return;
    const uint32_t r = (uint32_t)(item / a.qh), h = (uint32_t)(item % a.qh), kvh = h / (a.qh / a.c.hkv);
    uint32_t i = r;
    int pos;
    if (a.starts) {  // the last sequence that starts at or before row r
        uint32_t lo = 0, hi = a.n;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (a.starts[mid + 1] <= r)
                lo = mid + 1;
            else
                hi = mid;
        }
        if (lo >= a.n || a.starts[lo] > r) return;
        i = lo;
        const uint32_t seq = a.seqs ? a.seqs[i] : i;
        pos = paged_length(a.c, seq) - (int)(min(a.starts[i + 1], a.rows) - r);
    } else {
        pos = paged_length(a.c, a.seqs ? a.seqs[i] : i) - 1;
    }
    const uint32_t seq = a.seqs ? a.seqs[i] : i;
    float q[N], o[N], m = -INFINITY, l = 0.f;
    for (int j = 0; j < N; ++j) {
        q[j] = bf2f(a.q[r * a.q_stride + h * DIM + lane + 32 * j]);
        o[j] = 0.f;
    }
    if (seq < a.c.seqs && pos >= 0) {
        const KeySpan ks = key_span(pos, a.window, a.sinks);
        for (int t = ks.first > 0 ? 0 : ks.low; t <= pos; ++t) {
            if (t >= ks.first && t < ks.low) t = ks.low;
            const uint32_t page = a.c.table[(uint64_t)seq * a.c.max_pages + (t >> a.c.tshift)];
            if (page >= a.c.pages) continue;
            const uint64_t row = paged_row(a.c, page, kvh) + (t & ((1 << a.c.tshift) - 1));
            float kx[N], vx[N], s = 0.f;
            for (int j = 0; j < N; ++j) {
                const uint64_t e = row * DIM + lane + 32 * j;
                if constexpr (KV8) {
                    kx[j] = (float)reinterpret_cast<const int8_t *>(a.c.k)[e] * a.c.ks[row];
                    vx[j] = (float)reinterpret_cast<const int8_t *>(a.c.v)[e] * a.c.vs[row];
                } else {
                    kx[j] = bf2f(reinterpret_cast<const uint16_t *>(a.c.k)[e]);
                    vx[j] = bf2f(reinterpret_cast<const uint16_t *>(a.c.v)[e]);
                }
                s += q[j] * kx[j];
            }
            s = warp_sum(s) * a.scale;
            const float m2 = fmaxf(m, s), f = expf(m - m2), p = expf(s - m2);
            l = l * f + p;
            for (int j = 0; j < N; ++j) o[j] = o[j] * f + p * vx[j];
            m = m2;
        }
    }
    for (int j = 0; j < N; ++j)
        a.ctx[r * a.ctx_stride + h * DIM + lane + 32 * j] = f2bf(l > 0.f ? o[j] / l : 0.f);
}

static int launch_attn(const PagedAttnArgs &a, cudaStream_t st) {
    const uint64_t blocks = ((uint64_t)a.rows * a.qh + 3) / 4;
    auto *kernel = a.format == QWEN_B200_KV8 ? (a.dim == 64 ? paged_attn_kernel<true, 64> : paged_attn_kernel<true, 128>)
                                             : (a.dim == 64 ? paged_attn_kernel<false, 64> : paged_attn_kernel<false, 128>);
    kernel<<<(unsigned)blocks, 128, 0, st>>>(a);
    return QB_LAUNCH_CHECK();
}

size_t paged_prefill_ws(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 256; }
int launch_paged_prefill(const PagedAttnArgs &a, const qwen_b200_paged_kv &, uint32_t, void *, cudaStream_t st) {
    return launch_attn(a, st);
}

}  // namespace qb
