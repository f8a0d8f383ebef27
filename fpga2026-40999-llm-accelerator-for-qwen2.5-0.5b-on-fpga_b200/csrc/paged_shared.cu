// Attention of one token per sequence where groups of sequences share their
// first tokens: the group's prefix is read from its first sequence's pages, the
// rest from each sequence's own.
//
// Mathematics, per (row, query head), P the group's prefix, over keys j < len:
//   x_j = log2(e) scale q.k_j,  p_j = 2^(x_j - m),  ctx = sum p_j v_j / sum p_j
// where key j < P is the first sequence's and key j >= P the row's own.
#include "kernels.h"
#include "paged.cuh"

namespace qb {

// One warp per (row, query head), a lane has DIM / 32 neighbouring dims.
template <bool KV8, int DIM>
__global__ void __launch_bounds__(128) paged_shared_kernel(PagedSharedArgs a) {
    constexpr int PER = DIM / 32;
    const int lane = threadIdx.x & 31;
    const uint64_t n = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint32_t row = (uint32_t)(n / a.qh), h = (uint32_t)(n % a.qh), kvh = h / (a.qh / a.c.hkv);
    if (row >= a.rows || row >= a.starts[a.n] || row < a.starts[0]) return;
    uint32_t g = 0, g1 = a.n;  // starts[g] <= row < starts[g1]
    while (g1 - g > 1) {
        const uint32_t mid = (g + g1) / 2;
        if (a.starts[mid] <= row) g = mid; else g1 = mid;
    }
    const uint32_t head = a.starts[g], seq = a.seqs ? a.seqs[row] : row, seq0 = a.seqs ? a.seqs[head] : head;
    const int len = paged_length(a.c, seq), P = min((int)min(a.prefix[g], 0x7fffffffu), paged_length(a.c, seq0));
    float q[PER], o[PER], m = -INFINITY, l = 0.f;
    for (int i = 0; i < PER; ++i) {
        q[i] = bf2f(a.q[row * a.q_stride + (uint64_t)h * DIM + lane * PER + i]);
        o[i] = 0.f;
    }
    const float fac = a.scale * 1.44269504f;
    for (int j = 0; j < len; ++j) {
        const uint32_t page = a.c.table[(uint64_t)(j < P ? seq0 : seq) * a.c.max_pages + (j >> a.c.tshift)];
        if (page >= a.c.pages) continue;
        const uint64_t r = paged_row(a.c, page, kvh) + (j & ((1 << a.c.tshift) - 1));
        float k[PER], v[PER], x = 0.f;
        for (int i = 0; i < PER; ++i) {
            const uint64_t e = r * DIM + lane * PER + i;
            if constexpr (KV8) {
                k[i] = (float)reinterpret_cast<const int8_t *>(a.c.k)[e];
                v[i] = (float)reinterpret_cast<const int8_t *>(a.c.v)[e] * a.c.vs[r];
            } else {
                k[i] = bf2f(reinterpret_cast<const uint16_t *>(a.c.k)[e]);
                v[i] = bf2f(reinterpret_cast<const uint16_t *>(a.c.v)[e]);
            }
            x = fmaf(q[i], k[i], x);
        }
        x = warp_sum(x) * fac;
        if constexpr (KV8) x *= a.c.ks[r];
        const float top = fmaxf(m, x), f = m == top ? 1.f : exp2f(m - top), p = exp2f(x - top);
        m = top;
        l = l * f + p;
        for (int i = 0; i < PER; ++i) o[i] = o[i] * f + p * v[i];
    }
    for (int i = 0; i < PER; ++i)
        a.ctx[row * a.ctx_stride + (uint64_t)h * DIM + lane * PER + i] = f2bf(l == 0.f ? 0.f : o[i] / l);
}

size_t paged_shared_ws(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 256; }

int launch_paged_shared(const PagedSharedArgs &a, void *, cudaStream_t st) {
    auto *kernel = a.format == QWEN_B200_KV8 ? (a.dim == 64 ? paged_shared_kernel<true, 64> : paged_shared_kernel<true, 128>)
                                             : (a.dim == 64 ? paged_shared_kernel<false, 64> : paged_shared_kernel<false, 128>);
    const uint64_t warps = (uint64_t)a.rows * a.qh;
    if ((warps + 3) / 4 >= 1ull << 31) return -1;
    kernel<<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(a);
    return QB_LAUNCH_CHECK();
}

}  // namespace qb
