// paged_attn.hip -- causal GQA attention of the new rows of a batch over a
// paged fp16 cache (rf_paged_attention_launch; the header states what it
// computes).  No counterpart in the reference, which runs one sequence over a
// contiguous cache.
#include <hip/hip_fp16.h>

#include <climits>
#include <cmath>

#include "paged_common.h"
#include "qk_common.h"

namespace rf {

// One workgroup a row and head.  D / 8 lanes hold a position, 8 dims a lane; a
// wave takes every fourth group of 512 / D positions with a running maximum,
// sum and output, and the waves' states are joined through LDS.
template <int D>
__global__ __launch_bounds__(256) void rf_paged_attn_rows_kernel(const rf_paged_attention a, const rf_paged_cache c) {
    constexpr int LPP = D / 8, PW = 64 / LPP, W = 4;
    __shared__ float part[W * PW][D + 2];
    const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (r >= a.q_start[a.num_seqs]) return;
    int lo = 0, hi = a.num_seqs;                 // q_start[lo] <= r < q_start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= r)
            lo = mid;
        else
            hi = mid;
    }
    const int n = a.q_start[lo + 1] - a.q_start[lo], i = r - a.q_start[lo];
    const int kv = (int)min((int64_t)max(a.kv_lens[lo], 0), (int64_t)a.max_blocks * c.page_size);
    const int p = kv - n + i, from = a.window > 0 ? max(0, p - a.window + 1) : 0;
    const int sub = lane % LPP, slot = wave * PW + lane / LPP;
    const int kvh = h / (a.num_heads / c.num_kv_heads);
    const int* table = a.block_tables + (int64_t)lo * a.max_blocks;

    float q[8], o[8] = {0, 0, 0, 0, 0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
    auto load8 = [](const uint16_t* s, float v[8]) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(s);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = half_bits_to_float(w[k] & 0xffffu);
            v[2 * k + 1] = half_bits_to_float(w[k] >> 16);
        }
    };
    load8(a.q + r * a.ld_q + (int64_t)h * D + 8 * sub, q);
    for (int t0 = from; t0 <= p; t0 += W * PW) {
        const int t = t0 + slot;
        const int page = t <= p ? table[t / c.page_size] : 0;
        const bool bad = page < 0 || page >= c.num_pages;
        const int64_t at = (int64_t)(bad ? 0 : page) * c.page_stride + (t % c.page_size) * c.row_stride +
                           kvh * c.head_stride + 8 * sub;
        float k[8] = {}, v[8] = {};
        if (t <= p) {
            load8(c.k + at, k);
            load8(c.v + at, v);
        }
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __fmaf_rn(q[e], k[e], s);
        s = xor_sum<LPP / 2, 1>(s) * a.scale;
        if (bad) s = NAN;
        if (t <= p) {
            const float mn = fmaxf(m, s), f = m == mn ? 1.0f : expf(m - mn), w = expf(s - mn);
            m = mn;
            l = l * f + w;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = o[e] * f + w * v[e];
        }
    }
    float* mine = part[slot];
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[8 * sub + e] = o[e];
    if (sub == 0) {
        mine[D] = m;
        mine[D + 1] = l;
    }
    __syncthreads();
    for (int d = tid; d < D; d += 256) {
        float mx = -INFINITY, sum = 0.0f, acc = 0.0f;
        for (int k = 0; k < W * PW; ++k) mx = fmaxf(mx, part[k][D]);
        for (int k = 0; k < W * PW; ++k) {
            const float lk = part[k][D + 1];
            if (lk == 0.0f) continue;            // nothing seen there
            const float f = part[k][D] == mx ? 1.0f : expf(part[k][D] - mx);
            sum += lk * f;
            acc += part[k][d] * f;
        }
        const float res = sum == 0.0f ? 0.0f : acc / sum;
        if (a.out_f32)
            static_cast<float*>(a.out)[r * a.ld_out + (int64_t)h * D + d] = res;
        else
            static_cast<uint16_t*>(a.out)[r * a.ld_out + (int64_t)h * D + d] = f16_bits_rn(res);
    }
}

}  // namespace rf

// ---- launchers -----------------------------------------------------------------------------

extern "C" size_t rf_paged_attention_workspace_bytes(int num_heads, int num_kv_heads, int head_dim) {
    if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
        (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return 0;
    return 16;
}

extern "C" hipError_t rf_paged_attention_launch(const rf_paged_attention* step, const rf_paged_cache* cache,
                                                hipStream_t stream) {
    if (step == nullptr || cache == nullptr) return hipErrorInvalidValue;
    const rf_paged_attention& a = *step;
    const rf_paged_cache& c = *cache;
    if (!rf::cache_ok(c) || a.num_seqs < 0 || a.rows < 0 || a.rows > (1 << 23) || a.max_blocks < 0 ||
        a.num_heads <= 0 || a.num_heads > 65535 || a.num_heads % c.num_kv_heads != 0 ||
        a.num_heads / c.num_kv_heads > 64 || a.window < 0 || !std::isfinite(a.scale))
        return hipErrorInvalidValue;
    if (a.rows == 0 || a.num_seqs == 0) return hipSuccess;
    const int64_t width = (int64_t)a.num_heads * c.head_dim;
    if (!a.q || !a.out || !a.block_tables || !a.q_start || !a.kv_lens || !a.workspace || a.ld_q % 8 || a.ld_out % 8 ||
        a.ld_q < width || a.ld_out < width ||
        ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) |
          reinterpret_cast<uintptr_t>(a.workspace)) & 15u) != 0 ||
        a.workspace_bytes < rf_paged_attention_workspace_bytes(a.num_heads, c.num_kv_heads, c.head_dim))
        return hipErrorInvalidValue;
    const dim3 grid(a.rows, a.num_heads), blk(256);
    switch (c.head_dim) {
    case 64: hipLaunchKernelGGL(rf::rf_paged_attn_rows_kernel<64>, grid, blk, 0, stream, a, c); break;
    case 128: hipLaunchKernelGGL(rf::rf_paged_attn_rows_kernel<128>, grid, blk, 0, stream, a, c); break;
    default: hipLaunchKernelGGL(rf::rf_paged_attn_rows_kernel<256>, grid, blk, 0, stream, a, c); break;
    }
    return hipGetLastError();
}
