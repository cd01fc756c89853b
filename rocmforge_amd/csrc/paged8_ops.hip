// paged8_ops.hip -- the rotary step into 8-bit pages, and reading them back.
// What each computes is declared in the header.  No counterpart in the reference.
#include <hip/hip_fp16.h>

#include <algorithm>
#include <climits>

#include "paged8.h"

namespace rf {

// ---- the rotary step into the pages --------------------------------------------------------
//
// A block's exponent needs all its new rows, so a workgroup takes whole runs of rows that
// share a block: those that start among 16 rows, at most 31 of them (a prompt's 16, or
// 16 requests' single tokens).  D / 8 lanes a row, 8 elements a lane, the rows of a head at
// once and one head after the other; a lane's four pairs turn by the same angles in all
// heads, so it takes their cosines once.  A run's largest value meets through LDS.
constexpr int kRunRows = 16;                     // first rows of runs a workgroup looks at

template <int D, bool NEOX>
__global__ __launch_bounds__(256) void rf_paged_rope8_kernel(const rf_paged_rope s, const rf_paged_cache8 c, int per) {
    constexpr int LPH = D / 8, RPP = 256 / LPH, PASSES = (2 * kRunRows - 1 + RPP - 1) / RPP;
    __shared__ float tops[2][2 * kRunRows];      // a row's largest finite value
    __shared__ int olds[2][2 * kRunRows];        // the exponent before, at a run's first row
    const int tid = threadIdx.x, lane = tid & 63, u = tid % LPH;
    const int bsh = block_shift(c), slots = c.num_pages * c.page_size;
    const int r0 = kRunRows * blockIdx.x;
    // a run: rows one behind the other with rising slots of one block
    const int at = r0 + lane;
    const bool there = lane < 3 * kRunRows && at < s.rows;
    const int now = there ? s.slots[at] : -1, before = there && at > 0 ? s.slots[at - 1] : -1;
    const bool lead = !there || (unsigned)now >= (unsigned)slots || (unsigned)before >= (unsigned)slots ||
                      now <= before || (now >> bsh) != (before >> bsh);
    const uint64_t leads = __ballot(lead);
    if ((leads & 0xffffu) == 0) return;
    const int a0 = __builtin_ctzll(leads), first = r0 + a0;
    const int n = min(kRunRows + __builtin_ctzll(leads >> kRunRows), s.rows - r0) - a0;
    if (n <= 0) return;

    const int half = s.rot_dim / 2, heads = s.num_heads + 2 * c.num_kv_heads;
    const bool turned = u < s.rot_dim / 8;
    const int e0 = NEOX && turned ? 4 * u : 8 * u, e1 = NEOX && turned ? half + 4 * u : e0 + 4;
    const int h0 = blockIdx.y * per, h1 = min(h0 + per, heads);
    int row[PASSES], slot[PASSES], run[PASSES], end[PASSES];     // run, end: rows of this row's run, from `first` on
    float4 a[PASSES], b[PASSES];
    auto load = [&](int h, int p) {
        const int64_t r = first + row[p];
        const float* src = h < s.num_heads ? s.q + r * s.ld_q + (int64_t)h * D
                           : h < s.num_heads + c.num_kv_heads
                               ? s.k + r * s.ld_k + (int64_t)(h - s.num_heads) * D
                               : s.v + r * s.ld_v + (int64_t)(h - s.num_heads - c.num_kv_heads) * D;
        a[p] = *reinterpret_cast<const float4*>(src + e0);
        b[p] = *reinterpret_cast<const float4*>(src + e1);
    };
    float2 cs[PASSES][4];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        row[p] = RPP * p + tid / LPH;
        slot[p] = -1;
        if (row[p] >= n) continue;
        const int r = first + row[p], bit = a0 + row[p];
        slot[p] = s.slots[r];
        if ((unsigned)slot[p] >= (unsigned)slots) {
            slot[p] = -1;
            continue;
        }
        load(h0, p);
        run[p] = 63 - __builtin_clzll(leads & ((2ull << bit) - 1)) - a0;
        end[p] = min(bit + 1 + __builtin_ctzll(leads >> (bit + 1)) - a0, n);
        if (turned)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double turn = (double)s.positions[r] * s.turns[4 * u + i];
                float sn, co;
                sincospif(2.0f * (float)(turn - rint(turn)), &sn, &co);
                cs[p][i] = make_float2(co * s.attn_factor, sn * s.attn_factor);
            }
    }
    for (int h = h0; h < h1; ++h) {
        const bool is_q = h < s.num_heads, is_v = h >= s.num_heads + c.num_kv_heads;
        const int kvh = is_v ? h - s.num_heads - c.num_kv_heads : h - s.num_heads;
        const float* w = is_v ? nullptr : is_q ? s.q_norm : s.k_norm;
        uint8_t* codes = (is_v ? c.v : c.k) + (is_q ? 0 : kvh) * c.head_stride;
        uint8_t* scales = (is_v ? c.v_scale : c.k_scale) + (is_q ? 0 : kvh);
        const int buf = h & 1;
        float y[PASSES][8];
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            if (slot[p] < 0) continue;
            float x[8] = {a[p].x, a[p].y, a[p].z, a[p].w, b[p].x, b[p].y, b[p].z, b[p].w};
            if (h + 1 < h1) load(h + 1, p);
            // (every lane of a row takes the same way, and rows do not share lanes)
            if (w != nullptr) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = __fmaf_rn(x[i], x[i], ss);
                ss = xor_sum<LPH / 2, 1>(ss);
                const float inv = 1.0f / sqrtf(ss * (1.0f / D) + s.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[(i < 4 ? e0 : e1 - 4) + i];
            }
            if (!is_v && turned) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 t = cs[p][i];
                    constexpr int P = NEOX ? 1 : 2, Q = NEOX ? 4 : 1;
                    const float f = x[P * i], g = x[P * i + Q];
                    x[P * i] = __fmaf_rn(f, t.x, -(g * t.y));
                    x[P * i + Q] = __fmaf_rn(f, t.y, g * t.x);
                }
            }
            if (is_q) {
                uint16_t* dst = s.q16 + (int64_t)(first + row[p]) * s.ld_q16 + (int64_t)h * D;
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[i] = (uint32_t)f16_bits_rn(x[2 * i]) | ((uint32_t)f16_bits_rn(x[2 * i + 1]) << 16);
                *reinterpret_cast<uint2*>(dst + e0) = make_uint2(o[0], o[1]);
                *reinterpret_cast<uint2*>(dst + e1) = make_uint2(o[2], o[3]);
                continue;
            }
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[p][i] = x[i];
                top = fmaxf(top, nan_unless_finite(x[i]) == 0.0f ? fabsf(x[i]) : 0.0f);
            }
            top = xor_max<LPH / 2, 1>(top);
            if (u == 0) {
                tops[buf][row[p]] = top;
                // (one lane reads it, and writes it again below)
                if (run[p] == row[p])
                    olds[buf][row[p]] = scale_byte(scales[(int64_t)(slot[p] >> bsh) * c.num_kv_heads]);
            }
        }
        if (is_q) continue;
        __syncthreads();                         // (of the other buffer's readers all have passed the barrier before)
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            if (slot[p] < 0) continue;
            float top = 0.0f;
            for (int i = run[p]; i < end[p]; ++i) top = fmaxf(top, tops[buf][i]);
            // the place in the block of the run's first row: rows of a run need not be all of its rows
            const int from = s.slots[first + run[p]] & ((1 << bsh) - 1);
            const int old = olds[buf][run[p]], fit = scale_for(top), e = from == 0 ? fit : max(fit, old);
            const float by = pow2_of(254 - e);
            uint8_t* dst = codes + (int64_t)(slot[p] / c.page_size) * c.page_stride +
                           (int64_t)(slot[p] % c.page_size) * c.row_stride;
            const float lo[4] = {y[p][0], y[p][1], y[p][2], y[p][3]}, hi[4] = {y[p][4], y[p][5], y[p][6], y[p][7]};
            *reinterpret_cast<uint32_t*>(dst + e0) = codes_of(lo, by);
            *reinterpret_cast<uint32_t*>(dst + e1) = codes_of(hi, by);
            if (run[p] == row[p]) {
                if (from > 0 && e > old) {
                    const float less = pow2_of(127 + old - e);
                    for (int i = 1; i <= from; ++i) {
                        uint8_t* was = dst - i * c.row_stride;
                        uint32_t* w0 = reinterpret_cast<uint32_t*>(was + e0);
                        uint32_t* w1 = reinterpret_cast<uint32_t*>(was + e1);
                        *w0 = recoded(*w0, less);
                        *w1 = recoded(*w1, less);
                    }
                }
                if (u == 0) scales[(int64_t)(slot[p] >> bsh) * c.num_kv_heads] = (uint8_t)e;
            }
        }
    }
}

// ---- reading back ----------------------------------------------------------------------------
//
// A workgroup takes kReadRows rows: where they lie is found once, and then 8 codes a
// thread become 16 bytes.  Memory-bound, one byte in and two out a value.
constexpr int kReadRows = 16;

__global__ __launch_bounds__(256) void rf_paged_read8_kernel(const rf_paged_read s, const rf_paged_cache8 c, uint32_t inv) {
    __shared__ int64_t codes_at[kReadRows], scales_at[kReadRows];
    const int tid = threadIdx.x, lane = tid & 63, r0 = kReadRows * blockIdx.x;
    const int bsh = block_shift(c), dsh = __ffs(c.head_dim) - 4;         // pieces of 8 a head
    const int pieces = c.num_kv_heads << dsh;
    if (tid < 64) {
        // the last request that starts at or before row r0, by 64 probes at a time
        int lo = 0, len = s.num_seqs;
        while (len > 1) {
            const int step = (len + 63) >> 6, i = lane * step;
            const uint64_t below = __ballot(i < len && s.row_start[lo + min(i, len - 1)] <= r0);
            const int k = max(__popcll(below) - 1, 0) * step;
            lo += k;
            len = min(step, len - k);
        }
        if (lane < kReadRows) {
            const int r = r0 + lane;
            int b = lo;
            while (b < s.num_seqs && s.row_start[b + 1] <= r) ++b;
            int64_t at = -1;
            if (r < s.rows && b < s.num_seqs && s.row_start[b] <= r) {
                const int64_t pos = (int64_t)(s.first != nullptr ? s.first[b] : 0) + (r - max(s.row_start[b], 0));
                const int psh = __ffs(c.page_size) - 1;
                if (pos >= 0 && pos < (int64_t)s.max_blocks * c.page_size) {
                    const int page = s.block_tables[(int64_t)b * s.max_blocks + (pos >> psh)];
                    const int row = (int)pos & (c.page_size - 1);
                    if ((unsigned)page < (unsigned)c.num_pages) {
                        at = page * c.page_stride + row * c.row_stride;
                        scales_at[lane] = scale_at(c, page, row, bsh);
                    }
                }
            }
            codes_at[lane] = at;
        }
    }
    __syncthreads();
    constexpr int U = 4;
    for (int i0 = tid; i0 < kReadRows * pieces; i0 += 256 * U) {
        u32x2 w[U][2];
        int byte[U][2];
        int64_t to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u;
            const int r = min(inv ? (int)__umulhi((uint32_t)i, inv) : i / pieces, kReadRows - 1), piece = i - r * pieces;
            const int64_t at = i < kReadRows * pieces ? codes_at[r] : -1;
            const int h = piece >> dsh, d = 8 * (piece & ((1 << dsh) - 1));
            to[u] = at < 0 ? -1 : (int64_t)(r0 + r) * s.ld_out + (int64_t)h * c.head_dim + d;
            if (at >= 0)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    w[u][v] = *reinterpret_cast<const u32x2*>((v ? c.v : c.k) + at + h * c.head_stride + d);
                    byte[u][v] = (v ? c.v_scale : c.k_scale)[scales_at[r] + h];
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (to[u] < 0) continue;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                uint16_t* out = v ? s.v : s.k;
                if (out == nullptr) continue;
                const float scale = pow2_of(scale_byte(byte[u][v]));
                u32x4 o;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    o[2 * k] = __builtin_bit_cast(uint32_t, two_of<false>(w[u][v][k], scale));
                    o[2 * k + 1] = __builtin_bit_cast(uint32_t, two_of<true>(w[u][v][k], scale));
                }
                *reinterpret_cast<u32x4*>(out + to[u]) = o;
            }
        }
    }
}

}  // namespace rf

// ---- launchers -----------------------------------------------------------------------------

static bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

extern "C" hipError_t rf_paged_rope_write8_launch(const rf_paged_rope* step, const rf_paged_cache8* cache,
                                                  hipStream_t stream) {
    if (step == nullptr || cache == nullptr) return hipErrorInvalidValue;
    const rf_paged_rope& s = *step;
    if (!rf::cache8_ok(*cache) || s.rows < 0 || s.rows > (1 << 23) || s.num_heads <= 0 || s.num_heads > 65535 ||
        s.rot_dim < 0 || s.rot_dim > cache->head_dim || s.rot_dim % 8)
        return hipErrorInvalidValue;
    if (s.rows == 0) return hipSuccess;
    if (!s.q || !s.k || !s.v || !s.q16 || !s.positions || !s.slots || (s.rot_dim > 0 && !s.turns))
        return hipErrorInvalidValue;
    if (!aligned(s.q, 16) || !aligned(s.k, 16) || !aligned(s.v, 16) || !aligned(s.q16, 16) || !aligned(s.q_norm, 16) ||
        !aligned(s.k_norm, 16) || !aligned(s.turns, 8) || s.ld_q % 4 || s.ld_k % 4 || s.ld_v % 4 || s.ld_q16 % 8 ||
        s.ld_q < 0 || s.ld_k < 0 || s.ld_v < 0 || s.ld_q16 < (int64_t)s.num_heads * cache->head_dim)
        return hipErrorInvalidValue;
    const int heads = s.num_heads + 2 * cache->num_kv_heads, chunks = (s.rows + rf::kRunRows - 1) / rf::kRunRows;
    // as many heads a workgroup as leave eight of them a CU, so that cosines are shared
    const int64_t most = 8ll * rf::device_cu_count();
    const int per = (int)std::min<int64_t>(std::max<int64_t>(((int64_t)chunks * heads + most - 1) / most, (heads + 65534) / 65535), heads);
    const dim3 grid(chunks, (heads + per - 1) / per), blk(256);
#define ROPE_GO(D)                                                                                         \
    if (s.neox)                                                                                            \
        hipLaunchKernelGGL((rf::rf_paged_rope8_kernel<D, true>), grid, blk, 0, stream, s, *cache, per);    \
    else                                                                                                   \
        hipLaunchKernelGGL((rf::rf_paged_rope8_kernel<D, false>), grid, blk, 0, stream, s, *cache, per);
    switch (cache->head_dim) {
    case 64: ROPE_GO(64) break;
    case 128: ROPE_GO(128) break;
    default: ROPE_GO(256) break;
    }
#undef ROPE_GO
    return hipGetLastError();
}

extern "C" hipError_t rf_paged_read8_launch(const rf_paged_read* read, const rf_paged_cache8* cache, hipStream_t stream) {
    if (read == nullptr || cache == nullptr) return hipErrorInvalidValue;
    const rf_paged_read& s = *read;
    if (!rf::cache8_ok(*cache) || s.rows < 0 || s.rows > (1 << 27) || s.num_seqs < 0 || s.max_blocks < 0)
        return hipErrorInvalidValue;
    if (s.rows == 0 || s.num_seqs == 0 || (!s.k && !s.v)) return hipSuccess;
    const int64_t width = (int64_t)cache->num_kv_heads * cache->head_dim;
    if (!s.block_tables || !s.row_start || !aligned(s.k, 16) || !aligned(s.v, 16) || s.ld_out < width || s.ld_out % 8)
        return hipErrorInvalidValue;
    // (i / pieces is the high word of i inv while 16 pieces^2 and what a pass reads past the end stay below 2^32)
    const uint32_t pieces = (uint32_t)(width / 8);
    const uint32_t inv = pieces <= 8192 ? (uint32_t)(((1ull << 32) + pieces - 1) / pieces) : 0;
    hipLaunchKernelGGL(rf::rf_paged_read8_kernel, dim3((unsigned)((s.rows + rf::kReadRows - 1) / rf::kReadRows)), dim3(256),
                       0, stream, s, *cache, inv);
    return hipGetLastError();
}
