// paged8_ops.hip -- the rotary step into 8-bit pages, and reading them back.
// What each computes is declared in the header.  No counterpart in the reference.
#include <hip/hip_fp16.h>

#include <algorithm>
#include <climits>

#include "paged8.h"

namespace rf {

// ---- the rotary step into the pages --------------------------------------------------------
//
// Queries go a row at a time, their loads two heads ahead (4000 rows of 32 + 16 heads 36 us, 3.9 TB/s; a head ahead,
// under the barriers of keys and values, 39).  Of keys and values a block's exponent needs all its new rows,
// so a workgroup takes whole runs of rows that share a block: those that start among 16 rows (32 at head_dim 64), up
// to 15 more with the last one's (a prompt's 16, or 16 requests' single tokens).  D / 8 lanes a row, 8 elements a
// lane, the rows of a head at once and one head after the other; a lane's four pairs turn by the same angles in all
// heads, so it takes their cosines once.  A run's largest value meets through LDS.  Where the runs have more rows than
// the threads take, the last one goes by itself.
constexpr int kRunRows = 16;                     // the most rows of a run
template <int D>
constexpr int rope8_threads() { return D == 256 ? 512 : 256; }
template <int D>
constexpr int start_rows() { return rope8_threads<D>() / (D / 8); }

// A lane's eight elements of a row, of any head: from e0 on and from e1 on four each, which make up pairs.
template <int D, bool NEOX>
struct Rope8 {
    static constexpr int LPH = D / 8;
    int u, e0, e1;
    bool turned;
    float2 cs[4];                                // of its four pairs
    __device__ __forceinline__ explicit Rope8(const rf_paged_rope& s) : u(threadIdx.x % LPH), turned(u < s.rot_dim / 8) {
        e0 = NEOX && turned ? 4 * u : 8 * u;
        e1 = NEOX && turned ? s.rot_dim / 2 + 4 * u : e0 + 4;
    }
    __device__ __forceinline__ void angles(const rf_paged_rope& s, int r) {
        if (!turned) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double turn = (double)s.positions[r] * s.turns[4 * u + i];
            float sn, co;
            sincospif(2.0f * (float)(turn - rint(turn)), &sn, &co);
            cs[i] = make_float2(co * s.attn_factor, sn * s.attn_factor);
        }
    }
    // (every lane of a row takes the same way, and rows do not share lanes)
    __device__ __forceinline__ void norm(float (&x)[8], float4 w0, float4 w1, float eps) const {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __fmaf_rn(x[i], x[i], ss);
        ss = xor_sum<LPH / 2, 1>(ss);
        const float inv = 1.0f / sqrtf(ss * (1.0f / D) + eps);
        const float by[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * by[i];
    }
    __device__ __forceinline__ void turn(float (&x)[8]) const {
        if (!turned) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            constexpr int P = NEOX ? 1 : 2, Q = NEOX ? 4 : 1;
            const float f = x[P * i], g = x[P * i + Q];
            x[P * i] = __fmaf_rn(f, cs[i].x, -(g * cs[i].y));
            x[P * i + Q] = __fmaf_rn(f, cs[i].y, g * cs[i].x);
        }
    }
};

// The query heads [h0, h1) of the workgroup's rows.
template <int D, bool NEOX>
__device__ __forceinline__ void rope8_queries(const rf_paged_rope& s, int slots, int h0, int h1) {
    constexpr int AHEAD = 2;                     // heads whose loads are on their way
    Rope8<D, NEOX> t(s);
    const int r = start_rows<D>() * blockIdx.x + threadIdx.x / (D / 8);
    if (r >= s.rows || (unsigned)s.slots[r] >= (unsigned)slots) return;
    const float* src = s.q + (int64_t)r * s.ld_q;
    uint16_t* dst = s.q16 + (int64_t)r * s.ld_q16;
    float4 a[AHEAD], b[AHEAD];
    auto load = [&](int h, int k) {
        const float* from = src + (int64_t)min(h, h1 - 1) * D;
        a[k] = *reinterpret_cast<const float4*>(from + t.e0);
        b[k] = *reinterpret_cast<const float4*>(from + t.e1);
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) load(h0 + k, k);
    float4 w0 = {1, 1, 1, 1}, w1 = w0;           // the norm's weights
    if (s.q_norm != nullptr) {
        w0 = *reinterpret_cast<const float4*>(s.q_norm + t.e0);
        w1 = *reinterpret_cast<const float4*>(s.q_norm + t.e1);
    }
    t.angles(s, r);
    for (int h = h0; h < h1; h += AHEAD)
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (h + k >= h1) return;
            float x[8] = {a[k].x, a[k].y, a[k].z, a[k].w, b[k].x, b[k].y, b[k].z, b[k].w};
            load(h + k + AHEAD, k);
            if (s.q_norm != nullptr) t.norm(x, w0, w1, s.eps);
            t.turn(x);
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] = (uint32_t)f16_bits_rn(x[2 * i]) | ((uint32_t)f16_bits_rn(x[2 * i + 1]) << 16);
            uint16_t* to = dst + (int64_t)(h + k) * D;
            *reinterpret_cast<uint2*>(to + t.e0) = make_uint2(o[0], o[1]);
            *reinterpret_cast<uint2*>(to + t.e1) = make_uint2(o[2], o[3]);
        }
}

// per: heads a workgroup; the grid's rows are those of q, then of k and v.
template <int D, bool NEOX>
__global__ __launch_bounds__(rope8_threads<D>(), 5)
void rf_paged_rope8_kernel(const rf_paged_rope s, const rf_paged_cache8 c, int per) {
    constexpr int ROWS = start_rows<D>(), LPH = D / 8;
    static_assert(ROWS >= kRunRows && ROWS + kRunRows < 64, "the threads take a run, a wave's ballot all rows");
    __shared__ float tops[2][ROWS];              // a row's largest finite value
    __shared__ int olds[2][ROWS];                // the exponent before, at a run's first row
    const int slots = c.num_pages * c.page_size, q_groups = (s.num_heads + per - 1) / per;
    if ((int)blockIdx.y < q_groups) {
        const int h0 = blockIdx.y * per;
        return rope8_queries<D, NEOX>(s, slots, h0, min(h0 + per, s.num_heads));
    }
    const int tid = threadIdx.x, lane = tid & 63;
    const int bsh = block_shift(c), psh = __ffs(c.page_size) - 1;
    const int r0 = ROWS * blockIdx.x;
    // a run: rows one behind the other with rising slots of one block
    const int at = r0 + lane;
    const bool there = lane < ROWS + kRunRows && at < s.rows;
    const int now = there ? s.slots[at] : -1, before = there && at > 0 ? s.slots[at - 1] : -1;
    const bool lead = !there || (unsigned)now >= (unsigned)slots || (unsigned)before >= (unsigned)slots ||
                      now <= before || (now >> bsh) != (before >> bsh);
    const uint64_t leads = __ballot(lead), mine = leads & ((1ull << ROWS) - 1);
    if (mine == 0) return;
    const int a0 = __builtin_ctzll(mine), last = 63 - __builtin_clzll(mine);
    const int a2 = min(ROWS + __builtin_ctzll(leads >> ROWS), s.rows - r0);      // (rows from r0 on)
    if (a2 <= a0) return;
    const int a1 = a2 - a0 <= ROWS ? a2 : last;

    Rope8<D, NEOX> t(s);
    const int u = t.u, nkv = c.num_kv_heads;     // heads: k's, then v's
    const int h0 = ((int)blockIdx.y - q_groups) * per, h1 = min(h0 + per, 2 * nkv);
    int buf = 0;
    for (int begin = a0, n = a1 - a0; n > 0; begin += n, n = a2 - begin) {
        const int first = r0 + begin;
        const int row = tid / LPH;               // from `first` on, as run and end, its run's
        int slot = -1, run = 0, end = 0, from = 0;       // from: place in the block of the run's first row
        float4 a, b;
        auto load = [&](int h) {
            const int64_t r = first + row;
            const float* src = h < nkv ? s.k + r * s.ld_k + (int64_t)h * D : s.v + r * s.ld_v + (int64_t)(h - nkv) * D;
            a = *reinterpret_cast<const float4*>(src + t.e0);
            b = *reinterpret_cast<const float4*>(src + t.e1);
        };
        const int r = first + row, bit = begin + row;
        if (row < n) slot = s.slots[r];
        const bool live = (unsigned)slot < (unsigned)slots;
        if (live) {
            load(h0);
            run = 63 - __builtin_clzll(leads & ((2ull << bit) - 1)) - begin;
            end = min(bit + 1 + __builtin_ctzll(leads >> (bit + 1)) - begin, n);
            from = s.slots[first + run] & ((1 << bsh) - 1);
            if (h0 < nkv) t.angles(s, r);
        }
        float4 w0 = {1, 1, 1, 1}, w1 = w0;       // the norm's weights
        if (s.k_norm != nullptr && h0 < nkv) {
            w0 = *reinterpret_cast<const float4*>(s.k_norm + t.e0);
            w1 = *reinterpret_cast<const float4*>(s.k_norm + t.e1);
        }
        for (int h = h0; h < h1; ++h) {
            const bool is_v = h >= nkv;
            const int kvh = is_v ? h - nkv : h;
            uint8_t* codes = (is_v ? c.v : c.k) + kvh * c.head_stride;
            uint8_t* scales = (is_v ? c.v_scale : c.k_scale) + kvh;
            float x[8];
            if (live) {
                const float loaded[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = loaded[i];
                if (h + 1 < h1) load(h + 1);
                if (!is_v) {
                    if (s.k_norm != nullptr) t.norm(x, w0, w1, s.eps);
                    t.turn(x);
                }
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, nan_unless_finite(x[i]) == 0.0f ? fabsf(x[i]) : 0.0f);
                top = xor_max<LPH / 2, 1>(top);
                if (u == 0) {
                    tops[buf][row] = top;
                    // (one lane reads it, and writes it again below)
                    if (run == row) olds[buf][row] = scale_byte(scales[(int64_t)(slot >> bsh) * nkv]);
                }
            }
            __syncthreads();                     // (of the other buffer's readers all have passed the barrier before)
            if (live) {
                float top = 0.0f;
                for (int i = run + u; i < end; i += LPH) top = fmaxf(top, tops[buf][i]);
                top = xor_max<LPH / 2, 1>(top);
                const int old = olds[buf][run], fit = scale_for(top), e = from == 0 ? fit : max(fit, old);
                const float by = pow2_of(254 - e);
                uint8_t* dst = codes + (int64_t)(slot >> psh) * c.page_stride +
                               (int64_t)(slot & (c.page_size - 1)) * c.row_stride;
                const float lo[4] = {x[0], x[1], x[2], x[3]}, hi[4] = {x[4], x[5], x[6], x[7]};
                *reinterpret_cast<uint32_t*>(dst + t.e0) = codes_of(lo, by);
                *reinterpret_cast<uint32_t*>(dst + t.e1) = codes_of(hi, by);
                if (run == row) {
                    if (from > 0 && e > old) {
                        // the block's rows before, two at a time (more cost registers, and so the prompts time)
                        const float less = pow2_of(127 + old - e);
                        constexpr int AT_ONCE = 2;
                        for (int i0 = 1; i0 <= from; i0 += AT_ONCE) {
                            uint32_t was[AT_ONCE][2];
#pragma unroll
                            for (int i = 0; i < AT_ONCE; ++i) {
                                const uint8_t* src = dst - min(i0 + i, from) * c.row_stride;
                                was[i][0] = *reinterpret_cast<const uint32_t*>(src + t.e0);
                                was[i][1] = *reinterpret_cast<const uint32_t*>(src + t.e1);
                            }
#pragma unroll
                            for (int i = 0; i < AT_ONCE; ++i) {
                                if (i0 + i > from) continue;
                                uint8_t* to = dst - (i0 + i) * c.row_stride;
                                *reinterpret_cast<uint32_t*>(to + t.e0) = recoded(was[i][0], less);
                                *reinterpret_cast<uint32_t*>(to + t.e1) = recoded(was[i][1], less);
                            }
                        }
                    }
                    if (u == 0) scales[(int64_t)(slot >> bsh) * nkv] = (uint8_t)e;
                }
            }
            buf ^= 1;
        }
    }
}

// ---- reading back ----------------------------------------------------------------------------
//
// A workgroup takes a few rows: where they lie is found once, and then 8 codes a
// thread become 16 bytes.  Memory-bound, one byte in and two out a value.
constexpr int kReadRows = 4;                     // at most

__global__ __launch_bounds__(256) void rf_paged_read8_kernel(const rf_paged_read s, const rf_paged_cache8 c, int per,
                                                            uint32_t inv) {
    __shared__ int64_t codes_at[kReadRows], scales_at[kReadRows];
    const int tid = threadIdx.x, lane = tid & 63, r0 = per * (int)(blockIdx.x + blockIdx.y * gridDim.x);
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
        // and how many more start by each of the others, 64 starts at a time
        int b = lo;
        for (int b0 = lo + 1;; b0 += 64) {
            const int start = lane <= s.num_seqs - b0 ? s.row_start[b0 + lane] : INT_MAX;
            for (int i = 0; i < per; ++i) {
                const int more = __popcll(__ballot(start <= r0 + i));
                if (lane == i) b += more;
            }
            if (__builtin_amdgcn_readlane(start, 63) >= r0 + per) break;
        }
        if (lane < per) {
            const int r = r0 + lane;
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
    // (what is not asked for is not read: its loads are the other's again)
    const uint8_t* from[2] = {s.k ? c.k : c.v, s.v ? c.v : c.k};
    const uint8_t* bytes[2] = {s.k ? c.k_scale : c.v_scale, s.v ? c.v_scale : c.k_scale};
    for (int i0 = tid; i0 < per * pieces; i0 += 256 * U) {
        u32x2 w[U][2];
        int byte[U][2];
        int64_t to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u;
            const int r = min(inv ? (int)__umulhi((uint32_t)i, inv) : i / pieces, per - 1), piece = i - r * pieces;
            const int64_t at = i < per * pieces ? codes_at[r] : -1;
            const int h = piece >> dsh, d = 8 * (piece & ((1 << dsh) - 1));
            to[u] = at < 0 ? -1 : (int64_t)(r0 + r) * s.ld_out + (int64_t)h * c.head_dim + d;
            if (at >= 0)
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    w[u][v] = *reinterpret_cast<const u32x2*>(from[v] + at + h * c.head_stride + d);
                    byte[u][v] = bytes[v][scales_at[r] + h];
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
    const int heads = s.num_heads + 2 * cache->num_kv_heads, starts = cache->head_dim == 64 ? rf::start_rows<64>() : rf::start_rows<128>();
    const int chunks = (s.rows + starts - 1) / starts;
    // as many heads a workgroup as leave some sixteen of them a CU, so that cosines are shared: 4000 rows
    // of 48 heads and their read back 42.0 us, with eight a CU 46.7; 1500 rows 19.3, with twenty 21.4
    const int64_t most = 16ll * rf::device_cu_count();
    const int per = (int)std::min<int64_t>(std::max<int64_t>(((int64_t)chunks * heads + most - 1) / most, (heads + 65532) / 65533), heads);
    const dim3 grid(chunks, (s.num_heads + per - 1) / per + (2 * cache->num_kv_heads + per - 1) / per);
#define ROPE_GO(D)                                                                                         \
    if (s.neox)                                                                                            \
        hipLaunchKernelGGL((rf::rf_paged_rope8_kernel<D, true>), grid, dim3(rf::rope8_threads<D>()), 0, stream, s, *cache, per);    \
    else                                                                                                   \
        hipLaunchKernelGGL((rf::rf_paged_rope8_kernel<D, false>), grid, dim3(rf::rope8_threads<D>()), 0, stream, s, *cache, per);
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
    // few rows in twos (640 rows of 8 heads of 128 3.5 us, in fours 3.7, in sixteens 6.4), many in fours (48
    // ragged requests 210 us, in sixteens 214)
    const int per = s.rows <= 4096 ? 2 : rf::kReadRows;
    const unsigned blocks = (unsigned)((s.rows + per - 1) / per), wide = std::min(blocks, 1u << 20);
    hipLaunchKernelGGL(rf::rf_paged_read8_kernel, dim3(wide, (blocks + wide - 1) / wide), dim3(256), 0, stream, s, *cache,
                       per, inv);
    return hipGetLastError();
}
