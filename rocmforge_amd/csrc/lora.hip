// lora.hip -- low-rank adapters of many requests beside a shared projection
// (rf_lora_add_launch; the header states what it computes).  No counterpart in
// the reference.
//
// y = base + s B (A x).  A workgroup takes a tile of up to 16 rows of a request, a target
// and a piece of the output's columns, and computes the tile's A x itself: that is r / N-th
// of nothing beside reading A, which the pieces of one tile share in an XCD's L2, and it
// saves a second launch and the trip of A x through memory.  Both products run on 16x16x32
// MFMAs.  fp32 operands are split into two of fp16 (22 bits), so that sums are as good as in fp32:
// x as hi + 2^-11 lo, A x as hi + lo after its row is brought to [2^14, 2^15) by a power of two.
#include <hip/hip_fp16.h>

#include <algorithm>
#include <climits>

#include "../../include/rocmforge_cdna4.h"
#include "qk_common.h"

namespace rf {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kLoraRows = 16, kLoraWaves = 4, kLoraTargets = 3;

struct LoraTargets {
    rf_lora_target t[kLoraTargets];
};

struct LoraTile {
    int b, row, rows;            // the request, the tile's first row and how many
};

// Tile j over the requests; wave-uniform.
__device__ __forceinline__ bool lora_tile(const rf_lora& s, int j, LoraTile& t) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0; b0 < s.num_seqs; b0 += 64) {
        const int b = b0 + lane;
        int q0 = 0, n = 0;
        if (b < s.num_seqs) {
            q0 = min(max(s.q_start[b], 0), s.rows);
            n = max(min(s.q_start[b + 1], s.rows) - q0, 0);
        }
        const int tiles = (n + kLoraRows - 1) / kLoraRows;
        int end = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(end, o);
            if (lane >= o) end += u;
        }
        end += before;
        const uint64_t past = __ballot(end > j);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int k = j - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(tiles, l));
            t.b = b0 + l;
            t.row = __builtin_amdgcn_readlane(q0, l) + kLoraRows * k;
            t.rows = min(__builtin_amdgcn_readlane(n, l) - kLoraRows * k, kLoraRows);
            return true;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return false;
}

// RB: blocks of 16 ranks.
template <bool X16, int RB>
__global__ __launch_bounds__(64 * kLoraWaves) void rf_lora_kernel(const rf_lora s, const LoraTargets targets, int splits) {
    constexpr int NW = kLoraWaves, J = (RB + 1) / 2, HS = 16 * RB + 4;           // k-steps of the second product, floats a row of A x
    __shared__ __align__(16) float part[NW][kLoraRows][HS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const rf_lora_target& g = targets.t[blockIdx.y];
    // (workgroups i and i + 8 share an XCD's L2: the pieces of a tile)
    const int split = (blockIdx.x >> 3) % splits, item = ((blockIdx.x >> 3) / splits) * 8 + (blockIdx.x & 7);
    const int blocks = (g.out_dim + 15) / 16, each = (blocks + splits - 1) / splits;
    const int nb0 = split * each, nb1 = min(nb0 + each, blocks);
    LoraTile t;
    if (nb0 >= nb1 || !lora_tile(s, item, t)) return;
    const int id = s.adapters[t.b];
    const bool on = (unsigned)id < (unsigned)s.num_adapters;
    const int rank = on ? min(max(s.ranks[id], 0), s.max_rank) : 0;
    if (rank == 0 && g.base == g.y) return;
    const int my_row = t.row + min(col, t.rows - 1);
    h8 hi[J], lo[J];
    int back = 0;                                // A x is 2^back times what hi + lo say
    if (rank > 0) {
        const uint16_t* a = g.a + id * g.a_stride;
        f4 acc[RB], low[X16 ? 1 : RB];
#pragma unroll
        for (int i = 0; i < RB; ++i) acc[i] = f4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < (X16 ? 1 : RB); ++i) low[i] = f4{0, 0, 0, 0};
        const int64_t xrow = my_row * s.ld_x;
        for (int k0 = 32 * wave; k0 < s.in_dim; k0 += 32 * NW) {
            const int k = k0 + 8 * quad, kk = min(k, s.in_dim - 8);
            h8 xh, xl;
            if constexpr (X16) {
                xh = *reinterpret_cast<const h8*>(static_cast<const uint16_t*>(s.x) + xrow + kk);
            } else {
                const float* x = static_cast<const float*>(s.x) + xrow + kk;
                const f4 u = *reinterpret_cast<const f4*>(x), v = *reinterpret_cast<const f4*>(x + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float f = i < 4 ? u[i & 3] : v[i & 3];
                    xh[i] = (_Float16)f;
                    xl[i] = (_Float16)((f - (float)xh[i]) * 2048.0f);
                }
            }
            const bool in = k < s.in_dim;
            if (!in) xh = xl = h8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                if (16 * i >= rank) break;
                h8 w = *reinterpret_cast<const h8*>(a + (int64_t)min(16 * i + col, rank - 1) * s.in_dim + kk);
                if (!in) w = h8{0, 0, 0, 0, 0, 0, 0, 0};
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, xh, acc[i], 0, 0, 0);
                if constexpr (!X16) low[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, xl, low[i], 0, 0, 0);
            }
        }
        // lane: row col, ranks 16 i + 4 quad ..
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            f4 v = acc[i];
            if constexpr (!X16) v += low[i] * (1.0f / 2048.0f);
            *reinterpret_cast<f4*>(&part[wave][col][16 * i + 4 * quad]) = v;
        }
        __syncthreads();
        float h[J][8], top = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int j0 = 32 * j + 8 * quad;
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                f4 v = {0, 0, 0, 0};
                if (j0 < 16 * RB)
#pragma unroll
                    for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const f4*>(&part[w][col][j0 + e]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    h[j][e + i] = j0 + e + i < rank ? v[i] : 0.0f;
                    top = fmaxf(top, fabsf(h[j][e + i]));
                }
            }
        }
        top = xor_max<32, 16>(top);
        if (top > 0.0f && top < INFINITY) back = (int)(__float_as_uint(top) >> 23) - 127 - 14;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = ldexpf(h[j][e], -back);
                hi[j][e] = (_Float16)f;
                lo[j][e] = (_Float16)(f - (float)hi[j][e]);
            }
    }
    const float scale = on ? s.scales[id] : 0.0f;
    const uint16_t* b = g.b + (on ? id : 0) * g.b_stride;
    for (int nb = nb0 + wave; nb < nb1; nb += NW) {
        const int n = 16 * nb + 4 * quad;
        f4 v = {0, 0, 0, 0};
        if (rank > 0) {
            const uint16_t* brow = b + (int64_t)min(16 * nb + col, g.out_dim - 1) * s.max_rank;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int j0 = 32 * j + 8 * quad;
                if (32 * j >= rank) break;
                h8 w = *reinterpret_cast<const h8*>(brow + min(j0, s.max_rank - 8));
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (j0 + i >= rank) w[i] = 0;
                v = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, hi[j], v, 0, 0, 0);
                v = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, lo[j], v, 0, 0, 0);
            }
        }
        if (col >= t.rows || n >= g.out_dim) continue;
        f4 y = *reinterpret_cast<const f4*>(g.base + my_row * g.ld_base + n);
        if (rank > 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(ldexpf(v[i], back), scale, y[i]);
        *reinterpret_cast<f4*>(g.y + my_row * g.ld_y + n) = y;
    }
}

}  // namespace rf

extern "C" hipError_t rf_lora_add_launch(const rf_lora* step, const rf_lora_target* targets, int num_targets,
                                         hipStream_t stream) {
    using namespace rf;
    if (step == nullptr || targets == nullptr || num_targets < 1 || num_targets > kLoraTargets)
        return hipErrorInvalidValue;
    const rf_lora& s = *step;
    if (s.rows < 0 || s.rows > (1 << 23) || s.num_seqs < 0 || s.num_adapters < 0 || s.max_rank < 8 || s.max_rank > 128 ||
        s.max_rank % 8 || s.in_dim < 8 || s.in_dim > (1 << 20) || s.in_dim % 8)
        return hipErrorInvalidValue;
    const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    LoraTargets all = {};
    int widest = 0;
    for (int i = 0; i < num_targets; ++i) {
        const rf_lora_target& t = targets[i];
        if (t.out_dim < 4 || t.out_dim > (1 << 20) || t.out_dim % 4) return hipErrorInvalidValue;
        all.t[i] = t;
        widest = std::max(widest, t.out_dim);
    }
    if (s.rows == 0 || s.num_seqs == 0) return hipSuccess;
    if (!s.x || !s.adapters || !s.q_start || !aligned(s.x) || s.ld_x < s.in_dim || s.ld_x % (s.x_f16 ? 8 : 4) ||
        (s.num_adapters > 0 && (!s.ranks || !s.scales)))
        return hipErrorInvalidValue;
    for (int i = 0; i < num_targets; ++i) {
        const rf_lora_target& t = all.t[i];
        if (!t.base || !t.y || !aligned(t.base) || !aligned(t.y) || t.ld_base < t.out_dim || t.ld_y < t.out_dim ||
            t.ld_base % 4 || t.ld_y % 4 || (t.base == t.y && t.ld_base != t.ld_y))
            return hipErrorInvalidValue;
        if (s.num_adapters > 0 && (!t.a || !t.b || !aligned(t.a) || !aligned(t.b) || t.a_stride % 8 || t.b_stride % 8 ||
                                   t.a_stride < (int64_t)s.max_rank * s.in_dim || t.b_stride < (int64_t)s.max_rank * t.out_dim))
            return hipErrorInvalidValue;
    }
    const int tiles = (int)std::min<int64_t>(s.rows, s.rows / kLoraRows + (int64_t)s.num_seqs);
    const int aim = 2 * device_cu_count();
    const int splits = std::min(std::max(aim / (tiles * num_targets), 1), (widest + 63) / 64);
    const dim3 grid((unsigned)((tiles + 7) / 8 * 8 * splits), num_targets), blk(64 * kLoraWaves);
    const int rb = (s.max_rank + 15) / 16;
#define LORA_GO(RB)                                                                                    \
    if (s.x_f16)                                                                                       \
        hipLaunchKernelGGL((rf_lora_kernel<true, RB>), grid, blk, 0, stream, s, all, splits);          \
    else                                                                                               \
        hipLaunchKernelGGL((rf_lora_kernel<false, RB>), grid, blk, 0, stream, s, all, splits);
    if (rb <= 1) {
        LORA_GO(1)
    } else if (rb <= 2) {
        LORA_GO(2)
    } else if (rb <= 4) {
        LORA_GO(4)
    } else {
        LORA_GO(8)
    }
#undef LORA_GO
    return hipGetLastError();
}
