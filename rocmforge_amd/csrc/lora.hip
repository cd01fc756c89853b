// lora.hip -- low-rank adapters of many requests beside a shared projection
// (rf_lora_add_launch; the header states what it computes).  No counterpart in
// the reference.
//
// y = base + s B (A x).  Rows of one adapter, from whichever requests, are cut into tiles; one launch computes the
// tiles' A x, its k cut into slices, and a second one B times it, cut over the columns.  (A single launch in which
// every piece of the columns computes A x again reads A as often, and is kept for few rows and a small A alone.)
// Both products run on 16x16x32 MFMAs.  fp32 operands are split into two of fp16 (22 bits) after a power of two has
// brought their row to fp16's range: x as hi + 2^-11 lo, its smallest step 2^-42 of the row's largest or less, and A x,
// the row's largest in [2^14, 2^15), as hi + lo, its smallest step 2^-38 of that.
#include <hip/hip_fp16.h>

#include <algorithm>
#include <climits>

#include "../../include/rocmforge_cdna4.h"
#include "qk_common.h"

namespace rf {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr int kLoraTargets = 3;
constexpr int kFewRows = 4;                      // of a tile, whose A x is taken with dot products

struct LoraTargets {
    rf_lora_target t[kLoraTargets];
};

// 2^n of a normal value
__device__ __forceinline__ float pow2(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }

// ---- tiles ---------------------------------------------------------------------------------

// What a workgroup does.
template <int MB>
struct LoraItem {
    int id, rank, rows;          // the adapter (-1: none), its rank (0 then too) and how many rows the tile has
    int piece;                   // which of the tile's pieces
    int64_t row[MB];             // of the batch: this lane's, 16 m + lane % 16 of the tile
    bool there[MB];
};

// This workgroup's piece of a tile; false where there is none.  Wave-uniform.
//
// Requests of one adapter among 64 that follow one another are a group (those of none another), so that what they
// share of A and B is read once; a group's rows, one request behind the other, are cut into tiles of up to 16 MB.  A
// lane has a request.  Workgroups i and i + 8 share an XCD's L2: with up to 64 requests an XCD has tiles that
// follow one another, with more of them every eighth.
template <int MB>
__device__ __forceinline__ bool lora_item(const rf_lora& s, int pieces, LoraItem<MB>& w) {
    constexpr int ROWS = 16 * MB;
    const int lane = threadIdx.x & 63, col = lane & 15;
    const int xcd = blockIdx.x & 7, slot = (blockIdx.x >> 3) / pieces;
    w.piece = (blockIdx.x >> 3) % pieces;
    int j = 8 * slot + xcd;
    for (int b0 = 0; b0 < s.num_seqs; b0 += 64) {
        const int b = b0 + lane;
        int id = -1, q0 = 0, n = 0;
        if (b < s.num_seqs) {
            id = s.adapters[b];
            q0 = min(max(s.q_start[b], 0), s.rows);
            n = max(min(s.q_start[b + 1], s.rows) - q0, 0);
        }
        // the group's requests bit by bit of their adapters, and sums of their rows bit by bit: ballots take a few
        // instructions a bit, comparisons with each of the 64 took 4 us
        const int key = (unsigned)id < (unsigned)s.num_adapters ? id : s.num_adapters;
        uint64_t same = ~0ull;
        for (int k = 0; s.num_adapters >> k; ++k) {
            const bool bit = (key >> k) & 1;
            const uint64_t m = __ballot(bit);
            same &= bit ? m : ~m;
        }
        const uint64_t lower = same & ((1ull << lane) - 1);
        const int first = __builtin_ctzll(same);
        int total = 0, before = 0;               // rows of the group, and those in front of this request's
        for (int k = 0; __ballot(n >> k != 0); ++k) {
            const uint64_t m = __ballot((n >> k) & 1);
            total += __popcll(same & m) << k;
            before += __popcll(lower & m) << k;
        }
        const int tiles = first == lane ? (total + ROWS - 1) / ROWS : 0, end = wave_scan(tiles);
        const int all = __builtin_amdgcn_readlane(end, 63);
        if (s.num_seqs <= 64) {
            const int per = (all + 7) / 8;
            if (slot >= per) return false;
            j = per * xcd + slot;
        }
        if (j >= all) {
            j -= all;
            continue;
        }
        const int l = __builtin_ctzll(__ballot(end > j));
        const int at = ROWS * (j - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(tiles, l)));
        w.id = __builtin_amdgcn_readlane(key, l);
        w.id = w.id < s.num_adapters ? w.id : -1;
        w.rank = w.id >= 0 ? min(max(s.ranks[w.id], 0), s.max_rank) : 0;
        w.rows = min(__builtin_amdgcn_readlane(total, l) - at, ROWS);
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            w.there[m] = 16 * m + col < w.rows;
            w.row[m] = 0;
        }
        // the requests that have rows of the tile
        for (uint64_t left = __ballot(first == l && before < at + w.rows && before + n > at); left; left &= left - 1) {
            const int r = __builtin_ctzll(left), p = __builtin_amdgcn_readlane(before, r) - at;
            const int q = __builtin_amdgcn_readlane(q0, r) - p, e = p + __builtin_amdgcn_readlane(n, r);
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                // (rows that the tile does not have are its last one once more)
                const int i = min(16 * m + col, w.rows - 1);
                w.row[m] = i >= p && i < e ? q + i : w.row[m];
            }
        }
        return true;
    }
    return false;
}

// A x over [k0, k1) of the tile's rows into part [wave][row][rank], a share each of the first waves; returns how
// many.  Few rows: dot products.  A wave takes 256 k of 16 ranks, a lane four of them, so that a row of A is
// read 512 bytes at a time; the waves are spread over the blocks of ranks, then over k.  AHEAD: loads are a turn ahead
// where there are more than two (64 single tokens on 40 adapters 44.1 -> 42.3 us, 200 90 -> 85, rank 128 70 -> 65; one
// token of rank 64, of two turns, 14.8 -> 15.3; eight waves do not have the registers).  It takes the kernel's registers
// to 256 and more, one wave a SIMD, for the tiles of many rows too: prompts of rank 128 178 -> 172 and 72 166 -> 140,
// rank 32 even, pieces of prompt of up to 200 rows 28.5 -> 29.4.
template <bool X16, bool AHEAD, int MB, int NW, int HS>
__device__ __forceinline__ int lora_dots(const rf_lora& s, const uint16_t* a, const LoraItem<MB>& w, int k0, int k1,
                                         float (*part)[16 * MB][HS]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rank = w.rank;
    const int ranks = (rank + 15) / 16, slices = min(max(NW / ranks, 1), (k1 - k0 + 255) / 256);
    const int slice = ranks <= NW ? wave / ranks : 0;
    if (slice >= slices) return slices;
    constexpr int R = kFewRows;
    struct Turn {
        h4 v[16];
        f4 x[R];
    };
#pragma unroll 1
    for (int r0 = 16 * (ranks <= NW ? wave - slice * ranks : wave); r0 < rank; r0 += 16 * NW) {
        float acc[R][16];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[r][i] = 0.0f;
        // (behind the end loads are of the last elements, and A is zero)
        auto load = [&](int kw, Turn& t) {
            const int kk = min(kw + 4 * lane, k1 - 4);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                t.v[i] = *reinterpret_cast<const h4*>(a + (int64_t)min(r0 + i, rank - 1) * s.in_dim + kk);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t at = (int64_t)__builtin_amdgcn_readlane((int)w.row[0], r) * s.ld_x + kk;
                if constexpr (X16) {
                    const h4 y = *reinterpret_cast<const h4*>(static_cast<const uint16_t*>(s.x) + at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) t.x[r][i] = (float)y[i];
                } else {
                    t.x[r] = *reinterpret_cast<const f4*>(static_cast<const float*>(s.x) + at);
                }
            }
        };
        auto multiply = [&](int kw, Turn& t) {
            if (kw + 4 * lane >= k1) {
#pragma unroll
                for (int i = 0; i < 16; ++i) t.v[i] = h4{0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < R; ++r) t.x[r] = f4{0, 0, 0, 0};
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r > 0 && r >= w.rows) break;
#pragma unroll
                for (int i = 0; i < 16; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r][i] = __builtin_fmaf((float)t.v[i][e], t.x[r][e], acc[r][i]);
            }
        };
        const int by = 256 * slices;
        int kw = k0 + 256 * slice;
        Turn t0;
        if constexpr (AHEAD) {
            if (kw + 2 * by < k1) {
                Turn t1;
                load(kw, t0);
                __builtin_amdgcn_sched_barrier(0);
                for (; kw < k1; kw += 2 * by) {
                    load(kw + by, t1);
                    __builtin_amdgcn_sched_barrier(0);
                    multiply(kw, t0);
                    __builtin_amdgcn_sched_barrier(0);
                    load(kw + 2 * by, t0);
                    __builtin_amdgcn_sched_barrier(0);
                    multiply(kw + by, t1);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        for (; kw < k1; kw += by) {
            load(kw, t0);
            __builtin_amdgcn_sched_barrier(0);
            multiply(kw, t0);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r > 0 && r >= w.rows) break;
            // 16 sums over 64 lanes: each step halves the values a lane has and doubles their lanes
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = acc[r][i];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (lane & 1 ? v[i + 8] : v[i]) + lane_xor<1>(lane & 1 ? v[i] : v[i + 8]);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (lane & 2 ? v[i + 4] : v[i]) + lane_xor<2>(lane & 2 ? v[i] : v[i + 4]);
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = (lane & 4 ? v[i + 2] : v[i]) + lane_xor<4>(lane & 4 ? v[i] : v[i + 2]);
            v[0] = (lane & 8 ? v[1] : v[0]) + lane_xor<8>(lane & 8 ? v[0] : v[1]);
            v[0] = xor_sum<16, 32>(v[0]);
            const int i = 8 * (lane & 1) + 4 * ((lane >> 1) & 1) + 2 * ((lane >> 2) & 1) + ((lane >> 3) & 1);
            if (lane < 16) part[slice][r][r0 + i] = v[0];
        }
    }
    return slices;
}

// Any rows: MFMAs.  U: k-steps of 32 that a wave takes at once.
//
// fp32 x: a wave's sums are of 2^power x, a power a row.  It is taken from the first values, to [2^7, 2^8), which leaves
// room for values 2^8 times as large.  Where one did not fit all the same, the wave, which has seen all of its values by
// then, takes that row's power from its largest and begins again.  The power costs 64 tokens on 40 adapters nothing
// (42.1 us), prompts of rank 32, 64 and 128 0.4 (83.9), 1.7 (102) and 3.8 us (190); a value of 10^6 in the middle of every
// row takes the first two to 98.5 and 119.
template <bool X16, int RB, int MB, int NW, int U, int HS>
__device__ __forceinline__ int lora_down(const rf_lora& s, const uint16_t* a, const LoraItem<MB>& w, int k0, int k1,
                                         float (*part)[16 * MB][HS]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4, rank = w.rank;
    // the operands of U k-steps
    struct Steps {
        h8 x16[X16 ? U : 1][MB];
        f4 x32[X16 ? 1 : U][MB][2];
        h8 a[U][RB];
    };
    const uint16_t* arow[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) arow[i] = a + (int64_t)min(16 * i + col, rank - 1) * s.in_dim;
    const int groups = (k1 - k0 + 32 * U - 1) / (32 * U);
    f4 acc[RB][MB], low[X16 ? 1 : RB][MB];
    auto load = [&](int group, Steps& v) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = min(k0 + 32 * (U * group + u) + 8 * quad, k1 - 8);
#pragma unroll
            for (int m = 0; m < MB; ++m)
                if constexpr (X16) {
                    v.x16[u][m] = *reinterpret_cast<const h8*>(static_cast<const uint16_t*>(s.x) + w.row[m] * s.ld_x + k);
                } else {
                    const float* x = static_cast<const float*>(s.x) + w.row[m] * s.ld_x + k;
                    v.x32[u][m][0] = *reinterpret_cast<const f4*>(x);
                    v.x32[u][m][1] = *reinterpret_cast<const f4*>(x + 4);
                }
#pragma unroll
            for (int i = 0; i < RB; ++i) v.a[u][i] = *reinterpret_cast<const h8*>(arow[i] + k);
        }
    };
    [[maybe_unused]] int power[MB];
    [[maybe_unused]] float top[MB] = {};         // this lane's largest magnitudes, NaN left out
    [[maybe_unused]] auto look = [&](const Steps& v) {
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) top[m] = fmaxf(top[m], fabsf(v.x32[u][m][i >> 2][i & 3]));
    };
    // what brings x to [2^to, 2^(to + 1)), as far as a power of 127 does
    [[maybe_unused]] auto power_to = [](int to, float x) { return min(to + 127 - (int)(__float_as_uint(x) >> 23), 127); };
    auto multiply = [&](int group, const Steps& v) {
        if constexpr (!X16) look(v);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (behind the end A is zero, and x once more its last elements)
            const bool in = k0 + 32 * (U * group + u) + 8 * quad < k1;
            const h8 none = {0, 0, 0, 0, 0, 0, 0, 0};
            h8 xh[MB], xl[MB];
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                if constexpr (X16) {
                    xh[m] = v.x16[u][m];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float f = v.x32[u][m][i >> 2][i & 3] * pow2(power[m]);
                        xh[m][i] = (_Float16)f;
                        // (one instruction takes the fp16 value off)
                        xl[m][i] = (_Float16)__builtin_fmaf((float)xh[m][i], -2048.0f, f * 2048.0f);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                if (i > 0 && 16 * i >= rank) break;
                const h8 v1 = in ? v.a[u][i] : none;
#pragma unroll
                for (int m = 0; m < MB; ++m) {
                    acc[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, xh[m], acc[i][m], 0, 0, 0);
                    if constexpr (!X16) low[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, xl[m], low[i][m], 0, 0, 0);
                }
            }
        }
    };
    // A group ahead of its loads, which are without conditions (addresses are clamped instead): past a branch
    // around loads the compiler waits for all of them, and without the barriers it moves them down to their uses.
    Steps v0, v1;
    for (bool first = true;; first = false) {
#pragma unroll
        for (int m = 0; m < MB; ++m) {
#pragma unroll
            for (int i = 0; i < RB; ++i) acc[i][m] = f4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < (X16 ? 1 : RB); ++i) low[i][m] = f4{0, 0, 0, 0};
        }
        load(wave, v0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!X16)
            if (first) {
                look(v0);
#pragma unroll
                for (int m = 0; m < MB; ++m) power[m] = power_to(7, xor_max<32, 16>(top[m]));
            }
        for (int k = wave; k < groups; k += 2 * NW) {
            load(k + NW, v1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(k, v0);
            __builtin_amdgcn_sched_barrier(0);
            load(k + 2 * NW, v0);
            __builtin_amdgcn_sched_barrier(0);
            multiply(k + NW, v1);
            __builtin_amdgcn_sched_barrier(0);
            // (the sums are read behind the loop, 8 wait states after the last product at the earliest: the compiler
            // left 6 where a branch skips the last block of ranks)
            asm volatile("s_nop 7");
        }
        if constexpr (X16) break;
        bool over = false;                       // (a row of an infinity is lost in any case)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const float most = xor_max<32, 16>(top[m]);
            const bool more = most * pow2(power[m]) > 65504.0f && most < INFINITY;
            power[m] = more ? power_to(14, most) : power[m];
            over = over || more;
        }
        if (__ballot(over) == 0) break;
    }
    // lane: row col, ranks 16 i + 4 quad ..
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            f4 v = acc[i][m];
            if constexpr (!X16) {
                v += low[i][m] * (1.0f / 2048.0f);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], -power[m]);
            }
            *reinterpret_cast<f4*>(&part[wave][16 * m + col][16 * i + 4 * quad]) = v;
        }
    return NW;
}

// Blocks of 16 columns that a wave takes at once.
constexpr int lora_cols(int rb) { return rb == 8 ? 2 : 4; }

// y = base + scale B (A x) for the columns [nb0, nb1) of 16; part(k, j): four of A x's k-th part, ranks j .. of the
// lane's row.  A wave takes 256 columns of a row in one go, 64 bytes an instruction: blocks further apart cost the
// prompts a fifth.
template <int RB, int NW, class Part>
__device__ __forceinline__ void lora_up(const rf_lora& s, const rf_lora_target& g, const LoraItem<1>& w, int nb0, int nb1,
                                        int slices, Part part) {
    constexpr int J = (RB + 1) / 2, V = lora_cols(RB);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4, rank = w.rank;
    const float scale = s.scales[w.id];
    struct Cols {
        h8 b[V][J];
        f4 y[V];
    };
    const uint16_t* b = g.b + w.id * g.b_stride;
    const float* base = g.base + w.row[0] * g.ld_base;
    float* out = g.y + w.row[0] * g.ld_y;
    int at[J];                                   // of a row of B; behind the rank its first elements, which are there
    u32x4 keep[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int j0 = 32 * j + 8 * quad;
        at[j] = j0 < rank ? j0 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            keep[j][i] = (j0 + 2 * i < rank ? 0xffffu : 0u) | (j0 + 2 * i + 1 < rank ? 0xffff0000u : 0u);
    }
    auto load_cols = [&](int nb, Cols& c) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int n0 = 16 * min(nb + v, nb1 - 1);
            const uint16_t* brow = b + (int64_t)min(n0 + col, g.out_dim - 1) * s.max_rank;
#pragma unroll
            for (int j = 0; j < J; ++j) c.b[v][j] = *reinterpret_cast<const h8*>(brow + at[j]);
            c.y[v] = *reinterpret_cast<const f4*>(base + min(n0 + 4 * quad, g.out_dim - 4));
        }
    };
    Cols c0, c1;
    load_cols(nb0 + V * wave, c0);
    f4 h[2 * J];
#pragma unroll
    for (int j = 0; j < 2 * J; ++j) h[j] = f4{0, 0, 0, 0};
#pragma unroll 2
    for (int k = 0; k < slices; ++k)
#pragma unroll
        for (int j = 0; j < 2 * J; ++j) h[j] += part(k, min(32 * (j >> 1) + 8 * quad + 4 * (j & 1), 16 * RB - 4));
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 2 * J; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h[j][e] = 32 * (j >> 1) + 8 * quad + 4 * (j & 1) + e < rank ? h[j][e] : 0.0f;
            top = fmaxf(top, fabsf(h[j][e]));
        }
    top = xor_max<32, 16>(top);
    // A x is 2^back times hi + lo
    const int back = top > 0.0f && top < INFINITY ? (int)(__float_as_uint(top) >> 23) - 127 - 14 : 0;
    h8 hi[J], lo[J];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = ldexpf(h[2 * j + (e >> 2)][e & 3], -back);
            hi[j][e] = (_Float16)f;
            lo[j][e] = (_Float16)(f - (float)hi[j][e]);
        }
    auto store_cols = [&](int nb, const Cols& c) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int n = 16 * (nb + v) + 4 * quad;
            f4 y = c.y[v], d = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < J; ++j) {
                if (j > 0 && 32 * j >= rank) break;
                const h8 m = __builtin_bit_cast(h8, __builtin_bit_cast(u32x4, c.b[v][j]) & keep[j]);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(m, hi[j], d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(m, lo[j], d, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(ldexpf(d[i], back), scale, y[i]);
            if (w.there[0] && nb + v < nb1 && n < g.out_dim) *reinterpret_cast<f4*>(out + n) = y;
        }
    };
    for (int nb = nb0 + V * wave; nb < nb1; nb += 2 * NW * V) {
        load_cols(nb + NW * V, c1);
        __builtin_amdgcn_sched_barrier(0);
        store_cols(nb, c0);
        __builtin_amdgcn_sched_barrier(0);
        load_cols(nb + 2 * NW * V, c0);
        __builtin_amdgcn_sched_barrier(0);
        store_cols(nb + NW * V, c1);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Rows of requests without an adapter: y = base.
template <int NW>
__device__ __forceinline__ void lora_copy(const rf_lora_target& g, const LoraItem<1>& w, int nb0, int nb1) {
    if (g.base == g.y) return;
    constexpr int V = 8;
    const int n1 = min(16 * nb1, g.out_dim), wave = threadIdx.x >> 6, quad = (threadIdx.x & 63) >> 4;
    const float* base = g.base + w.row[0] * g.ld_base;
    float* out = g.y + w.row[0] * g.ld_y;
    for (int n0 = 16 * (nb0 + V * wave) + 4 * quad; n0 < n1; n0 += 16 * NW * V) {
        f4 v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = *reinterpret_cast<const f4*>(base + min(n0 + 16 * i, n1 - 4));
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (w.there[0] && n0 + 16 * i < n1) *reinterpret_cast<f4*>(out + n0 + 16 * i) = v[i];
    }
}

// Few rows: one launch, and every piece of a tile's columns computes the tile's A x itself.
template <bool X16, int NW>
__global__ __launch_bounds__(64 * NW) void rf_lora_whole_kernel(const rf_lora s, const LoraTargets targets, int pieces) {
    constexpr int RB = 1, HS = 16 * RB + 4;
    __shared__ __align__(16) float part[NW][16][HS];
    const rf_lora_target& g = targets.t[blockIdx.y];
    const int blocks = (g.out_dim + 15) / 16, each = (blocks + pieces - 1) / pieces;
    LoraItem<1> w;
    if (!lora_item<1>(s, pieces, w)) return;
    const int nb0 = w.piece * each, nb1 = min(nb0 + each, blocks);
    if (nb0 >= nb1) return;
    if (w.rank == 0) return lora_copy<NW>(g, w, nb0, nb1);
    const int slices = lora_dots<X16, false, 1, NW, HS>(s, g.a + w.id * g.a_stride, w, 0, s.in_dim, part);
    lds_barrier();
    const int r = min((int)threadIdx.x & 15, w.rows - 1);
    lora_up<RB, NW>(s, g, w, nb0, nb1, slices, [&](int k, int j) { return *reinterpret_cast<const f4*>(&part[k][r][j]); });
}

// Many: A x by one launch, its k cut into slices ...
template <bool X16, int RB, int MB, int NW, int U>
__global__ __launch_bounds__(64 * NW) void rf_lora_down_kernel(const rf_lora s, const LoraTargets targets, float* sums,
                                                               int slices, int each) {
    constexpr int HS = 16 * RB + 4;
    __shared__ __align__(16) float part[NW][16 * MB][HS];
    __shared__ int rows[16 * MB];
    const rf_lora_target& g = targets.t[blockIdx.y];
    LoraItem<MB> w;
    if (!lora_item<MB>(s, slices, w) || w.rank == 0) return;
    if (threadIdx.x < 16)
#pragma unroll
        for (int m = 0; m < MB; ++m) rows[16 * m + threadIdx.x] = (int)w.row[m];
    const int k0 = w.piece * each, k1 = min(k0 + each, s.in_dim);
    const uint16_t* a = g.a + w.id * g.a_stride;
    const int parts = w.rows <= kFewRows ? lora_dots<X16, true, MB, NW, HS>(s, a, w, k0, k1, part)
                                         : lora_down<X16, RB, MB, NW, U, HS>(s, a, w, k0, k1, part);
    lds_barrier();
    float* to = sums + (int64_t)(blockIdx.y * slices + w.piece) * s.rows * (16 * RB);
    for (int i = threadIdx.x; i < 4 * RB * w.rows; i += 64 * NW) {
        const int r = i / (4 * RB), j = 4 * (i % (4 * RB));
        if (j >= w.rank) continue;
        f4 v = {0, 0, 0, 0};
        for (int k = 0; k < parts; ++k) v += *reinterpret_cast<const f4*>(&part[k][r][j]);
        *reinterpret_cast<f4*>(to + (int64_t)rows[r] * (16 * RB) + j) = v;
    }
}

// ... and B times it by a second.
template <int RB, int NW>
__global__ __launch_bounds__(64 * NW) void rf_lora_up_kernel(const rf_lora s, const LoraTargets targets, const float* sums,
                                                             int slices, int pieces) {
    const rf_lora_target& g = targets.t[blockIdx.y];
    const int blocks = (g.out_dim + 15) / 16, each = (blocks + pieces - 1) / pieces;
    LoraItem<1> w;
    if (!lora_item<1>(s, pieces, w)) return;
    const int nb0 = w.piece * each, nb1 = min(nb0 + each, blocks);
    if (nb0 >= nb1) return;
    if (w.rank == 0) return lora_copy<NW>(g, w, nb0, nb1);
    const int64_t next = (int64_t)s.rows * (16 * RB);
    const float* from = sums + blockIdx.y * slices * next + w.row[0] * (16 * RB);
    lora_up<RB, NW>(s, g, w, nb0, nb1, slices, [&](int k, int j) { return *reinterpret_cast<const f4*>(from + k * next + j); });
}

}  // namespace rf

// ---- launchers -----------------------------------------------------------------------------

namespace {

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// What a launch refuses, before its workspace; and whether there is anything to do.
bool lora_ok(const rf_lora* step, const rf_lora_target* targets, int num_targets) {
    if (step == nullptr || targets == nullptr || num_targets < 1 || num_targets > rf::kLoraTargets) return false;
    const rf_lora& s = *step;
    if (s.rows < 0 || s.rows > (1 << 23) || s.num_seqs < 0 || s.num_adapters < 0 || s.max_rank < 8 || s.max_rank > 128 ||
        s.max_rank % 8 || s.in_dim < 8 || s.in_dim > (1 << 20) || s.in_dim % 8)
        return false;
    const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    for (int i = 0; i < num_targets; ++i)
        if (targets[i].out_dim < 4 || targets[i].out_dim > (1 << 20) || targets[i].out_dim % 4) return false;
    if (s.rows == 0 || s.num_seqs == 0) return true;
    if (!s.x || !s.adapters || !s.q_start || !aligned(s.x) || s.ld_x < s.in_dim || s.ld_x % (s.x_f16 ? 8 : 4) ||
        (s.num_adapters > 0 && (!s.ranks || !s.scales)))
        return false;
    for (int i = 0; i < num_targets; ++i) {
        const rf_lora_target& t = targets[i];
        if (!t.base || !t.y || !aligned(t.base) || !aligned(t.y) || t.ld_base < t.out_dim || t.ld_y < t.out_dim ||
            t.ld_base % 4 || t.ld_y % 4 || (t.base == t.y && t.ld_base != t.ld_y))
            return false;
        if (s.num_adapters > 0 && (!t.a || !t.b || !aligned(t.a) || !aligned(t.b) || t.a_stride % 8 || t.b_stride % 8 ||
                                   t.a_stride < (int64_t)s.max_rank * s.in_dim || t.b_stride < (int64_t)s.max_rank * t.out_dim))
            return false;
    }
    return true;
}

struct LoraPlan {
    bool whole;                  // one launch
    int rb, mb;                  // blocks of 16 ranks, and of rows of a tile of A x
    int down, up;                // tiles (at least as many as there are, a multiple of 8) of either product
    int slices, each;            // of k
};

// Tiles of A x have 16 times as many rows.
int blocks_of_rows(int rows) { return rows < 768 ? 1 : rows < 2560 ? 2 : 4; }

// Workgroups that slices of k are to come to, and the most slices.
constexpr int kDownAim = 288, kSlices = 8;

LoraPlan lora_plan(const rf_lora& s, int num_targets) {
    LoraPlan p;
    // (a single token, 4096 -> 4096 + 1024 + 1024, rank 16, in a graph 8.3 us for 8.7, and a launch less to issue;
    // of rank 64 20 for 15, 16 rows of rank 16 20 for 13)
    p.whole = s.rows <= rf::kFewRows && s.max_rank <= 16 && (int64_t)s.max_rank * s.in_dim <= (1 << 17);
    const int blocks = ceil_div(s.max_rank, 16);
    p.rb = blocks <= 1 ? 1 : blocks <= 2 ? 2 : blocks <= 4 ? 4 : 8;
    // Tiles of more rows read A less often and leave fewer workgroups.  us, 16 / 32 / 64 rows, 12288 -> 4096 of rank
    // 32: 512 rows 19.8 / 20.0 / 25.9, 1024 27.7 / 26.1 / 28.9, 2048 49.5 / 43.4 / 46.1, 3059 of 30 requests 76 / 72 / 66
    p.mb = p.rb == 8 ? 1 : blocks_of_rows(s.rows);
    // (groups of 64 requests are no more than the adapters, and none)
    const int64_t groups = std::min<int64_t>(s.num_seqs, (int64_t)ceil_div(s.num_seqs, 64) * (std::min(63, s.num_adapters) + 1));
    const auto tiles = [&](int mb) { return ceil_div(std::min<int64_t>(s.rows, s.rows / (16 * mb) + groups), 8) * 8; };
    p.down = tiles(p.mb);
    p.up = tiles(1);
    // few tiles: k over more workgroups, at least 256 each (16 rows, 12288 -> 4096: 4 slices 17.9 us, 8 14.8)
    p.slices = std::min(std::max(kDownAim / (p.down * num_targets), 1), kSlices);
    p.each = ceil_div(ceil_div(s.in_dim, p.slices), 256) * 256;
    p.slices = ceil_div(s.in_dim, p.each);
    return p;
}

// No less than num_targets p.slices rows slots, and no less for a larger step, so that the largest one's workspace serves
// all: there are no fewer tiles than rows / (16 p.mb), and no more slices than these leave of kDownAim.
size_t lora_bytes(const rf_lora& s, const LoraPlan& p, int num_targets) {
    if (p.whole) return 0;
    const int64_t rows = (int64_t)num_targets * s.rows;
    const int64_t slots = std::min<int64_t>(rows * std::min(kSlices, ceil_div(s.in_dim, 256)),
                                            std::max<int64_t>(rows, kDownAim * 16 * blocks_of_rows(s.rows)));
    return (size_t)slots * 16 * p.rb * sizeof(float);
}

}  // namespace

extern "C" size_t rf_lora_workspace_bytes(const rf_lora* step, const rf_lora_target* targets, int num_targets) {
    if (!lora_ok(step, targets, num_targets) || step->rows == 0 || step->num_seqs == 0) return 0;
    return lora_bytes(*step, lora_plan(*step, num_targets), num_targets);
}

extern "C" hipError_t rf_lora_add_launch(const rf_lora* step, const rf_lora_target* targets, int num_targets,
                                         hipStream_t stream) {
    using namespace rf;
    if (!lora_ok(step, targets, num_targets)) return hipErrorInvalidValue;
    const rf_lora& s = *step;
    if (s.rows == 0 || s.num_seqs == 0) return hipSuccess;
    LoraTargets all = {};
    int widest = 0;
    for (int i = 0; i < num_targets; ++i) {
        all.t[i] = targets[i];
        widest = std::max(widest, targets[i].out_dim);
    }
    const LoraPlan p = lora_plan(s, num_targets);
    constexpr int NW = 4, WHOLE = 8;             // waves
    if (p.whole) {
        const int pieces = std::min(std::max(device_cu_count() / (p.up * num_targets), 1), ceil_div(widest, 64 * WHOLE));
        const dim3 grid((unsigned)(p.up * pieces), num_targets);
        if (s.x_f16)
            hipLaunchKernelGGL((rf_lora_whole_kernel<true, WHOLE>), grid, dim3(64 * WHOLE), 0, stream, s, all, pieces);
        else
            hipLaunchKernelGGL((rf_lora_whole_kernel<false, WHOLE>), grid, dim3(64 * WHOLE), 0, stream, s, all, pieces);
        return hipGetLastError();
    }
    if (s.workspace == nullptr || (reinterpret_cast<uintptr_t>(s.workspace) & 15u) != 0 ||
        s.workspace_bytes < lora_bytes(s, p, num_targets))
        return hipErrorInvalidValue;
    float* sums = static_cast<float*>(s.workspace);
    // Pieces of the columns: one workgroup a CU for few tiles (each starts with some 4 us of latencies), two for many,
    // whose ranks differ.  us, 256 / 512 / 768 workgroups: 2 tokens on adapters of up to 64, 4096 -> 2 x 12288, 14.1 /
    // 15.5 / 19.4, 16 18.7 / 22.7 / 22.7, 64 on 40 adapters 56.6 / 42.3 / 42.5
    const int tiles = p.up * num_targets;
    const int pieces = std::min(ceil_div(tiles < 64 ? 256 : 512, tiles), ceil_div(widest, 64 * NW));
    const dim3 down((unsigned)(p.down * p.slices), num_targets), up((unsigned)(p.up * pieces), num_targets), blk(64 * NW);
#define LORA_DOWN(RB, MB, U)                                                                                           \
    if (s.x_f16)                                                                                                       \
        hipLaunchKernelGGL((rf_lora_down_kernel<true, RB, MB, NW, U>), down, blk, 0, stream, s, all, sums, p.slices, p.each);  \
    else                                                                                                               \
        hipLaunchKernelGGL((rf_lora_down_kernel<false, RB, MB, NW, U>), down, blk, 0, stream, s, all, sums, p.slices, p.each);
#define LORA_BOTH(RB, U)                                                                                               \
    if (p.mb == 1) {                                                                                                   \
        LORA_DOWN(RB, 1, U)                                                                                            \
    } else if (p.mb == 2) {                                                                                            \
        LORA_DOWN(RB, 2, U)                                                                                            \
    } else {                                                                                                           \
        LORA_DOWN(RB, 4, U)                                                                                            \
    }                                                                                                                  \
    hipLaunchKernelGGL((rf_lora_up_kernel<RB, NW>), up, blk, 0, stream, s, all, sums, p.slices, pieces);
    if (p.rb == 1) {
        LORA_BOTH(1, 2)
    } else if (p.rb == 2) {
        LORA_BOTH(2, 2)
    } else if (p.rb == 4) {
        LORA_BOTH(4, 1)
    } else {
        LORA_DOWN(8, 1, 1)
        hipLaunchKernelGGL((rf_lora_up_kernel<8, NW>), up, blk, 0, stream, s, all, sums, p.slices, pieces);
    }
#undef LORA_BOTH
#undef LORA_DOWN
    return hipGetLastError();
}
