// paged_attn.hip -- causal GQA attention of the new rows of a batch over a
// paged fp16 cache (rf_paged_attention_launch; the header states what it
// computes; paged_attn.h how).  No counterpart in the reference, which runs one
// sequence over a contiguous cache.  K and V come by LDS DMA from the pages, 2 to 8
// rows an instruction (never across a page).
#include "paged_attn.h"

namespace rf {

// Least units of keys of a part (a workgroup costs about as much as 4 to 6 units
// before and behind its loop; wide ones, and narrow ones beside them, more).  us, wide parts of at least 4 / 8 / 16 / 24 units: 28 single tokens
// beside 4 pieces of prompt 39.5 / 33.4 / 28.5 / 28.4; 64 tokens behind 15936 66.1 / 66.2 / 50.7 / 52.9;
// 4 prompts of 200 behind 2800 64.4 / 64.9 / 64.9 / 64.9.
constexpr int kNarrowLeast = 4, kBesideLeast = 16;
constexpr int kWideLeast = 24;
// Where tables are no wider than these many units nothing is cut, and no join is launched.  us, cut ->
// whole, in tables of just these widths: few narrow tiles (one request of 256 positions 8.2 -> 5.9, of
// 500 8.8 -> 8.4, 8 of 500 9.7 -> 8.6), 256 tiles and more (32 requests of 20 to 1000 17.2 -> 15.3, 256 of 600
// 132 -> 126), beside wide ones (20 of 500 beside two prompts 28.0 -> 26.2), and wide tiles: a prompt of 1500
// 41.4 -> 41.0, but pieces behind a context lose by it (2 of 100 behind 1900 36.3 -> 46.0).
constexpr int kFewWhole = 16, kManyWhole = 32, kWideWhole = 32;

// ---- few rows -------------------------------------------------------------------------
//
// W waves; wave w takes the pieces of 32 positions w, w + W, .. of the part,
// each through its own S-stage ring in LDS (no barrier in the loop): S^T by
// 16x16x32 MFMAs, lane (row lane % 16, keys 4 (lane / 16) ..), and O^T alike.
// The waves' (m, l, O) are joined through LDS at the end.  16 KB of K and V a
// piece (head_dim 128), 64 KB and more in flight a CU.  A tile is 16 packed rows
// because a KV head's group rarely has more, and because what is left of them
// costs no bytes.  Bound by memory, and for short requests by the chain lengths ->
// share -> page -> K -> V and the join's launch.  48 requests of 60 to 16000
// positions (32 heads on 8, head_dim 128, 556 MB): 120 us with the join, 4.6 TB/s
// where a large copy reaches 5.1; one request of 640: 8.6 us.
template <int D, int W, int S>
__device__ __forceinline__ void narrow_part(const rf_paged_attention& a, const rf_paged_cache& c, const Plan& plan,
                                            int item, uint8_t* lds) {
    constexpr int ROWB = 2 * D, MAT = kNarrowKeys * ROWB, STAGE = 2 * MAT;
    constexpr int LPR = Dma<D>::LPR, RPI = Dma<D>::RPI, NI = kNarrowKeys / RPI;   // instructions a matrix
    constexpr int KS = D / 32, NB = D / 16;
    constexpr int PADD = D + 4;                          // floats a row of the join
    static_assert(kNarrowRows * (PADD + 2) * 4 <= S * STAGE, "the join fits the ring");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int nkv = c.num_kv_heads;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const uint32_t ring = lds0 + (uint32_t)wave * (S * STAGE);
    const int dr = lane / LPR, ds = lane % LPR;

    Share s;
    const int kvh = item % nkv;
    if (!find_share<kNarrowRows, kNarrowKeys>(a, c, plan, item / nkv, false, s)) return;
    const int rows = s.n * plan.group, r0 = kNarrowRows * s.tile;
    const Span t = span_of(plan, s, r0, min(r0 + kNarrowRows, rows) - 1, a.window);
    // the part's pieces
    const int p0 = t.lo / kNarrowKeys, p1 = (t.hi + kNarrowKeys - 1) / kNarrowKeys;
    const int each = (max(p1 - p0, 0) + s.parts - 1) / s.parts;
    const int begin = p0 + s.part * each, end = min(begin + each, p1);
    const int steps = max((end - begin - wave + W - 1) / W, 0);
    // this lane's packed row
    const int r = r0 + col, token = token_of(plan, min(r, rows - 1)), head = min(r, rows - 1) - token * plan.group;
    const int pos = s.kv - s.n + token;
    // the addresses of the units of 16 pieces to come, lane (step, unit of the piece)
    const Units<rf_paged_cache> units(a, c, s.b, kvh, t.lo, t.hi);
    bool bad = false;
    int window = 0;
    uint64_t address = 0;
    const uint64_t v_from_k = (uint64_t)c.v - (uint64_t)c.k;
    const uint32_t stride = (uint32_t)(2 * c.row_stride);
    auto load_units = [&](int step) {
        const int unit = 4 * (begin + wave + W * (step + (lane >> 2))) + (lane & 3);
        address = units.address(unit, units.page_of(unit), bad);
        window = step;
    };
    auto stage = [&](int step) {
        if (step >= steps) return;
        if (step - window >= 16) load_units(step);
        const int piece = begin + wave + W * step, k0 = kNarrowKeys * piece;
        const uint32_t dst = ring + (uint32_t)(step % S) * STAGE;
        const bool whole = k0 >= t.lo && k0 + kNarrowKeys <= t.hi;
        // the ring's last readers are done
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int lr = RPI * i + dr;
            int unit = 4 * piece + (RPI * i >> 3);
            uint32_t row = (uint32_t)((RPI * i & 7) + dr) * stride;
            if (!whole) {
                // positions that no row sees are taken from the nearest one that some row sees
                unit = units.seen(unit);
                row = (uint32_t)(min(max(k0 + lr, t.lo), t.hi - 1) - 8 * unit) * stride;
            }
            const uint64_t at = read_lane(address, 4 * (step - window) + unit - 4 * piece);
            lds_dma16(__builtin_amdgcn_readfirstlane(dst + 1024u * i), row + 16u * (uint32_t)(ds ^ k_swizzle<D>(lr)),
                      reinterpret_cast<const uint8_t*>(at));
            lds_dma16(__builtin_amdgcn_readfirstlane(dst + MAT + 1024u * i),
                      row + 16u * (uint32_t)(ds ^ v_swizzle<D>(lr)), reinterpret_cast<const uint8_t*>(at + v_from_k));
        }
    };
    h8 q[KS];
    const uint16_t* qrow = a.q + (int64_t)(s.q0 + token) * a.ld_q + (int64_t)(kvh * plan.group + head) * D + 8 * quad;
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const h8*>(qrow + 32 * k);
    if (steps > 0) load_units(0);
    // (q has arrived before the DMAs start, so that none but theirs are counted below)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < S - 1; ++i) stage(i);

    // operand addresses: 4 k + quad = 4 k ^ quad and so on, so one base and an xor each
    const uint32_t ka = ring + (uint32_t)col * ROWB + 16u * (uint32_t)(quad ^ k_swizzle<D>(col));
    const int vr = 4 * quad + (col >> 2);
    const uint32_t va = ring + MAT + (uint32_t)vr * ROWB + 16u * (uint32_t)(((col >> 1) & 1) ^ v_swizzle<D>(vr)) +
                        8u * (uint32_t)(col & 1);

    const float scale = a.scale * kLog2e;
    f4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f4{0, 0, 0, 0};
    float m = kNone, l = 0.0f;
    bool dirty = false;
    for (int step = 0; step < steps; ++step) {
        stage(step + S - 1);
        if (step + S <= steps)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * 2 * NI) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const int k0 = kNarrowKeys * (begin + wave + W * step);
        const uint32_t at = (uint32_t)(step % S) * STAGE;
        // (opaque, so that a piece's addresses are not kept in registers over the loop)
        uint32_t kt = ka + at, vt = va + at;
        asm("" : "+v"(kt), "+v"(vt));
        f4 x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int b = 0; b < 2; ++b)
                x[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(*(lds_h8)((kt ^ (64u * k)) + 16u * b * ROWB), q[k],
                                                              x[b], 0, 0, 0);
        const bool masked = k0 + kNarrowKeys - 1 > t.first || (a.window > 0 && k0 <= t.last - a.window);
        const int ahead = pos - k0 - 4 * quad, behind = a.window > 0 ? ahead - a.window : INT_MIN;
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[b][e] *= scale;
                if (masked && (16 * b + e > ahead || 16 * b + e <= behind)) x[b][e] = -INFINITY;
                top = fmaxf(top, x[b][e]);
            }
        top = xor_butterfly<32, 16>(top, max_raw);
        const bool up = top > m + kLag;
        if (__ballot(up)) {
            const float f = up ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            m = up ? top : m;
            l *= f;
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= f;
        }
        h8 p;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[4 * b + e] = (_Float16)__builtin_amdgcn_exp2f(x[b][e] - m);
        l = sum8(p, l);
        // V^T: lane (dim 16 i + col) takes keys 4 quad + {0 .. 3, 16 .. 19}, as p holds them.
        // Infinities and NaN among values that some rows do not see must not meet their zero
        // weights: finite ones take their place, and the rows that see them get them at the end.
        Finite fin;
#pragma unroll
        for (int i0 = 0; i0 < NB; i0 += 4) {
            h8 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t row = vt ^ (32u * (i0 + i));
                v[i] = join(read_tr(row), read_tr(row + 16u * ROWB));
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    fin.take(v[i]);
                    v[i] = finite_of(v[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i], p, o[i0 + i], 0, 0, 0);
        }
        if (masked) dirty = dirty || !fin.all();
    }
    if (dirty) {
        // the values that were replaced, to the rows that see them
        const int psh = units.psh, pmask = units.pmask;
        const int* table = units.table;
        const uint16_t* vc = c.v + kvh * c.head_stride;
#pragma unroll 1
        for (int k0 = kNarrowKeys * begin; k0 < kNarrowKeys * end; ++k0) {
            const int k32 = k0 & ~31;
            if (k32 / kNarrowKeys % W != (begin + wave) % W || k0 < t.lo || k0 >= t.hi) continue;
            if (!(k32 + 31 > t.first || (a.window > 0 && k32 <= t.last - a.window))) continue;
            const int page = table[k0 >> psh];
            if ((unsigned)page >= (unsigned)c.num_pages) continue;
            const uint16_t* row = vc + (int64_t)page * c.page_stride + (int64_t)(k0 & pmask) * c.row_stride + 4 * quad;
            const bool seen = k0 <= pos && (a.window == 0 || k0 > pos - a.window);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const h4 w = *reinterpret_cast<const h4*>(row + 16 * i), f = finite_of(w);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = seen ? o[i][e] + ((float)w[e] - (float)f[e]) : o[i][e];
            }
        }
    }
    l = xor_sum<32, 16>(l);
    if (bad) l = NAN;
    // the waves' states
    float* join_o = reinterpret_cast<float*>(lds);
    float* join_m = join_o + W * kNarrowRows * PADD;
    float* join_l = join_m + W * kNarrowRows;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NB; ++i)
        *reinterpret_cast<f4*>(join_o + (wave * kNarrowRows + col) * PADD + 16 * i + 4 * quad) = o[i];
    if (quad == 0) {
        join_m[wave * kNarrowRows + col] = m;
        join_l[wave * kNarrowRows + col] = l;
    }
    __syncthreads();
    const int live = min(rows - r0, kNarrowRows);
    float* part = slot_of<kNarrowRows, D>(plan.states, s, s.part, kvh, nkv);
    for (int i = threadIdx.x; i < live * (D / 4); i += 64 * W) {
        const int row = i / (D / 4), d = 4 * (i % (D / 4));
        float mx = kNone, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, join_m[w * kNarrowRows + row]);
        f4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = __builtin_amdgcn_exp2f(join_m[w * kNarrowRows + row] - mx);
            sum += join_l[w * kNarrowRows + row] * f;
            acc += *reinterpret_cast<f4*>(join_o + (w * kNarrowRows + row) * PADD + d) * f;
        }
        if (s.parts > 1) {
            *reinterpret_cast<f4*>(part + row * D + d) = acc;
            if (d == 0) {
                part[kNarrowRows * D + row] = mx;
                part[kNarrowRows * (D + 1) + row] = sum;
            }
        } else {
            const int tk = token_of(plan, r0 + row), hd = r0 + row - tk * plan.group;
            // (a row in front of position 0 sees nothing; one whose scores are all -inf is 0 / 0)
            store4(a, (int64_t)(s.q0 + tk) * a.ld_out + (int64_t)(kvh * plan.group + hd) * D + d,
                   s.kv - s.n + tk < 0 ? f4{0, 0, 0, 0} : acc * (1.0f / sum));
        }
    }
}

// ---- the launches -------------------------------------------------------------------------

// Head dims, waves and stages of the narrow part, waves of the wide one.
// W, S: heavy workgroups of the narrow launch, one a CU; LW, LS: light ones, two a CU, so
// that one's chain of loads runs beside the other's loop, for many tiles and beside wide
// items (256 requests of 600 positions 148 -> 126 us; one of 2000 9.0 -> 9.5).
template <int D> struct Shape;
template <> struct Shape<64> { static constexpr int W = 4, S = 4, LW = 4, LS = 2, NW = 4, M = 32; };
template <> struct Shape<128> { static constexpr int W = 4, S = 2, LW = 2, LS = 2, NW = 4, M = 32; };
template <> struct Shape<256> { static constexpr int W = 2, S = 2, LW = 1, LS = 2, NW = 8, M = 16; };
template <int D>
constexpr int narrow_lds(int w, int s) { return w * s * 2 * kNarrowKeys * 2 * D; }
template <int D>
constexpr int wide_lds() { return 4 * kWideKeys * 2 * D; }
template <int D>
constexpr int wide_rows() { return Shape<D>::M * Shape<D>::NW; }
static_assert(wide_rows<64>() == kWideRows && wide_rows<128>() == kWideRows && wide_rows<256>() == kWideRows,
              "the workspace's tiles");

template <int D, bool LIGHT>
__global__ __launch_bounds__(64 * (LIGHT ? Shape<D>::LW : Shape<D>::W))
void rf_paged_attn_narrow_kernel(const rf_paged_attention a, const rf_paged_cache c, const Plan plan) {
    constexpr int W = LIGHT ? Shape<D>::LW : Shape<D>::W, S = LIGHT ? Shape<D>::LS : Shape<D>::S;
    __shared__ __align__(1024) uint8_t lds[narrow_lds<D>(W, S)];
    narrow_part<D, W, S>(a, c, plan, (int)(blockIdx.x + blockIdx.y * gridDim.x), lds);
}

// Both kinds in one launch, the wide items first: their workgroups are the
// longer ones, and the narrow ones fill the CUs that they leave.
template <int D>
__global__ __launch_bounds__(64 * Shape<D>::NW) __attribute__((amdgpu_waves_per_eu(2)))
void rf_paged_attn_mixed_kernel(const rf_paged_attention a, const rf_paged_cache c, const Plan wide, const Plan narrow) {
    constexpr int LW = Shape<D>::LW, LS = Shape<D>::LS, NEED = narrow_lds<D>(LW, LS);
    __shared__ __align__(1024) uint8_t lds[NEED > wide_lds<D>() ? NEED : wide_lds<D>()];
    const int item = (int)(blockIdx.x + blockIdx.y * gridDim.x);
    if (item < wide.items) {
        wide_part<D, Shape<D>::NW, Shape<D>::M>(a, c, wide, item, lds);
    } else {
        if (threadIdx.x >= 64 * LW) return;      // whole waves, before any barrier
        narrow_part<D, LW, LS>(a, c, narrow, item - wide.items, lds);
    }
}

template <int D>
__global__ __launch_bounds__(256) void rf_paged_attn_join_kernel(const rf_paged_attention a, const rf_paged_cache c,
                                                                 const Plan wide, const Plan narrow, int wide_items) {
    __shared__ float weight[kJoinParts][kJoinRows];
    __shared__ f4 sums[256];
    const int item = blockIdx.x;
    if (item < wide_items)
        join_part<D, wide_rows<D>(), kWideKeys>(a, c, wide, item, weight, sums);
    else
        join_part<D, kNarrowRows, kNarrowKeys>(a, c, narrow, item - wide_items, weight, sums);
}

}  // namespace rf

extern "C" size_t rf_paged_attention_workspace_bytes(int num_heads, int num_kv_heads, int head_dim) {
    if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0) return 0;
    switch (head_dim) {
    case 64: return rf::narrow_bytes<64>() + rf::wide_bytes<64>();
    case 128: return rf::narrow_bytes<128>() + rf::wide_bytes<128>();
    case 256: return rf::narrow_bytes<256>() + rf::wide_bytes<256>();
    default: return 0;
    }
}

template <int D>
static void attn_go(const rf_paged_attention& a, const rf_paged_cache& c, hipStream_t stream) {
    using namespace rf;
    constexpr int ROWS = wide_rows<D>();
    const int nkv = c.num_kv_heads, group = a.num_heads / nkv;
    const int64_t packed = (int64_t)a.rows * group, positions = (int64_t)a.max_blocks * c.page_size;
    const bool both = (int64_t)a.max_new * group > kNarrowRows;
    float* ws = static_cast<float*>(a.workspace);
    const auto inverse = [](int n) { return (uint32_t)(((1ll << 32) + n - 1) / n); };
    const uint32_t inv = packed * group < (1ll << 32) ? inverse(group) : 0;
    const int64_t some = std::min<int64_t>(a.num_seqs, a.rows);        // requests with rows
    // The narrow launch.  Fewer than 64 tiles, or up to 256 of short tables: 256 parts, one round of
    // workgroups with most loads in flight.  Else up to 256: two workgroups a CU, and half a part less for
    // every tile, since the last part of a tile is half a one on average -- one round again.  Up to 511: two rounds
    // of heavy workgroups.  From 512 tiles on 512 parts of light ones.  us (graph, 8 KV heads of 128 unless
    // said), 256 parts of heavy ones / 512 of heavy ones / 512 of light ones / 512 - tiles / 2 of light ones:
    //   up to 63 tiles        2 requests of 8000         19.1 / 24.0 / 20.0 / 20.1
    //   64 to 256             8 of 100 to 8000           20.1 / 18.8 / 15.9 / 15.9
    //                         20 of 4000                 76.5 / 71.1 / 75.3 / 59.8
    //                         32 of 100 to 8000          82.5 / 75.5 / 83.3 / 69.7
    //     in a short table    8 of 2000                  18.8 / 22.2 / 18.5 / 19.7
    //                         32 of 1000                 25.8 / 30.9 / 27.6 / 27.6
    //   257 to 511            48 of 60 to 16000           134 /  125 /  140 /  128
    //                         the same, heads of 64      86.7 / 77.5 / 67.8 / 64.8
    //                         the same, heads of 256      249 /  206 /  233 /  225
    //   from 512 on           256 of 600                  149 /  149 /  126 /  126
    //                         64 of 2000                 98.0 / 98.5 / 96.0 / 95.7
    //                         300 of 20 to 4000           203 /  208 /  201 /  196
    //                         128 of 20 to 8000           168 /  149 /  160 /  201
    //                         the same, heads of 64       137 /  124 /  102 /  133
    //                         the same, heads of 256      379 /  322 /  352 /  522
    // So from 257 tiles on no choice wins throughout: very ragged batches of 512 tiles and more would run up to 9 %
    // faster with heavy workgroups, even ones 18 % slower, and heads of 64 in the band before with light ones.
    const int64_t tiles = some * nkv;
    const bool few = !both && (tiles < 64 || (tiles <= 256 && positions <= 2048)), some_tiles = !both && !few && tiles <= 256;
    const bool light = both || some_tiles || tiles >= 512;
    const int aim = few ? 256 : some_tiles ? kNarrowParts - (int)tiles / 2 : kNarrowParts;
    const auto least = [&](int keys, int whole, int cut) { return positions <= whole * keys ? whole : cut; };
    const int narrow_least = least(kNarrowKeys, both || tiles >= 256 ? kManyWhole : kFewWhole,
                                   both ? kBesideLeast : kNarrowLeast);
    Plan narrow = {group, inv, 0, both ? kNarrowRows : INT_MAX, aim, narrow_least, inverse(aim), 0, ws};
    // (fewer parts for many wide tiles likewise, a quarter of one a tile.  us, none less / a quarter / half of one:
    // 100 single tokens beside 4 prompts of 300 159 / 144 / 137, 512 tokens behind 8000 three times 223 / 224 / 235)
    const int64_t wide_tiles = (packed / ROWS + std::min(some, packed / kNarrowRows)) * nkv;
    const int wide_aim = (int)std::max<int64_t>(wide_parts<D>() - wide_tiles / 4, wide_parts<D>() / 4);
    Plan wide = {group, inv, kNarrowRows, INT_MAX, wide_aim, least(kWideKeys, kWideWhole, kWideLeast), inverse(wide_aim), 0,
                 ws + rf::narrow_bytes<D>() / sizeof(float)};
    // Items: every tile has a part, and there are at most as many parts more as are aimed at (each of
    // them a share long); no more either than the table's width gives room for.
    const auto items = [&](int64_t tiles, const Plan& p, int keys, int64_t* joins) {
        const int64_t most = std::max<int64_t>((positions + keys * p.least - 1) / (keys * p.least), 1);
        *joins = most > 1 ? std::min<int64_t>(tiles, p.parts) : 0;
        return (int)std::min(tiles + p.parts, tiles * most);
    };
    int64_t narrow_joins, wide_joins = 0;
    narrow.items = items((both ? some : packed / kNarrowRows + some) * nkv, narrow, kNarrowKeys, &narrow_joins);
    if (both) {
        wide.items = items(wide_tiles, wide, kWideKeys, &wide_joins);
        // (workgroups i and i + 8 share an XCD's L2, and items i and i + num_kv_heads their K and V)
        wide.items = (wide.items + 8 * nkv - 1) / (8 * nkv) * (8 * nkv);
    }
    const unsigned total = (unsigned)wide.items + (unsigned)narrow.items;
    const dim3 grid(std::min(total, 1u << 20), (total + (1u << 20) - 1) >> 20);
    if (both)
        hipLaunchKernelGGL(rf_paged_attn_mixed_kernel<D>, grid, dim3(64 * Shape<D>::NW), 0, stream, a, c, wide, narrow);
    else
        hipLaunchKernelGGL((light ? rf_paged_attn_narrow_kernel<D, true> : rf_paged_attn_narrow_kernel<D, false>), grid,
                           dim3(64 * (light ? Shape<D>::LW : Shape<D>::W)), 0, stream, a, c, narrow);
    const int wide_blocks = (int)wide_joins * (ROWS / kJoinRows);
    if (wide_joins + narrow_joins > 0)
        hipLaunchKernelGGL(rf_paged_attn_join_kernel<D>, dim3((unsigned)(wide_blocks + narrow_joins)), dim3(256), 0,
                           stream, a, c, wide, narrow, wide_blocks);
}

extern "C" hipError_t rf_paged_attention_launch(const rf_paged_attention* step, const rf_paged_cache* cache,
                                                hipStream_t stream) {
    if (step == nullptr || cache == nullptr) return hipErrorInvalidValue;
    rf_paged_attention a = *step;
    const rf_paged_cache& c = *cache;
    if (!rf::cache_ok(c) || !rf::attention_ok(a, c)) return hipErrorInvalidValue;
    if (a.rows == 0 || a.num_seqs == 0) return hipSuccess;
    if (!rf::attention_buffers_ok(a, c)) return hipErrorInvalidValue;
    if (a.window >= (int64_t)a.max_blocks * c.page_size) a.window = 0;     // reaches past every position
    switch (c.head_dim) {
    case 64: attn_go<64>(a, c, stream); break;
    case 128: attn_go<128>(a, c, stream); break;
    default: attn_go<256>(a, c, stream); break;
    }
    return hipGetLastError();
}
