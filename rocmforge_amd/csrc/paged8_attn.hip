// paged8_attn.hip -- causal GQA attention of the new rows of a batch over 8-bit
// pages (rf_paged_attention8_launch; the header states what it computes,
// paged_attn.h how a batch is cut).  No counterpart in the reference.
//
// Codes become fp16 values, exactly, on their way into the MFMAs: both the fp16
// kernels' sums and their rules for masks, infinities and NaN hold as they are.
#include "paged8.h"
#include "paged_attn.h"

namespace rf {

typedef int i2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i2* lds_i2;
typedef __attribute__((address_space(3))) const u32x4* lds_u4;

// A row of D codes in LDS lies as in memory, its 16-byte pieces permuted so that neither
// K's reads (one piece of 16 rows) nor V's transposing ones (one piece of the rows 8 i .. 8 i + 7
// and 16 further, i = 0 or 1) meet a bank twice; 256 / D rows fill the banks.
template <int D>
__device__ __forceinline__ int k_swizzle8(int row) {
    return D == 64 ? (row >> 2) & 3 : D == 128 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle8(int row) {
    const int far = (row >> 4) & 1;
    return D == 64 ? ((row >> 2) & 1) | (far << 1) : D == 128 ? ((row >> 1) & 3) | (far << 2) : (row & 7) | (far << 3);
}

// 16 bytes a lane from each lane's own address into LDS at m0 + 16 lane
__device__ __forceinline__ void lds_dma16_at(uint32_t lds_dst, uint64_t at) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_dst), "v"(at) : "memory", "m0");
}

// ---- few rows -------------------------------------------------------------------------
//
// As over fp16 pages (paged_attn.hip): wave w takes the pieces of 32 positions w, w + W, .. of
// the part through its own S-stage ring in LDS, codes as they are; they become fp16 in
// registers, K's under its row's exponent and V's under their keys' (lane 4 i + j of a window
// of 16 pieces holds address and exponents of piece i's unit j of 8 positions).
template <int D, int W, int S>
__device__ __forceinline__ void narrow8_part(const rf_paged_attention& a, const rf_paged_cache8& c, const Plan& plan,
                                             int item, uint8_t* lds) {
    constexpr int MAT = kNarrowKeys * D, STAGE = 2 * MAT;
    constexpr int LPR = D / 16, RPI = 64 / LPR, NI = kNarrowKeys / RPI;           // lanes a row, rows an instruction
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
    const Units<rf_paged_cache8> units(a, c, s.b, kvh, t.lo, t.hi);
    const int bsh = block_shift(c);
    bool bad = false;
    int window = 0;
    uint64_t address = 0;
    int scales = 0, scales_before = 0;                   // K's and V's byte; of the window before, whose pieces may still wait
    const uint64_t v_from_k = (uint64_t)c.v - (uint64_t)c.k;
    const uint32_t stride = (uint32_t)c.row_stride;
    auto load_units = [&](int step) {
        const int unit = 4 * (begin + wave + W * (step + (lane >> 2))) + (lane & 3);
        const int page = units.page_of(unit);
        address = units.address(unit, page, bad);
        const int64_t at = scale_at(c, (unsigned)page >= (unsigned)c.num_pages ? 0 : page,
                                    (8 * units.seen(unit)) & units.pmask, bsh) + kvh;
        scales_before = scales;
        scales = scale_byte(c.k_scale[at]) | (scale_byte(c.v_scale[at]) << 8);
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
            const uint32_t kp = 16u * (uint32_t)(ds ^ k_swizzle8<D>(lr)), vp = 16u * (uint32_t)(ds ^ v_swizzle8<D>(lr));
            const uint32_t kd = __builtin_amdgcn_readfirstlane(dst + 1024u * i);
            const uint32_t vd = __builtin_amdgcn_readfirstlane(dst + MAT + 1024u * i);
            // positions that no row sees are taken from the nearest one that some row sees
            if constexpr (RPI > 8) {
                // two units an instruction
                const int key = whole ? k0 + lr : min(max(k0 + lr, t.lo), t.hi - 1);
                const uint64_t lo = read_lane(address, 4 * (step - window) + 2 * i);
                const uint64_t hi = read_lane(address, 4 * (step - window) + 2 * i + 1);
                const int unit = units.seen(4 * piece + 2 * i + (lane >> 5));
                const uint64_t at = (lane < 32 ? lo : hi) + (uint64_t)((uint32_t)(key - 8 * unit) * stride);
                lds_dma16_at(kd, at + kp);
                lds_dma16_at(vd, at + v_from_k + vp);
            } else {
                int unit = 4 * piece + (RPI * i >> 3);
                uint32_t row = (uint32_t)((RPI * i & 7) + dr) * stride;
                if (!whole) {
                    unit = units.seen(unit);
                    row = (uint32_t)(min(max(k0 + lr, t.lo), t.hi - 1) - 8 * unit) * stride;
                }
                const uint64_t at = read_lane(address, 4 * (step - window) + unit - 4 * piece);
                lds_dma16(kd, row + kp, reinterpret_cast<const uint8_t*>(at));
                lds_dma16(vd, row + vp, reinterpret_cast<const uint8_t*>(at + v_from_k));
            }
        }
    };
    // dims 64 j + 16 quad + {0 .. 7, 8 .. 15} are this lane's of k-steps 2 j and 2 j + 1, as K's 16-byte reads have them
    h8 q[KS];
    const uint16_t* qrow = a.q + (int64_t)(s.q0 + token) * a.ld_q + (int64_t)(kvh * plan.group + head) * D + 16 * quad;
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const h8*>(qrow + 64 * (k >> 1) + 8 * (k & 1));
    if (steps > 0) load_units(0);
    // (q has arrived before the DMAs start, so that none but theirs are counted below)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < S - 1; ++i) stage(i);

    // operand addresses: one base and an xor each
    const uint32_t ka = ring + (uint32_t)col * D + 16u * (uint32_t)(quad ^ k_swizzle8<D>(col));
    const int vr = 4 * quad + ((col >> 1) & 3) + 16 * (col >> 3);
    const uint32_t va = ring + MAT + (uint32_t)vr * D + 16u * (uint32_t)v_swizzle8<D>(vr) + 8u * (uint32_t)(col & 1);

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
        // the exponents: K's of rows col and 16 + col, V's of keys 4 quad .. and 16 + 4 quad ..
        const int held = step >= window ? scales : scales_before, w0 = 4 * (step & 15);
        auto of_unit = [&](int unit) { return __builtin_amdgcn_ds_bpermute(4 * (w0 + unit), held); };
        float ks[2], vs[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            ks[b] = pow2_of(of_unit(2 * b + (col >> 3)) & 0xff);
            vs[b] = pow2_of(of_unit(2 * b + (quad >> 1)) >> 8);
        }
        f4 x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int j = 0; j < KS / 2; ++j)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                h8 lo, hi;
                values_of(*(lds_u4)((kt ^ (64u * j)) + 16u * b * D), ks[b], lo, hi);
                x[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, q[2 * j], x[b], 0, 0, 0);
                x[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, q[2 * j + 1], x[b], 0, 0, 0);
            }
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
        // V^T: lane (dim 16 i + col) takes keys 4 quad + {0 .. 3, 16 .. 19}, as p holds them.  NaN
        // among values that some rows do not see must not meet their zero weights: finite values
        // take its place, and the rows that see it get it at the end.
        Finite fin;
#pragma unroll
        for (int i0 = 0; i0 < NB; i0 += 4) {
            h8 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const i2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2)(vt ^ (16u * (i0 + i))));
                v[i] = join(__builtin_shufflevector(two_of<false>(w[0], vs[0]), two_of<true>(w[0], vs[0]), 0, 1, 2, 3),
                            __builtin_shufflevector(two_of<false>(w[1], vs[1]), two_of<true>(w[1], vs[1]), 0, 1, 2, 3));
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
        // the NaN that were replaced, to the rows that see them
        const uint8_t* vc = c.v + kvh * c.head_stride;
#pragma unroll 1
        for (int k0 = kNarrowKeys * begin; k0 < kNarrowKeys * end; ++k0) {
            const int k32 = k0 & ~31;
            if (k32 / kNarrowKeys % W != (begin + wave) % W || k0 < t.lo || k0 >= t.hi) continue;
            if (!(k32 + 31 > t.first || (a.window > 0 && k32 <= t.last - a.window))) continue;
            const int page = units.table[k0 >> units.psh];
            if ((unsigned)page >= (unsigned)c.num_pages) continue;
            const uint8_t* row = vc + (int64_t)page * c.page_stride + (int64_t)(k0 & units.pmask) * c.row_stride + 4 * quad;
            const bool seen = k0 <= pos && (a.window == 0 || k0 > pos - a.window);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 16 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = seen && ((w >> (8 * e)) & 0x7f) == 0x7f ? NAN : o[i][e];
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

// Waves and stages of the narrow part, waves of the wide one and their packed rows.  Two
// stages a wave, so that two and more workgroups share a CU: 48 requests of 60 to 16000 positions
// (head_dim 128) 52.4 us, with three stages and one workgroup a CU 67; at 64 a third stage is even
// (47.7 and 48.1 us, 64 requests of 2000).  At 256 two waves, for the same reason: 256 requests
// of 600 138 us, with four waves 166.
template <int D> struct Shape8;
template <> struct Shape8<64> { static constexpr int W = 4, S = 2, LW = 4, LS = 4, NW = 4, M = 32, PER_CU = 2; };
template <> struct Shape8<128> { static constexpr int W = 4, S = 2, LW = 4, LS = 2, NW = 4, M = 32, PER_CU = 2; };
template <> struct Shape8<256> { static constexpr int W = 2, S = 2, LW = 2, LS = 2, NW = 8, M = 16, PER_CU = 1; };
constexpr int kNarrowLeast8 = 4, kBesideLeast8 = 16, kWideLeast8 = 24;
constexpr int kFewWhole8 = 16, kManyWhole8 = 32, kWideWhole8 = 32;
template <int D>
constexpr int narrow8_lds(int w, int s) { return w * s * 2 * kNarrowKeys * D; }
template <int D>
constexpr int wide8_lds() { return 4 * kWideKeys * 2 * D; }
template <int D>
constexpr int wide8_rows() { return Shape8<D>::M * Shape8<D>::NW; }
template <int D>
constexpr int wide8_parts() { return 256 * Shape8<D>::PER_CU; }

template <int D>
__global__ __launch_bounds__(64 * Shape8<D>::W)
void rf_paged8_attn_narrow_kernel(const rf_paged_attention a, const rf_paged_cache8 c, const Plan plan) {
    constexpr int W = Shape8<D>::W, S = Shape8<D>::S;
    __shared__ __align__(1024) uint8_t lds[narrow8_lds<D>(W, S)];
    narrow8_part<D, W, S>(a, c, plan, (int)(blockIdx.x + blockIdx.y * gridDim.x), lds);
}

// Both kinds in one launch, the wide items first: their workgroups are the
// longer ones, and the narrow ones fill the CUs that they leave.
template <int D>
__global__ __launch_bounds__(64 * Shape8<D>::NW) __attribute__((amdgpu_waves_per_eu(2)))
void rf_paged8_attn_mixed_kernel(const rf_paged_attention a, const rf_paged_cache8 c, const Plan wide, const Plan narrow) {
    constexpr int LW = Shape8<D>::LW, LS = Shape8<D>::LS, NEED = narrow8_lds<D>(LW, LS);
    __shared__ __align__(1024) uint8_t lds[NEED > wide8_lds<D>() ? NEED : wide8_lds<D>()];
    const int item = (int)(blockIdx.x + blockIdx.y * gridDim.x);
    if (item < wide.items) {
        wide_part<D, Shape8<D>::NW, Shape8<D>::M>(a, c, wide, item, lds);
    } else {
        if (threadIdx.x >= 64 * LW) return;      // whole waves, before any barrier
        narrow8_part<D, LW, LS>(a, c, narrow, item - wide.items, lds);
    }
}

template <int D>
__global__ __launch_bounds__(256) void rf_paged8_attn_join_kernel(const rf_paged_attention a, const rf_paged_cache8 c,
                                                                  const Plan wide, const Plan narrow, int wide_items) {
    __shared__ float weight[kJoinParts][kJoinRows];
    __shared__ f4 sums[256];
    const int item = blockIdx.x;
    if (item < wide_items)
        join_part<D, wide8_rows<D>(), kWideKeys>(a, c, wide, item, weight, sums);
    else
        join_part<D, kNarrowRows, kNarrowKeys>(a, c, narrow, item - wide_items, weight, sums);
}

}  // namespace rf

template <int D>
static void attn8_go(const rf_paged_attention& a, const rf_paged_cache8& c, hipStream_t stream) {
    using namespace rf;
    constexpr int ROWS = wide8_rows<D>();
    const int nkv = c.num_kv_heads, group = a.num_heads / nkv;
    const int64_t packed = (int64_t)a.rows * group, positions = (int64_t)a.max_blocks * c.page_size;
    const bool both = (int64_t)a.max_new * group > kNarrowRows;
    float* ws = static_cast<float*>(a.workspace);
    const auto inverse = [](int n) { return (uint32_t)(((1ll << 32) + n - 1) / n); };
    const uint32_t inv = packed * group < (1ll << 32) ? inverse(group) : 0;
    const int64_t some = std::min<int64_t>(a.num_seqs, a.rows);        // requests with rows
    const int64_t tiles = some * nkv;
    // Few tiles in a part a CU, more in nearly two, as the joins cost little beside the ragged
    // end then (head_dim 128): one request of 16000 positions 17.3 us at 256 parts and 18.9 at 400,
    // 20 of 4000 49.1 and 44.1, 48 of 60 to 16000 56.9, 52.4 and, at 512, 57.8.
    const int aim = tiles < 64 ? 256 : 400;
    const auto least = [&](int keys, int whole, int cut) { return positions <= whole * keys ? whole : cut; };
    const int narrow_least = least(kNarrowKeys, both || tiles >= 256 ? kManyWhole8 : kFewWhole8,
                                   both ? kBesideLeast8 : kNarrowLeast8);
    Plan narrow = {group, inv, 0, both ? kNarrowRows : INT_MAX, aim, narrow_least, inverse(aim), 0, ws};
    const int64_t wide_tiles = (packed / ROWS + std::min(some, packed / kNarrowRows)) * nkv;
    const int wide_aim = (int)std::max<int64_t>(wide8_parts<D>() - wide_tiles / 4, wide8_parts<D>() / 4);
    Plan wide = {group, inv, kNarrowRows, INT_MAX, wide_aim, least(kWideKeys, kWideWhole8, kWideLeast8), inverse(wide_aim), 0,
                 ws + narrow_bytes<D>() / sizeof(float)};
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
        hipLaunchKernelGGL(rf_paged8_attn_mixed_kernel<D>, grid, dim3(64 * Shape8<D>::NW), 0, stream, a, c, wide, narrow);
    else
        hipLaunchKernelGGL(rf_paged8_attn_narrow_kernel<D>, grid, dim3(64 * Shape8<D>::W), 0, stream, a, c, narrow);
    const int wide_blocks = (int)wide_joins * (ROWS / kJoinRows);
    if (wide_joins + narrow_joins > 0)
        hipLaunchKernelGGL(rf_paged8_attn_join_kernel<D>, dim3((unsigned)(wide_blocks + narrow_joins)), dim3(256), 0,
                           stream, a, c, wide, narrow, wide_blocks);
}

extern "C" hipError_t rf_paged_attention8_launch(const rf_paged_attention* step, const rf_paged_cache8* cache,
                                                 hipStream_t stream) {
    if (step == nullptr || cache == nullptr) return hipErrorInvalidValue;
    rf_paged_attention a = *step;
    const rf_paged_cache8& c = *cache;
    if (!rf::cache8_ok(c) || !rf::attention_ok(a, c)) return hipErrorInvalidValue;
    if (a.rows == 0 || a.num_seqs == 0) return hipSuccess;
    if (!rf::attention_buffers_ok(a, c)) return hipErrorInvalidValue;
    if (a.window >= (int64_t)a.max_blocks * c.page_size) a.window = 0;     // reaches past every position
    switch (c.head_dim) {
    case 64: attn8_go<64>(a, c, stream); break;
    case 128: attn8_go<128>(a, c, stream); break;
    default: attn8_go<256>(a, c, stream); break;
    }
    return hipGetLastError();
}
